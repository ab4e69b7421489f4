// New keys and values into a paged cache, keys normed and turned by their
// positions on the way, queries alike (include/templit_cuda.h:
// tl_cache_append).
//
// Bound by memory, and by latency where there are few tokens: a warp finds its
// token's sequence (one or two rounds of 32 starts), position and page, and
// takes a run of the token's query, key or value heads, as in k_rotary.cu.
// 64 tokens, one a sequence, 32 query and 8 key heads of 128 bf16: 7 us, a launch and that
// chain of lookups; the new tokens of 16 sequences, up to 1000 each, from fp32: 20.6 us
// (102 MB, 4.9 TB/s), where a warp's item begins with that chain, which no other covers.
#include "paged_cache.cuh"

#include <cmath>

namespace tl {
namespace paged {

int check_cache(const char *who, tl_paged_cache &c, bool *aligned) {
  const std::string w = std::string(who) + ": ";
  if (!heads::known_type(c.type)) return fail(TL_ERR_INVALID, w + "unknown cache type");
  if (c.D == 0 || c.D > TL_HEAD_MAX_DIM) return fail(TL_ERR_RANGE, w + "a head has 1 to 256 elements");
  if (!c.heads) return fail(TL_ERR_INVALID, w + "no key heads");
  if (!c.page_size) return fail(TL_ERR_INVALID, w + "empty pages");
  if (c.sequences > 1u << 30) return fail(TL_ERR_RANGE, w + "more than 2^30 sequences");
  if (!c.page_stride && !c.slot_stride && !c.head_stride) {
    c.head_stride = c.D;
    c.slot_stride = static_cast<uint64_t>(c.heads) * c.D;
    c.page_stride = c.slot_stride * c.page_size;
  }
  const uint64_t e = heads::type_size(c.type), most = (1ull << 62) / e;
  const auto far = [&](uint64_t n, uint64_t stride) { return n > 1 && stride > most / (n - 1) / 4; };
  if (far(c.pages, c.page_stride) || far(c.page_size, c.slot_stride) || far(c.heads, c.head_stride))
    return fail(TL_ERR_RANGE, w + "the cache leaves the address space");
  if ((c.pages > 1 && c.page_stride < c.D) || (c.page_size > 1 && c.slot_stride < c.D) ||
      (c.heads > 1 && c.head_stride < c.D))
    return fail(TL_ERR_INVALID, w + "a cache stride is too small");
  if (c.sequences && c.tokens) {
    if (!c.starts || !c.lengths) return fail(TL_ERR_INVALID, w + "null starts or lengths");
    if (c.table_stride && !c.table) return fail(TL_ERR_INVALID, w + "null table");
    if (c.pages && (!c.k || !c.v)) return fail(TL_ERR_INVALID, w + "null cache");
    if ((reinterpret_cast<uintptr_t>(c.starts) | reinterpret_cast<uintptr_t>(c.lengths) | reinterpret_cast<uintptr_t>(c.table)) % 4)
      return fail(TL_ERR_INVALID, w + "starts, lengths or table not aligned");
    if (reinterpret_cast<uintptr_t>(c.k) % e || reinterpret_cast<uintptr_t>(c.v) % e)
      return fail(TL_ERR_INVALID, w + "the cache is not aligned to its type");
  }
  const uint64_t v = 16 / e;
  *aligned = aligned16(c.k) && aligned16(c.v) && c.page_stride % v == 0 && c.slot_stride % v == 0 &&
             c.head_stride % v == 0;
  return TL_OK;
}

namespace {

using heads::Slot;

constexpr int kWarps = 4, kThreads = kWarps * 32, kBatch = 4;

struct AppendPart {
  tl_head_view x;
  void *out;  // queries: [tokens, heads, D]; keys and values: the cache's pointer
  uint64_t out_row, out_head;
  const float *weight;
  uint32_t heads, ctas, chunks, run;  // runs of `run` heads
  bool cache, turned;
};
struct AppendArgs {
  tl_paged_cache cache;
  AppendPart part[3];  // queries, keys, values
  uint32_t parts, rotary, lanes;
  uint32_t checks;  // CTAs behind the parts' that look the sequences over
  bool interleaved, norm;
  float eps, inv_d, magnitude;
  const uint64_t *frequencies;
  uint32_t *status;
};

// By vectors (V > 1) or by single elements (V = 1, a head at a time).
template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
  pdl_enter();
  const tl_paged_cache &c = a.cache;
  const uint64_t most = table_keys(c);
  uint32_t cta = blockIdx.x, which = 0;
  if (cta >= gridDim.x - a.checks) {
    // also sequences that no row leads to
    for (uint32_t s = (gridDim.x - 1 - cta) * kThreads + threadIdx.x; s < c.sequences; s += a.checks * kThreads)
      if (sequence_of(c, s, most).bad) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
    return;
  }
  while (which + 1 < a.parts && cta >= a.part[which].ctas) cta -= a.part[which++].ctas;
  const AppendPart &part = a.part[which];
  const uint32_t lane = threadIdx.x & 31, lanes = a.lanes, at = lane & (lanes - 1), sub = lane / lanes, per = 32 / lanes;
  const bool norm = a.norm && part.turned;
  const uint64_t items = static_cast<uint64_t>(c.tokens) * part.chunks;
  const uint64_t warps = static_cast<uint64_t>(part.ctas) * kWarps;
  for (uint64_t item = static_cast<uint64_t>(cta) * kWarps + threadIdx.x / 32; item < items; item += warps) {
    const uint32_t token = static_cast<uint32_t>(item / part.chunks), chunk = static_cast<uint32_t>(item % part.chunks);
    const uint32_t first = chunk * part.run, end = min(first + part.run, part.heads);
    const TI *x = static_cast<const TI *>(part.x.p) + token * part.x.row_stride;
    // the first heads are on their way while the token's place is looked up
    const uint32_t rotary = part.turned ? a.rotary : 0;
    const Slot slot = heads::slot_of(at, V, c.D, rotary, a.interleaved);
    constexpr int W = V > 1 ? V : 4;  // (arrays of the single elements' form are not used)
    heads::Raw<TI, W> ra[kBatch], rb[kBatch];
    const auto load = [&](uint32_t h0) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t h = h0 + u * per + sub;
        const TI *row = x + h * part.x.head_stride;
        ra[u] = rb[u] = heads::Raw<TI, W>{};
        if (h < end && slot.has_a) ra[u].load(row + slot.a);
        if (h < end && slot.has_b) rb[u].load(row + slot.b);
      }
    };
    if constexpr (V > 1) load(first);
    const uint32_t s = sequence_at(c, token, lane);
    if (s == 0xffffffffu) continue;
    const uint32_t start = c.starts[s], stop = c.starts[s + 1], length = c.lengths[s];
    if (stop <= token) continue;  // behind the last sequence
    const int64_t position = static_cast<int64_t>(length) - (stop - token);
    bool ok = stop <= c.tokens && start <= token && length >= stop - start && static_cast<uint64_t>(position) < most;
    uint32_t page = 0;
    if (ok) {
      page = c.table[static_cast<uint64_t>(s) * c.table_stride + static_cast<uint32_t>(position) / c.page_size];
      ok = page < c.pages;
    }
    if (!ok) {
      if (lane == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
      continue;
    }
    TO *out = static_cast<TO *>(part.out);
    out += part.cache ? page * c.page_stride + static_cast<uint32_t>(position) % c.page_size * c.slot_stride
                      : token * part.out_row;
    if constexpr (V > 1) {
      float cos[V], sin[V], wa[V], wb[V];
      heads::angles<V>(a.frequencies, static_cast<uint32_t>(position), a.magnitude, at, lanes, rotary, cos, sin);
      if (norm) heads::load_weights<V>(part.weight, slot, wa, wb);
      for (uint32_t h0 = first; h0 < end; h0 += kBatch * per) {
        if (h0 != first) load(h0);
        float r[kBatch];
        if (norm) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u) r[u] = heads::squares(ra[u], rb[u]);
          heads::head_sums<kBatch>(r, lanes);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const uint32_t h = h0 + u * per + sub;
          heads::finish_head<TI, TO, V>(ra[u], rb[u], slot, cos, sin, wa, wb, norm ? rsqrtf(fmaf(r[u], a.inv_d, a.eps)) : 1.0f, norm,
                                        a.interleaved, h < end, out + h * part.out_head);
        }
      }
    } else {
      for (uint32_t h = first; h < end; ++h)
        heads::scalar_head<TI, TO>(x + h * part.x.head_stride, out + h * part.out_head, c.D, rotary, a.frequencies,
                                   static_cast<uint32_t>(position), a.magnitude, part.weight, norm, a.interleaved, a.inv_d, a.eps);
    }
  }
}

template <typename TI, typename TO> void launch_append(const AppendArgs &a, bool vectors, unsigned grid, cudaStream_t s) {
  constexpr int V = heads::vector_of(sizeof(TI), sizeof(TO));
  if (vectors) launch_pdl(append_kernel<TI, TO, V>, grid, kThreads, 0, s, a);
  else launch_pdl(append_kernel<TI, TO, 1>, grid, kThreads, 0, s, a);
}

// One launch for parts [0, a.parts) of one output type.
int append(const char *who, AppendArgs a, int32_t type, int32_t out_type, bool aligned, cudaStream_t s) {
  const heads::Shape shape = heads::shape_for(a.cache.D, a.rotary, heads::vector_for(type, out_type), aligned);
  a.lanes = shape.lanes;
  // Short runs of heads while the tokens are few: each warp's chain of loads
  // is what a small call costs.
  const uint32_t per = 32 / a.lanes, wanted = kNumSMs * 8;
  unsigned grid = 0;
  for (uint32_t i = 0; i < a.parts; ++i) {
    AppendPart &p = a.part[i];
    const uint32_t all = (p.heads + per - 1) / per;
    uint32_t steps = all;
    while (steps > 1 && static_cast<uint64_t>(a.cache.tokens) * ((all + steps - 1) / steps) < wanted)
      steps = (steps + 1) / 2;
    p.run = steps * per;
    p.chunks = (all + steps - 1) / steps;
    const uint64_t ctas = (static_cast<uint64_t>(a.cache.tokens) * p.chunks + kWarps - 1) / kWarps;
    p.ctas = static_cast<uint32_t>(ctas < kNumSMs * 256ull ? ctas : kNumSMs * 256ull);
    grid += p.ctas;
  }
  a.checks = a.cache.sequences / 1024 + 1 < kNumSMs ? a.cache.sequences / 1024 + 1 : kNumSMs;
  grid += a.checks;
#define L(TI, TO) launch_append<TI, TO>(a, shape.vectors, grid, s)
  if (type == TL_FLOAT16 && out_type == TL_BFLOAT16) L(__half, __nv_bfloat16);
  else if (type == TL_BFLOAT16 && out_type == TL_FLOAT16) L(__nv_bfloat16, __half);
  else TL_BY_TYPES(type, out_type, L)
#undef L
  return launch_status(who);
}

}  // namespace
}  // namespace paged
}  // namespace tl

using namespace tl;
using namespace tl::paged;

extern "C" int tl_cache_append(const tl_cache_append_desc *d, void *stream) {
  const char *who = "tl_cache_append";
  const std::string w = std::string(who) + ": ";
  if (!d) return fail(TL_ERR_INVALID, w + "null descriptor");
  if (!heads::known_type(d->type) || (d->q_heads && !heads::known_type(d->q_out_type)))
    return fail(TL_ERR_INVALID, w + "unknown type");
  AppendArgs a{};
  a.cache = d->cache;
  bool cache_aligned = false;
  if (int rc = check_cache(who, a.cache, &cache_aligned)) return rc;
  const tl_paged_cache &c = a.cache;
  // rows of one 16-bit type into a cache of the other, their queries to the type that the
  // attention over it reads; other mixtures have no reader
  if (d->q_heads && d->q_out_type != c.type && (heads::mixed_halves(d->type, c.type) || heads::mixed_halves(d->type, d->q_out_type)))
    return fail(TL_ERR_UNSUPPORTED, w + "fp16 and bf16 in one call with q_out of another type than the cache");
  if (int rc = heads::check_turn(who, c.D, d->rotary_dim, d->layout, d->norm, d->eps, d->magnitude, d->frequencies))
    return rc;
  if (!c.tokens || !c.sequences) return TL_OK;
  if (int rc = heads::check_view(who, "k", d->k, d->type, 1, c.tokens, c.heads, c.D, false)) return rc;
  if (int rc = heads::check_view(who, "v", d->v, d->type, 1, c.tokens, c.heads, c.D, false)) return rc;
  if ((reinterpret_cast<uintptr_t>(d->q_weight) | reinterpret_cast<uintptr_t>(d->k_weight)) % 4)
    return fail(TL_ERR_INVALID, w + "a weight is not aligned");
  bool q_aligned = true;
  if (d->q_heads) {
    if (int rc = heads::check_view(who, "q", d->q, d->type, 1, c.tokens, d->q_heads, c.D, false)) return rc;
    if (int rc = heads::check_view(who, "q_out", d->q_out, d->q_out_type, 1, c.tokens, d->q_heads, c.D, true)) return rc;
    if (heads::half_in_place(d->q_out, d->q_out_type, d->q, d->type, false))
      return fail(TL_ERR_INVALID, w + "q_out is q with another layout or type");
    q_aligned = heads::aligned_view(d->q, d->type, false, heads::vector_for(d->type, d->q_out_type)) &&
                heads::aligned_view(d->q_out, d->q_out_type, false, heads::vector_for(d->type, d->q_out_type));
  }
  a.rotary = d->rotary_dim;
  a.interleaved = d->layout == TL_ROTARY_INTERLEAVED;
  a.norm = d->norm;
  a.eps = d->eps;
  a.inv_d = 1.0f / c.D;
  a.magnitude = d->magnitude;
  a.frequencies = d->frequencies;
  a.status = device_status_ptr();
  if (!a.status) return fail(TL_ERR_CUDA, w + "no status word");
  const AppendPart q{d->q, const_cast<void *>(d->q_out.p), d->q_out.row_stride, d->q_out.head_stride, d->q_weight,
                     d->q_heads, 0, 0, 0, false, true};
  const AppendPart k{d->k, c.k, 0, c.head_stride, d->k_weight, c.heads, 0, 0, 0, true, true};
  const AppendPart v{d->v, c.v, 0, c.head_stride, nullptr, c.heads, 0, 0, 0, true, false};
  const bool aligned = cache_aligned && heads::aligned_view(d->k, d->type, false, heads::vector_for(d->type, c.type)) &&
                       heads::aligned_view(d->v, d->type, false, heads::vector_for(d->type, c.type));
  cudaStream_t s = as_stream(stream);
  if (d->q_heads && d->q_out_type != c.type) {
    // queries of another type than the cache's: a launch of their own
    a.parts = 1;
    a.part[0] = q;
    if (int rc = append(who, a, d->type, d->q_out_type, q_aligned, s)) return rc;
  }
  a.parts = 0;
  if (d->q_heads && d->q_out_type == c.type) a.part[a.parts++] = q;
  a.part[a.parts++] = k;
  a.part[a.parts++] = v;
  return append(who, a, d->type, c.type, aligned && (a.parts == 2 || q_aligned), s);
}
