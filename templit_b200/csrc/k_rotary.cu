// Queries and keys turned by their positions, optionally normed per head
// (include/templit_cuda.h: tl_rotary_frequencies, tl_rotary_heads), and the
// checks shared with the gradient and the cache.
//
//   y = x / sqrt(mean(x^2) + eps) * w          (norm)
//   (y_a, y_b) -> mag (y_a cos - y_b sin, y_a sin + y_b cos), angle = p f_i
//
// Bound by memory: every element is read once and written once.  A warp takes
// one token (its angles are worked out once, shared by the lanes) and a run of
// its heads, some side by side.
//
// 12288 x 12 heads of 64 fp32, rotation alone: 17 us (75 MB, 4.5 TB/s).  16384 x 40 heads of
// 128 bf16, norm and rotation: 68 us (336 MB, 4.9 TB/s), where the instructions of an element
// (issue 61 %) and loads (memory 54 %) share the time; 64 tokens of it 7 us, a launch.
#include "rotary.cuh"

#include <cmath>

namespace tl {
namespace heads {

int check_turn(const char *who, uint32_t D, uint32_t rotary_dim, int32_t layout, int32_t norm, float eps,
               float magnitude, const uint64_t *frequencies) {
  const std::string w = std::string(who) + ": ";
  if (D == 0 || D > TL_HEAD_MAX_DIM) return fail(TL_ERR_RANGE, w + "a head has 1 to 256 elements");
  if (rotary_dim % 2 || rotary_dim > D) return fail(TL_ERR_INVALID, w + "rotary_dim is even and at most D");
  if (layout != TL_ROTARY_HALF && layout != TL_ROTARY_INTERLEAVED) return fail(TL_ERR_INVALID, w + "unknown layout");
  if (norm != 0 && norm != 1) return fail(TL_ERR_INVALID, w + "norm is 0 or 1");
  if (norm && !(eps >= 0.0f && std::isfinite(eps))) return fail(TL_ERR_INVALID, w + "eps is finite and not negative");
  if (rotary_dim && !std::isfinite(magnitude)) return fail(TL_ERR_INVALID, w + "magnitude is finite");
  if (rotary_dim && !frequencies) return fail(TL_ERR_INVALID, w + "null frequencies");
  if (reinterpret_cast<uintptr_t>(frequencies) % 8) return fail(TL_ERR_INVALID, w + "frequencies not aligned");
  return TL_OK;
}

int check_view(const char *who, const char *name, const tl_head_view &v, int32_t type, uint64_t batches,
               uint64_t rows, uint64_t heads, uint32_t D, bool written) {
  const std::string w = std::string(who) + ": " + name;
  if (!v.p) return fail(TL_ERR_INVALID, w + " is null");
  if (reinterpret_cast<uintptr_t>(v.p) % type_size(type)) return fail(TL_ERR_INVALID, w + " is not aligned to its type");
  // the farthest element's offset, kept clear of 64 bits
  const uint64_t most = (1ull << 62) / type_size(type);
  const auto far = [&](uint64_t n, uint64_t stride) { return n > 1 && stride > most / (n - 1) / 4; };
  if (far(batches, v.batch_stride) || far(rows, v.row_stride) || far(heads, v.head_stride))
    return fail(TL_ERR_RANGE, w + " leaves the address space");
  if (written && ((batches > 1 && v.batch_stride < D) || (rows > 1 && v.row_stride < D) ||
                  (heads > 1 && v.head_stride < D)))
    return fail(TL_ERR_INVALID, w + " has a stride that is too small");
  return TL_OK;
}

namespace {

constexpr int kRotateRows = 2;  // head rows of a lane's batch

template <typename TI, typename TO, int V, int U, bool NORM, bool INTER>
__global__ void __launch_bounds__(kThreads, 4) rotate_kernel(const RotaryArgs a) {
  pdl_enter();
  const uint32_t lane = threadIdx.x & 31, lanes = a.lanes, at = lane & (lanes - 1), sub = lane / lanes, per = 32 / lanes;
  const uint64_t first_groups = static_cast<uint64_t>(a.tokens) * a.part[0].chunks;
  const uint64_t groups = a.whole ? a.tokens : first_groups + static_cast<uint64_t>(a.tokens) * a.part[1].chunks;
  const uint64_t warps = static_cast<uint64_t>(gridDim.x) * kWarps;
  const Slot slot = slot_of(at, V, a.D, a.rotary, INTER);

  Batch s;
  s.group = static_cast<uint64_t>(blockIdx.x) * kWarps + threadIdx.x / 32;
  set_batch(a, s, first_groups, groups);
  if (!s.any) return;
  const TI *x = static_cast<const TI *>(a.part[s.part].x.p) + place(a.part[s.part].x, s, sub);
  uint64_t x_step = per * a.part[s.part].x.head_stride;
  const auto left_of = [&](const Batch &s) { return s.end > s.head + sub ? s.end - s.head - sub : 0u; };
  HeadRows<TI, V, U> even, odd;
  even.clear();
  odd.clear();
  even.template load<false>(x, x_step, slot, left_of(s), per);
  uint64_t turned = ~0ull;  // the token whose angles are in cos and sin
  uint64_t of = ~0ull;      // the run that wa, wb and out are for
  float cos[V], sin[V], wa[V], wb[V];
  TO *out = nullptr;
  uint64_t out_step = 0;
  // one batch from `rows`, the next one into `next`; false behind the last
  const auto work = [&](const HeadRows<TI, V, U> &rows, HeadRows<TI, V, U> &next) {
    Batch n = s;
    if (next_batch(a, n, U * per, warps, first_groups, groups)) {
      x += U * x_step;
    } else if (n.any) {
      x = static_cast<const TI *>(a.part[n.part].x.p) + place(a.part[n.part].x, n, sub);
      x_step = per * a.part[n.part].x.head_stride;
    }
    if (n.any) next.template load<false>(x, x_step, slot, left_of(n), per);
    if (2 * s.group + s.part != of) {
      of = 2 * s.group + s.part;
      const RotaryPart &part = a.part[s.part];
      if (s.token != turned) {
        turned = s.token;
        angles<V>(a.frequencies, s.position, a.magnitude, at, lanes, a.rotary, cos, sin);
      }
      if (NORM) load_weights<V>(part.weight, slot, wa, wb);
      out = static_cast<TO *>(const_cast<void *>(part.out.p)) + place(part.out, s, sub);
      out_step = per * part.out.head_stride;
    }
    float r[U];
    if (NORM) {
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = squares(rows.a[u], rows.b[u]);
      head_sums<U>(r, lanes);
    }
    const uint32_t left = left_of(s);
#pragma unroll
    for (int u = 0; u < U; ++u)
      finish_head<TI, TO, V>(rows.a[u], rows.b[u], slot, cos, sin, wa, wb, NORM ? rsqrtf(fmaf(r[u], a.inv_d, a.eps)) : 1.0f, NORM, INTER,
                             u * per < left, out + u * out_step);
    out += U * out_step;
    s = n;
    return n.any;
  };
  while (work(even, odd) && work(odd, even)) {
  }
}

// A warp a head, by single elements.
template <typename TI, typename TO> __global__ void __launch_bounds__(kThreads) rotate_elements_kernel(const RotaryArgs a) {
  pdl_enter();
  const uint64_t heads = a.part[0].heads + static_cast<uint64_t>(a.part[1].heads), items = a.tokens * heads;
  const uint64_t warps = static_cast<uint64_t>(gridDim.x) * kWarps;
  for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * kWarps + threadIdx.x / 32; item < items; item += warps) {
    const uint32_t token = static_cast<uint32_t>(item / heads), b = token / a.T, t = token - b * a.T;
    uint32_t h = static_cast<uint32_t>(item - token * heads);
    const RotaryPart &p = a.part[h >= a.part[0].heads];
    if (h >= a.part[0].heads) h -= a.part[0].heads;
    const TI *x = static_cast<const TI *>(p.x.p) + b * p.x.batch_stride + t * p.x.row_stride + h * p.x.head_stride;
    TO *out = static_cast<TO *>(const_cast<void *>(p.out.p)) + b * p.out.batch_stride + t * p.out.row_stride + h * p.out.head_stride;
    scalar_head<TI, TO>(x, out, a.D, a.rotary, a.frequencies, a.positions ? a.positions[token] : a.first_position + t,
                        a.magnitude, p.weight, a.norm, a.interleaved, a.inv_d, a.eps);
  }
}

template <typename TI, typename TO> void launch_rotate(RotaryArgs &a, cudaStream_t s) {
  constexpr int V = vector_of(sizeof(TI), sizeof(TO)), U = kRotateRows;
  if (!a.vectors) {
    const uint64_t heads = a.part[0].heads + static_cast<uint64_t>(a.part[1].heads);
    launch_pdl(rotate_elements_kernel<TI, TO>, grid_for(a.tokens * heads, kWarps, 16), kThreads, 0, s, a);
    return;
  }
  const unsigned grid = share_out(a, U, kMaxCtas, false);
  if (a.norm) {
    if (a.interleaved) launch_pdl(rotate_kernel<TI, TO, V, U, true, true>, grid, kThreads, 0, s, a);
    else launch_pdl(rotate_kernel<TI, TO, V, U, true, false>, grid, kThreads, 0, s, a);
  } else {
    if (a.interleaved) launch_pdl(rotate_kernel<TI, TO, V, U, false, true>, grid, kThreads, 0, s, a);
    else launch_pdl(rotate_kernel<TI, TO, V, U, false, false>, grid, kThreads, 0, s, a);
  }
}

}  // namespace

int rotary_args(const char *who, const tl_rotary_desc *d, bool backward, RotaryArgs &a) {
  const std::string w = std::string(who) + ": ";
  if (!d) return fail(TL_ERR_INVALID, w + "null descriptor");
  if (!known_type(d->type) || !known_type(d->out_type)) return fail(TL_ERR_INVALID, w + "unknown type");
  if (mixed_halves(d->type, d->out_type)) return fail(TL_ERR_UNSUPPORTED, w + "fp16 and bf16 in one call");
  if (int rc = check_turn(who, d->D, d->rotary_dim, d->layout, d->norm, d->eps, d->magnitude, d->frequencies))
    return rc;
  const uint64_t tokens = static_cast<uint64_t>(d->B) * d->T;
  if (tokens >> 32) return fail(TL_ERR_RANGE, w + "more than 2^32 - 1 tokens");
  if (reinterpret_cast<uintptr_t>(d->positions) % 4) return fail(TL_ERR_INVALID, w + "positions not aligned");
  if (!d->positions && d->T && d->first_position > UINT32_MAX - (d->T - 1))
    return fail(TL_ERR_RANGE, w + "positions behind 2^32 - 1");
  if (!d->q.heads && !d->k.heads) return fail(TL_ERR_INVALID, w + "no heads");
  a.D = d->D;
  a.T = d->T;
  a.tokens = static_cast<uint32_t>(tokens);
  a.rotary = d->rotary_dim;
  a.interleaved = d->layout == TL_ROTARY_INTERLEAVED;
  a.norm = d->norm;
  a.eps = d->eps;
  a.inv_d = 1.0f / d->D;
  a.magnitude = d->magnitude;
  a.frequencies = d->frequencies;
  a.positions = d->positions;
  a.first_position = d->first_position;
  const uint32_t V = vector_for(d->type, d->out_type);
  bool aligned = true;
  const tl_rotary_part *parts[2] = {&d->q, &d->k};
  for (int i = 0; i < 2 && tokens; ++i) {
    const tl_rotary_part &p = *parts[i];
    RotaryPart &r = a.part[i];
    r.heads = p.heads;
    if (!p.heads) continue;
    if ((reinterpret_cast<uintptr_t>(p.weight) | reinterpret_cast<uintptr_t>(p.dweight)) % 4)
      return fail(TL_ERR_INVALID, w + "weight or dweight not aligned");
    const auto view = [&](const char *name, const tl_head_view &v, int32_t type, bool written) {
      aligned = aligned && aligned_view(v, type, d->B > 1, V);
      return check_view(who, name, v, type, d->B, d->T, p.heads, d->D, written);
    };
    if (!backward || d->norm)
      if (int rc = view("x", p.x, d->type, false)) return rc;
    if (!backward) {
      if (int rc = view("out", p.out, d->out_type, true)) return rc;
    } else {
      if (int rc = view("d_out", p.d_out, d->out_type, false)) return rc;
      if (int rc = view("dx", p.dx, d->type, true)) return rc;
      if (p.dweight && !d->norm) return fail(TL_ERR_INVALID, w + "dweight without a norm");
    }
    if (!backward && half_in_place(p.out, d->out_type, p.x, d->type, d->B > 1))
      return fail(TL_ERR_INVALID, w + "out is x with another layout or type");
    if (backward && (half_in_place(p.dx, d->type, p.d_out, d->out_type, d->B > 1) ||
                     (d->norm && half_in_place(p.dx, d->type, p.x, d->type, d->B > 1))))
      return fail(TL_ERR_INVALID, w + "dx in place with another layout or type");
    r.x = p.x;
    r.out = p.out;
    r.d_out = p.d_out;
    r.dx = p.dx;
    r.weight = p.weight;
    r.dweight = backward ? p.dweight : nullptr;
  }
  if (a.part[0].dweight && a.part[1].dweight) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.part[0].dweight), y = reinterpret_cast<uintptr_t>(a.part[1].dweight);
    if ((x < y ? y - x : x - y) < d->D * sizeof(float)) return fail(TL_ERR_INVALID, w + "q and k share a dweight, which each sets");
  }
  const Shape shape = shape_for(d->D, d->rotary_dim, V, aligned);
  a.lanes = shape.lanes;
  a.vectors = shape.vectors;
  return TL_OK;
}

unsigned share_out(RotaryArgs &a, uint32_t rows, uint32_t most, bool apart) {
  // A warp's run of a token's heads: all of them where the tokens alone keep two warps a
  // scheduler busy, shorter where they do not.
  const uint32_t per = 32 / a.lanes * rows, wanted = kNumSMs * 8;
  uint64_t groups = 0;
  for (RotaryPart &p : a.part) {
    p.chunks = p.ctas = 0;
    if (!p.heads) continue;
    const uint32_t batches = (p.heads + per - 1) / per;
    uint32_t run = batches;
    while (run > 1 && static_cast<uint64_t>(a.tokens) * ((batches + run - 1) / run) < wanted) run = (run + 1) / 2;
    p.run = run * per;
    p.chunks = (batches + run - 1) / run;
    groups += static_cast<uint64_t>(a.tokens) * p.chunks;
  }
  const auto fewest = [](uint64_t x, uint64_t y) { return static_cast<uint32_t>(x < y ? x : y); };
  a.whole = !apart && a.part[0].chunks <= 1 && a.part[1].chunks <= 1;
  if (a.whole) groups = a.tokens;
  if (!apart) return fewest((groups + kWarps - 1) / kWarps, most);
  const uint64_t heads = a.part[0].heads + static_cast<uint64_t>(a.part[1].heads);
  uint32_t left = most;
  for (RotaryPart &p : a.part) {
    if (!p.heads) continue;
    const bool last = &p == &a.part[1] || !a.part[1].heads;
    uint64_t share = last ? left : most * static_cast<uint64_t>(p.heads) / heads;
    share = share < 1 ? 1 : share > most - 1 ? most - 1 : share;
    p.ctas = fewest((static_cast<uint64_t>(a.tokens) * p.chunks + kWarps - 1) / kWarps, share);
    left -= p.ctas;
  }
  return a.part[0].ctas + a.part[1].ctas;
}

}  // namespace heads
}  // namespace tl

using namespace tl;
using namespace tl::heads;

extern "C" {

int tl_rotary_frequencies(const tl_rotary_spec *spec, uint64_t *frequencies, float *magnitude) {
  const std::string w = "tl_rotary_frequencies: ";
  if (!spec || !frequencies) return fail(TL_ERR_INVALID, w + "null argument");
  const tl_rotary_spec &s = *spec;
  if (s.dim < 2 || s.dim % 2 || s.dim > TL_HEAD_MAX_DIM) return fail(TL_ERR_RANGE, w + "dim is even, 2 to 256");
  if (s.scaling < TL_ROTARY_PLAIN || s.scaling > TL_ROTARY_SMOOTH) return fail(TL_ERR_INVALID, w + "unknown scaling");
  if (!(s.base > 1.0) || !std::isfinite(s.base)) return fail(TL_ERR_INVALID, w + "base is above 1");
  if (s.scaling != TL_ROTARY_PLAIN && (!(s.factor >= 1.0) || !std::isfinite(s.factor)))
    return fail(TL_ERR_INVALID, w + "factor is at least 1");
  const bool split = s.scaling == TL_ROTARY_PARTS || s.scaling == TL_ROTARY_SMOOTH;
  if (split && (!(s.original_length > 0.0) || !std::isfinite(s.original_length) || !(s.low > 0.0) ||
                !(s.high > s.low) || !std::isfinite(s.high)))
    return fail(TL_ERR_INVALID, w + "original_length and 0 < low < high are needed");
  if (s.scaling == TL_ROTARY_NTK && s.dim == 2 && s.factor != 1.0)
    return fail(TL_ERR_INVALID, w + "the base cannot stretch a single pair");

  const double two_pi = 6.283185307179586;
  const uint32_t n = s.dim / 2;
  double base = s.base;
  if (s.scaling == TL_ROTARY_NTK && s.dim > 2) base *= std::pow(s.factor, s.dim / (s.dim - 2.0));
  double from = 0, to = 0;
  if (s.scaling == TL_ROTARY_PARTS) {
    // the pair that turns `r` times over original_length
    const auto pair = [&](double r) {
      return s.dim * std::log(s.original_length / (r * two_pi)) / (2 * std::log(base));
    };
    from = std::fmax(std::floor(pair(s.high)), 0.0);
    to = std::fmin(std::ceil(pair(s.low)), s.dim - 1.0);
    if (to - from < 0.001) to = from + 0.001;
  }
  for (uint32_t i = 0; i < n; ++i) {
    double f = std::pow(base, -2.0 * i / s.dim), stretched = f / s.factor;
    if (s.scaling == TL_ROTARY_LINEAR) f = stretched;
    if (split) {
      const double ramp = s.scaling == TL_ROTARY_PARTS
                                   ? (i - from) / (to - from)
                                   : 1 - (s.original_length * f / two_pi - s.low) / (s.high - s.low);
      const double part = std::fmin(std::fmax(ramp, 0.0), 1.0);
      f = f * (1 - part) + stretched * part;
    }
    frequencies[i] = static_cast<uint64_t>(std::round(f / two_pi * 18446744073709551616.0));
  }
  if (magnitude) *magnitude = s.scaling == TL_ROTARY_PARTS ? static_cast<float>(0.1 * std::log(s.factor) + 1.0) : 1.0f;
  return TL_OK;
}

int tl_rotary_heads(const tl_rotary_desc *desc, void *stream) {
  const char *who = "tl_rotary_heads";
  RotaryArgs a{};
  if (int rc = rotary_args(who, desc, false, a)) return rc;
  if (a.tokens == 0) return TL_OK;
#define L(TI, TO) launch_rotate<TI, TO>(a, as_stream(stream))
  TL_BY_TYPES(desc->type, desc->out_type, L)
#undef L
  return launch_status(who);
}

}  // extern "C"
