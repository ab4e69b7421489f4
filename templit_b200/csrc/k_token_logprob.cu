// Token scoring: log probability of given tokens, entropy and top
// alternatives of rows of logits, and their gradient
// (tl_token_logprob_rows, tl_token_logprob_backward_rows).
#include "token_score.cuh"

#include <cooperative_groups.h>

namespace tl {
namespace token {

static int bad(const char *who, const char *what) {
  return fail(TL_ERR_INVALID, std::string(who) + ": " + what);
}

int check_rows(const char *who, const void *logits, int32_t type, uint32_t rows, uint32_t vocab,
               float temperature, uint64_t &row_stride) {
  if (type != TL_FLOAT32 && type != TL_FLOAT16 && type != TL_BFLOAT16)
    return bad(who, "unknown logit type");
  if (vocab == 0) return bad(who, "logits need a non-empty final dimension");
  if (vocab > 1u << 31) return fail(TL_ERR_RANGE, std::string(who) + ": more than 2^31 tokens");
  if (!(temperature > 0.0f) || std::isinf(temperature))
    return bad(who, "temperature must be positive and finite");
  if (1.4426950408889634 / temperature > FLT_MAX)  // or every product with it is NaN
    return fail(TL_ERR_RANGE, std::string(who) + ": temperature's reciprocal is beyond fp32");
  if (rows == 0) return TL_OK;
  if (row_stride == 0) row_stride = vocab;
  if (row_stride < vocab && rows > 1) return bad(who, "row stride below the row's length");
  if (row_stride > static_cast<uint64_t>(LLONG_MAX) / 4 / rows)
    return fail(TL_ERR_RANGE, std::string(who) + ": rows reach beyond the address space");
  if (!logits) return bad(who, "null logits");
  if (reinterpret_cast<uintptr_t>(logits) % type_size(type))
    return bad(who, "logits not aligned to their type");
  return TL_OK;
}

int check_gradient(const char *who, const void *logits, uint64_t row_stride, void *dlogits,
                   int32_t type, uint32_t rows, uint32_t vocab, uint64_t &d_row_stride) {
  if (d_row_stride == 0) d_row_stride = vocab;
  if (d_row_stride < vocab && rows > 1) return bad(who, "gradient row stride below the row's length");
  if (d_row_stride > static_cast<uint64_t>(LLONG_MAX) / 4 / rows)
    return fail(TL_ERR_RANGE, std::string(who) + ": gradient rows reach beyond the address space");
  if (!dlogits) return bad(who, "null dlogits");
  if (reinterpret_cast<uintptr_t>(dlogits) % type_size(type))
    return bad(who, "dlogits not aligned to their type");
  if (dlogits == logits && rows > 1 && d_row_stride != row_stride)
    return bad(who, "a gradient in place of the logits needs their row stride");
  return TL_OK;
}

dim3 gradient_grid(uint32_t rows, uint32_t vecs) {
  uint32_t parts = 1;
  while (static_cast<uint64_t>(rows) * parts < 16 * kNumSMs && vecs / parts > 8 * 256) ++parts;
  return dim3(rows < kNumSMs * 64u ? rows : kNumSMs * 64u, parts);
}

uint32_t cluster_parts(uint32_t rows, uint32_t vecs) {
  uint32_t parts = 1;
  while (parts < kMaxCluster && static_cast<uint64_t>(rows) * parts <= kNumSMs / 2 && vecs / parts > 4 * 256)
    parts *= 2;
  return parts;
}

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;          // vectors of a thread in flight
constexpr uint32_t kSegments = 16; // most segments that have their own maximum
constexpr uint32_t kList = 512;    // candidates, and vectors and segments that hold some

struct ScoreShared {
  Sums scratch[kWarps];
  Pow2Sums sums[kMaxCluster * kWarps];
  float largest[kMaxCluster * kWarps];
  float group[kThreads];  // maxima of the row's 256 groups of threads
  uint32_t entries, hits, candidates, least, count[kWarps];
  uint32_t entry[kList];  // segments with candidates
  uint32_t at[kList];     // vectors with candidates: where they are
  uint4 hit[kList];       // and what they hold
  alignas(16) uint64_t candidate[kList];
};

// The sums of a row by add_logit, for rows that Pow2Sums cannot hold.
template <typename T>
__device__ __noinline__ Sums careful_sums(const T *z, uint32_t vocab, float c, Sums *scratch) {
  Sums v = empty_sums();
  for (uint32_t j = threadIdx.x; j < vocab; j += kThreads) add_logit(v, to_float(z[j]), c);
  return block_merge<kWarps>(v, c, scratch);
}

// The `top` largest (logit, lowest id) of a row whatever the data: bisects
// the order of the logits for the top-th largest value v (32 counts of the
// row at most; rows of many equals end at the first), takes the logits
// above v and the first ids at v.  For rows where a threshold leaves too
// many candidates (long runs of equal logits, masks that leave fewer tokens
// than alternatives, NaN).
template <typename T>
__device__ __noinline__ void careful_top(const T *z, uint32_t vocab, uint32_t top, uint32_t least,
                                         ScoreShared &sh) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const auto count_from = [&](uint32_t from) {
    uint32_t n = 0;
    for (uint32_t j = threadIdx.x; j < vocab; j += kThreads) n += order_of(to_float(z[j])) >= from;
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if (lane == 0) sh.count[warp] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < kWarps; ++w) n += sh.count[w];
    return n;
  };
  // count_from(lo) >= top > count_from(hi)
  uint32_t lo = count_from(least) >= top ? least : 0u, hi = 0xffffffffu;
  if (count_from(lo + 1) < top) hi = lo + 1;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (count_from(mid) >= top) lo = mid;
    else hi = mid;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.candidates = 0;
  __syncthreads();
  for (uint32_t j = threadIdx.x; j < vocab; j += kThreads) {
    const float x = to_float(z[j]);
    if (order_of(x) > lo) sh.candidate[atomicAdd(&sh.candidates, 1u)] = key_of(x, j);
  }
  __syncthreads();
  uint32_t have = sh.candidates;
  for (uint32_t at = 0; have < top; at += kThreads) {
    const uint32_t j = at + threadIdx.x;
    const float x = j < vocab ? to_float(z[j]) : 0.0f;
    const bool equal = j < vocab && order_of(x) == lo;
    const uint32_t mask = __ballot_sync(0xffffffffu, equal);
    __syncthreads();
    if (lane == 0) sh.count[warp] = __popc(mask);
    __syncthreads();
    uint32_t before = have + __popc(mask & ((1u << lane) - 1));
    for (uint32_t w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.count[w];
      have += sh.count[w];
    }
    if (equal && before < top) sh.candidate[before] = key_of(x, j);
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.candidates = top;
  __syncthreads();
}

// One CTA per row, or a cluster of CTAs that share a row.  One pass over the
// row: every thread keeps its sums in powers of two and the largest logit of
// each segment of its vectors.  Alternatives: the top-th largest of the
// maxima of 256 groups of threads is a logit that at least `top` reach, so
// the alternatives are among the logits from there on, and only segments
// whose maximum reaches it are looked at again; their ranks among one
// another order the few candidates.  The registers hold four vectors of a
// thread and five CTAs share an SM: while one joins and ranks, the others
// read.  4096 x 128000 bf16: 208 us with 20 alternatives (5.0 TB/s; at full
// clock, for a few calls, 188, and 174 without the alternatives), bound by
// the instructions of a logit (issue slots 66 %, exponentials 70 %, memory
// 69 % busy).  A copy through a ring in shared memory, running ahead over the
// rows' ends, took 1.2 instructions a logit more and 243 us.  A short call
// waits for its steps one after the other: 3.3 us for 2048 logits, 8.5 for 64
// x 50001.
template <typename T, bool ENTROPY, bool TOP, bool CLUSTER, bool ONCE>
__global__ void __launch_bounds__(kThreads, CLUSTER || ONCE ? 3 : 5) score_kernel(const ScoreArgs a) {
  extern __shared__ float segment[];  // [segments][kThreads] maxima (TOP)
  __shared__ ScoreShared sh;
  constexpr uint32_t E = Vec<T>::kElems;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts = CLUSTER ? cluster.num_blocks() : 1, part = CLUSTER ? cluster.block_rank() : 0;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const auto everyone = [&] {
    if (CLUSTER) cluster.sync();
    else __syncthreads();
  };
  if (CLUSTER) cluster.barrier_arrive();  // this CTA runs: its memory may be written to
  pdl_enter();
  for (size_t row = blockIdx.x / parts; row < a.rows; row += gridDim.x / parts) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, part, parts);
    if (TOP && tid == 0) sh.entries = sh.hits = sh.candidates = 0;
    uint32_t t = TL_NO_TOKEN;
    float zt = 0.0f;
    if (tid == 32 && part == 0 && a.targets) {
      t = a.targets[row];
      if (t < a.vocab) zt = to_float(z[t]);
    }
    const uint4 *vec = reinterpret_cast<const uint4 *>(z + p.head);
    Pow2Sums v = {-kFar, 0.0f, 0.0f};
    float largest = -INFINITY, in_segment = -INFINITY;
    uint32_t batch = 0;
    bool masked = false;
    uint4 q[kBatch];
    const auto add = [&](auto full, uint32_t at) {  // full: no vector of the batch is past the end
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t i = at + u * kThreads + tid;
        q[u] = full || i < p.end ? vec[i] : make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
      }
      float most = Vec<T>::largest(q[0]);
#pragma unroll
      for (int u = 1; u < kBatch; ++u) most = fmaxf(most, Vec<T>::largest(q[u]));
      largest = fmaxf(largest, most);
      if (TOP && !ONCE) {
        in_segment = batch & ((1u << a.segment_shift) - 1) ? fmaxf(in_segment, most) : most;
        segment[(batch >> a.segment_shift) * kThreads + tid] = in_segment;
      }
      move_to<ENTROPY>(v, fmaxf(v.n, shift_of(most, a.c)));
      add_batch<ENTROPY, T>(v, q, a.c, masked);
    };
    if (ONCE) {
      add(std::false_type{}, p.begin);
    } else {
      // whole batches by themselves: 177 -> 174 us on 4096 x 128000 bf16, but
      // 188 -> 191 with alternatives, whose code has no register to spare
      uint32_t at = p.begin;
      if constexpr (TOP) {
        for (; at < p.end; at += kThreads * kBatch, ++batch) add(std::false_type{}, at);
      } else {
        for (; at + kThreads * kBatch <= p.end; at += kThreads * kBatch) add(std::true_type{}, at);
        if (at < p.end) add(std::false_type{}, at);
      }
    }
    float loose = -INFINITY;
    if (tid < p.loose) {
      loose = to_float(z[loose_at(p, tid)]);
      largest = fmaxf(largest, loose);
      move_to<ENTROPY>(v, fmaxf(v.n, shift_of(loose, a.c)));
      add_term<ENTROPY>(v, loose, a.c);
    }
    // join the row's sums in every CTA of it
    if (CLUSTER && row == blockIdx.x / parts) cluster.barrier_wait();
    warp_join<ENTROPY>(v);
    const float warp_largest = warp_max(largest);
    float group = largest;
    if (TOP && CLUSTER)
      for (uint32_t o = 1; o < parts; o <<= 1) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, o));
    for (uint32_t c = 0; c < parts; ++c) {
      ScoreShared *to = CLUSTER ? cluster.map_shared_rank(&sh, c) : &sh;
      if (lane == 0) {
        to->sums[part * kWarps + warp] = v;
        to->largest[part * kWarps + warp] = warp_largest;
      }
      if (TOP && tid % parts == 0) to->group[(part * kThreads + tid) / parts] = group;
    }
    everyone();
    v = {-kFar, 0.0f, 0.0f};
    RowSums r;
    r.m = -INFINITY;
    for (uint32_t i = lane; i < parts * kWarps; i += 32) {
      Pow2Sums w = sh.sums[i];
      const float n = fmaxf(v.n, w.n);
      move_to<ENTROPY>(v, n);
      move_to<ENTROPY>(w, n);
      v.s += w.s;
      v.h += w.h;
      r.m = fmaxf(r.m, sh.largest[i]);
    }
    warp_join<ENTROPY>(v);
    r.m = warp_max(r.m);
    r.s = sum_at(v.s, v.n, r.m, a.c);
    r.log_s = logf(r.s);
    if (ENTROPY)
      r.entropy = v.s == 0.0f ? 0.0f : (log2f(v.s) - v.h / v.s) * 0.6931471805599453f;
    if (far_out(r.m, a.c)) {
      const Sums w = careful_sums(z, a.vocab, a.c, sh.scratch);
      r.s = w.s;
      r.log_s = logf(r.s);
      r.entropy = r.log_s - w.h * a.inv_t / w.s;
    }
    if (tid == 32 && part == 0) {
      if (a.targets) {
        a.logprob[row] = t < a.vocab ? log_q(zt, r, a.inv_t) : 0.0f;
        if (t >= a.vocab && t != TL_NO_TOKEN) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
      }
      if (ENTROPY) a.entropy[row] = r.entropy;
      if (a.stats) {
        a.stats[2 * row] = r.m;
        a.stats[2 * row + 1] = r.s;
      }
    }
    if (TOP) {
      if (warp == 0) {
        // a value that `top` to a few more of the 256 maxima reach, bisected
        // between the least and the largest of them (with no more than a
        // value a lane asked for, between the lanes' largest)
        uint32_t key[kThreads / 32], lo = 0xffffffffu, hi = 0;
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) {
          key[i] = order_of_number(sh.group[i * 32 + lane]);
          lo = min(lo, key[i]);
          hi = max(hi, key[i]);
        }
        lo = __reduce_min_sync(0xffffffffu, a.top <= 32 ? hi : lo);
        hi = __reduce_max_sync(0xffffffffu, hi) + 1;
        while (hi - lo > 1) {
          const uint32_t mid = lo + (hi - lo) / 2;
          uint32_t n = 0;
#pragma unroll
          for (int i = 0; i < kThreads / 32; ++i) count_ge(n, key[i], mid);
          n = __reduce_add_sync(0xffffffffu, n);
          if (n >= a.top) lo = mid;
          else hi = mid;
          if (n >= a.top && n <= a.top + a.top / 8 + 1) break;
        }
        if (lane == 0) sh.least = lo;
      }
      __syncthreads();
      const uint32_t least = sh.least;
      const float from = logit_of(static_cast<uint64_t>(least) << 32);
      ScoreShared *first = CLUSTER ? cluster.map_shared_rank(&sh, 0) : &sh;
      const auto candidate = [&](float x, uint32_t id) {
        const uint32_t i = atomicAdd(&first->candidates, 1u);
        if (i < kList) first->candidate[i] = key_of(x, id);
      };
      // vectors with candidates go to shared memory: code for one logit does
      // for all (unrolled, it is the instruction cache that a short call
      // waits for)
      const auto keep = [&](const uint4 &r4, uint32_t at) {
        const uint32_t i = atomicAdd(&sh.hits, 1u);
        if (i < kList) sh.hit[i] = r4, sh.at[i] = p.head + at * E;
      };
      if constexpr (ONCE) {
        if (largest >= from) {
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const uint32_t i = p.begin + u * kThreads + tid;
            if (i < p.end && Vec<T>::largest(q[u]) >= from) keep(q[u], i);
          }
        }
      } else {
        if (largest >= from) {
          const uint32_t segments = (batch + (1u << a.segment_shift) - 1) >> a.segment_shift;
          for (uint32_t s = 0; s < segments; ++s)
            if (segment[s * kThreads + tid] >= from) {
              const uint32_t i = atomicAdd(&sh.entries, 1u);
              if (i < kList) sh.entry[i] = s * kThreads + tid;
            }
        }
        __syncthreads();
        const uint32_t entries = min(sh.entries, kList);
        const uint32_t each = kBatch << a.segment_shift;  // vectors of a segment
        for (uint32_t i = tid; i < entries * each; i += kThreads) {
          const uint32_t en = sh.entry[i / each];
          const uint32_t at = p.begin + (en / kThreads * each + i % each) * kThreads + en % kThreads;
          if (at >= p.end) continue;
          const uint4 r4 = vec[at];
          if (Vec<T>::largest(r4) >= from) keep(r4, at);
        }
      }
      __syncthreads();
      const uint32_t hits = sh.hits;
      const bool over = hits > kList || (!ONCE && sh.entries > kList);
      const uint32_t logits_in = over ? 0 : hits * E;
      for (uint32_t i = tid; i < logits_in + p.loose; i += kThreads) {
        const uint32_t j = i - logits_in;
        const float x = i < logits_in ? to_float(reinterpret_cast<const T *>(sh.hit)[i]) : to_float(z[loose_at(p, j)]);
        if (x >= from) candidate(x, i < logits_in ? sh.at[i / E] + i % E : loose_at(p, j));
      }
      if (over && tid == 0) atomicAdd(&first->candidates, kList + 1);
      everyone();
      if (part == 0) {
        if (sh.candidates > kList || sh.candidates < a.top) careful_top(z, a.vocab, a.top, least, sh);
        const uint32_t n = sh.candidates;
        for (uint32_t i = tid; i < n; i += kThreads) {
          const uint64_t key = sh.candidate[i];
          uint32_t rank = 0;
#pragma unroll 8
          for (uint32_t j = 0; j < n; ++j) rank += sh.candidate[j] > key;
          if (rank < a.top) {
            a.top_ids[row * a.top + rank] = ~static_cast<uint32_t>(key);
            a.top_logprob[row * a.top + rank] = log_q(logit_of(key), r, a.inv_t);
          }
        }
      }
    }
    if (row + gridDim.x / parts < a.rows) everyone();  // shared memory is free for the next row
  }
}

// The gradient of part of a row.  The target's element is written again at
// the end by the part that holds it.  Bound by memory: 4096 x 50001 bf16, one
// row in eight aligned, 138 us (5.9 TB/s of reads and writes).
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads) score_backward_kernel(const ScoreArgs a) {
  const uint32_t tid = threadIdx.x, parts = gridDim.y, part = blockIdx.y;
  pdl_enter();
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
    const float m = a.stats[2 * row], s = a.stats[2 * row + 1];
    uint32_t t = TL_NO_TOKEN;
    float gl = 0.0f, ge = 0.0f, entropy = 0.0f;
    if (a.d_logprob) {
      t = a.targets[row];
      if (t < a.vocab) {
        gl = a.d_logprob[row] * a.inv_t;
      } else {
        if (t != TL_NO_TOKEN && tid == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
        t = TL_NO_TOKEN;
      }
    }
    if (ENTROPY) {
      ge = a.d_entropy[row] * a.inv_t;
      if (ge != 0.0f) entropy = a.entropy[row];
    }
    const Part p = part_of(z, a.vocab, part, parts);
    const ScoreGradient g = score_gradient(a, m, s, entropy, gl, ge);
    const auto fast = [&](float x) { return score_dz<ENTROPY>(g, a.c, x); };
    const Pair c2 = pair(a.c, a.c);
    const auto fast2 = [&](Pair x) { return score_dz2<ENTROPY>(g, c2, x); };
    const auto careful = [&](float x) { return careful_score_dz(g, a, x); };
    float zt = 0.0f;
    const bool mine = tid == 0 && t != TL_NO_TOKEN && !g.none && holds<T>(p, t);
    if (mine) zt = to_float(z[t]);
    __syncthreads();  // dz may be z
    if (g.none) write_elements<kThreads>(z, dz, p, [](float) { return 0.0f; });
    else if (g.far) write_elements<kThreads>(z, dz, p, careful);
    else write_vectors<kThreads, kBatch, false, false>(z, dz, p, fast2, fast);
    __syncthreads();
    if (mine) dz[t] = from_float<T>((g.far ? careful(zt) : fast(zt)) + gl);
  }
}

template <typename T, bool ENTROPY, bool TOP, bool CLUSTER>
void launch_score_team(ScoreArgs &a, uint32_t parts, cudaStream_t s) {
  const uint32_t vecs = a.vocab / Vec<T>::kElems, most = kNumSMs * 64u;
  const uint32_t batches = ((vecs + parts - 1) / parts + kThreads * kBatch - 1) / (kThreads * kBatch);
  size_t smem = 0;
  if (TOP && batches > 1) {
    a.segment_shift = 0;
    while ((batches + (1u << a.segment_shift) - 1) >> a.segment_shift > kSegments) ++a.segment_shift;
    smem = ((batches + (1u << a.segment_shift) - 1) >> a.segment_shift) * kThreads * sizeof(float);
  }
  const auto kernel = TOP && batches <= 1 ? score_kernel<T, ENTROPY, TOP, CLUSTER, TOP>
                                          : score_kernel<T, ENTROPY, TOP, CLUSTER, false>;
  const unsigned grid = (a.rows < most ? a.rows : most) * parts;
  if (CLUSTER) launch_pdl_cluster(kernel, grid, kThreads, smem, s, parts, a);
  else launch_pdl(kernel, grid, kThreads, smem, s, a);
}

template <typename T, bool ENTROPY, bool TOP>
void launch_score_form(ScoreArgs &a, cudaStream_t s) {
  const uint32_t parts = cluster_parts(a.rows, a.vocab / Vec<T>::kElems);
  if (parts > 1) launch_score_team<T, ENTROPY, TOP, true>(a, parts, s);
  else launch_score_team<T, ENTROPY, TOP, false>(a, 1, s);
}

template <typename T> void launch_score(ScoreArgs &a, cudaStream_t s) {
  if (a.entropy) a.top ? launch_score_form<T, true, true>(a, s) : launch_score_form<T, true, false>(a, s);
  else a.top ? launch_score_form<T, false, true>(a, s) : launch_score_form<T, false, false>(a, s);
}

template <typename T> void launch_score_backward(const ScoreArgs &a, cudaStream_t s) {
  const dim3 grid = gradient_grid(a.rows, a.vocab / Vec<T>::kElems);
  if (a.d_entropy) launch_pdl(score_backward_kernel<T, true>, grid, kThreads, 0, s, a);
  else launch_pdl(score_backward_kernel<T, false>, grid, kThreads, 0, s, a);
}

int score_args(const char *who, const tl_token_logprob_desc *d, ScoreArgs &a) {
  if (!d) return bad(who, "null descriptor");
  a.row_stride = d->row_stride;
  if (int rc = check_rows(who, d->logits, d->type, d->rows, d->vocab, d->temperature, a.row_stride))
    return rc;
  a.logits = d->logits;
  a.rows = d->rows;
  a.vocab = d->vocab;
  a.top = d->top;
  a.c = static_cast<float>(1.4426950408889634 / d->temperature);
  a.inv_t = static_cast<float>(1.0 / d->temperature);
  a.targets = d->targets;
  a.logprob = d->logprob;
  a.entropy = d->entropy;
  a.stats = d->stats;
  a.top_logprob = d->top_logprob;
  a.top_ids = d->top_ids;
  a.d_logprob = d->d_logprob;
  a.d_entropy = d->d_entropy;
  a.dlogits = d->dlogits;
  a.d_row_stride = d->d_row_stride;
  return TL_OK;
}

}  // namespace
}  // namespace token
}  // namespace tl

using namespace tl;
using namespace tl::token;

extern "C" {

int tl_token_logprob_rows(const tl_token_logprob_desc *desc, void *stream) {
  const char *who = "tl_token_logprob_rows";
  ScoreArgs a{};
  if (int rc = score_args(who, desc, a)) return rc;
  if (a.top > TL_TOKEN_MAX_TOP) return fail(TL_ERR_RANGE, std::string(who) + ": more than 128 alternatives");
  if (a.top > a.vocab) return bad(who, "more alternatives than tokens");
  if (a.rows == 0) return TL_OK;
  if (!a.targets != !a.logprob) return bad(who, "targets and logprob go together");
  if (a.top && (!a.top_logprob || !a.top_ids)) return bad(who, "null top_logprob or top_ids");
  if (!a.logprob && !a.entropy && !a.stats && !a.top) return bad(who, "no output");
  a.status = device_status_ptr();
  if (!a.status) return fail(TL_ERR_CUDA, std::string(who) + ": no status word");
  if (score_short(a, desc->type, as_stream(stream))) return launch_status(who);
#define L(T) launch_score<T>(a, as_stream(stream))
  TL_BY_TYPE(desc->type, L)
#undef L
  return launch_status(who);
}

int tl_token_logprob_backward_rows(const tl_token_logprob_desc *desc, void *stream) {
  const char *who = "tl_token_logprob_backward_rows";
  ScoreArgs a{};
  if (int rc = score_args(who, desc, a)) return rc;
  if (a.rows == 0) return TL_OK;
  if (int rc = check_gradient(who, a.logits, a.row_stride, a.dlogits, desc->type, a.rows, a.vocab,
                              a.d_row_stride))
    return rc;
  if (!a.stats) return bad(who, "null stats");
  if (!a.d_logprob && !a.d_entropy) return bad(who, "no incoming gradient");
  if (a.d_logprob && !a.targets) return bad(who, "d_logprob without targets");
  if (a.d_entropy && !a.entropy) return bad(who, "d_entropy without entropy");
  a.status = device_status_ptr();
  if (!a.status) return fail(TL_ERR_CUDA, std::string(who) + ": no status word");
  if (score_backward_short(a, desc->type, as_stream(stream))) return launch_status(who);
#define L(T) launch_score_backward<T>(a, as_stream(stream))
  TL_BY_TYPE(desc->type, L)
#undef L
  return launch_status(who);
}

}  // extern "C"
