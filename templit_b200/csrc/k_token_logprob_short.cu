// Token scoring of many short rows: a warp per row, the row in registers.
#include "token_score.cuh"

namespace tl {
namespace token {
namespace {

constexpr uint32_t kHits = 192;        // vectors that hold candidates
constexpr uint32_t kCandidates = 256;

struct WarpList {
  uint4 hit[kHits];
  uint32_t at[kHits];
  uint64_t candidate[kCandidates];
};

// The value that `top` or a few more of the warp's keys (N a lane) reach:
// bisected from -inf.
template <int N>
__device__ __forceinline__ uint32_t threshold(const uint32_t (&key)[N], uint32_t top) {
  uint32_t hi = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) hi = max(hi, key[i]);
  uint32_t lo = order_of(-INFINITY);
  hi = __reduce_max_sync(0xffffffffu, hi) + 1;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += key[i] >= mid;
    n = __reduce_add_sync(0xffffffffu, n);
    if (n >= top) lo = mid;
    else hi = mid;
    if (n >= top && n <= top + top / 8) break;
  }
  return lo;
}

// The alternatives of a row whatever the data: see careful_top in
// k_token_logprob.cu.
template <typename T>
__device__ __noinline__ void careful_warp_top(const T *z, uint32_t vocab, uint32_t top, uint32_t least,
                                              uint64_t *candidate) {
  const uint32_t lane = threadIdx.x & 31;
  const auto count_from = [&](uint32_t from) {
    uint32_t n = 0;
    for (uint32_t j = lane; j < vocab; j += 32) n += order_of(to_float(z[j])) >= from;
    return __reduce_add_sync(0xffffffffu, n);
  };
  uint32_t lo = count_from(least) >= top ? least : 0u, hi = 0xffffffffu;
  if (count_from(lo + 1) < top) hi = lo + 1;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (count_from(mid) >= top) lo = mid;
    else hi = mid;
  }
  // those above lo first, then the first ids at lo
  uint32_t have = 0;
  for (int equal = 0; equal < 2; ++equal)
    for (uint32_t at = 0; at < vocab && have < top; at += 32) {
      const uint32_t j = at + lane;
      const float x = j < vocab ? to_float(z[j]) : 0.0f;
      const bool take = j < vocab && (equal ? order_of(x) == lo : order_of(x) > lo);
      const uint32_t mask = __ballot_sync(0xffffffffu, take);
      const uint32_t i = have + __popc(mask & ((1u << lane) - 1));
      if (take && i < top) candidate[i] = key_of(x, j);
      have += __popc(mask);
    }
  __syncwarp();
}

// Alternatives: 128 groups of vectors (or every vector, for more than 64)
// give a threshold that at least `top` logits reach; the vectors that reach
// it go to shared memory, their candidates are ranked among one another.
template <typename T, int NV, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(kShortWarps * 32) score_short_kernel(const ScoreArgs a) {
  __shared__ WarpList lists[TOP ? kShortWarps : 1];
  constexpr int E = Vec<T>::kElems;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t before = (1u << lane) - 1;
  pdl_enter();
  for (size_t row = static_cast<size_t>(blockIdx.x) * kShortWarps + warp; row < a.rows;
       row += static_cast<size_t>(gridDim.x) * kShortWarps) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, 0, 1);
    uint4 r[NV];
    load_row<T, NV>(z, p, lane, r);
    const float loose = lane < p.loose ? to_float(z[loose_at(p, lane)]) : -INFINITY;
    uint32_t t = TL_NO_TOKEN;
    float zt = 0.0f;
    if (lane == 0 && a.targets) {
      t = a.targets[row];
      if (t < a.vocab) zt = to_float(z[t]);
    }
    float group[4] = {loose, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < NV; ++i) group[i * 4 / NV] = fmaxf(group[i * 4 / NV], Vec<T>::largest(r[i]));
    RowSums s;
    s.m = warp_max(fmaxf(fmaxf(group[0], group[1]), fmaxf(group[2], group[3])));
    Pow2Sums v = {shift_of(s.m, a.c), 0.0f, 0.0f};
    add_term<ENTROPY>(v, loose, a.c);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * 32 >= p.end) break;
      float f[E];
      Vec<T>::unpack(r[i], f);
#pragma unroll
      for (int e = 0; e < E; ++e) add_term<ENTROPY>(v, f[e], a.c);
    }
    v.s = warp_sum(v.s);
    if (ENTROPY) v.h = warp_sum(v.h);
    s.s = sum_at(v.s, v.n, s.m, a.c);
    s.log_s = logf(s.s);
    if (ENTROPY) s.entropy = v.s == 0.0f ? 0.0f : (log2f(v.s) - v.h / v.s) * 0.6931471805599453f;
    if (far_out(s.m, a.c)) {
      Sums w = empty_sums();
      for (uint32_t j = lane; j < a.vocab; j += 32) add_logit(w, to_float(z[j]), a.c);
      w = warp_merge(w, a.c);
      s.s = w.s;
      s.log_s = logf(s.s);
      s.entropy = s.log_s - w.h * a.inv_t / w.s;
    }
    if (lane == 0) {
      if (a.targets) {
        a.logprob[row] = t < a.vocab ? log_q(zt, s, a.inv_t) : 0.0f;
        if (t >= a.vocab && t != TL_NO_TOKEN) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
      }
      if (ENTROPY) a.entropy[row] = s.entropy;
      if (a.stats) {
        a.stats[2 * row] = s.m;
        a.stats[2 * row + 1] = s.s;
      }
    }
    if (!TOP) continue;
    WarpList &list = lists[warp];
    uint32_t least;
    if (NV > 4 && a.top > 64) {
      uint32_t key[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) key[i] = order_of(Vec<T>::largest(r[i]));
      least = threshold<NV>(key, a.top);
    } else {
      uint32_t key[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) key[i] = order_of(group[i]);
      least = threshold<4>(key, a.top);
    }
    const float from = logit_of(static_cast<uint64_t>(least) << 32);
    uint32_t hits = 0, candidates = 0;
    const auto candidate = [&](bool take, float x, uint32_t id) {
      const uint32_t mask = __ballot_sync(0xffffffffu, take);
      if (!mask) return;
      const uint32_t i = candidates + __popc(mask & before);
      if (take && i < kCandidates) list.candidate[i] = key_of(x, id);
      candidates += __popc(mask);
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i * 32 >= p.end) break;
      const bool hit = i * 32 + lane < p.end && Vec<T>::largest(r[i]) >= from;
      const uint32_t mask = __ballot_sync(0xffffffffu, hit);
      if (mask) {
        const uint32_t j = hits + __popc(mask & before);
        if (hit && j < kHits) {
          list.hit[j] = r[i];
          list.at[j] = p.head + (i * 32 + lane) * E;
        }
        hits += __popc(mask);
      }
    }
    __syncwarp();
    candidate(lane < p.loose && loose >= from, loose, loose_at(p, lane));
    if (hits <= kHits)
      for (uint32_t base = 0; base < hits; base += 32) {
        const bool some = base + lane < hits;
        const uint4 q = some ? list.hit[base + lane] : make_uint4(0, 0, 0, 0);
        const uint32_t at = some ? list.at[base + lane] : 0;
        float f[E];
        Vec<T>::unpack(q, f);
#pragma unroll
        for (int e = 0; e < E; ++e) candidate(some && f[e] >= from, f[e], at + e);
      }
    __syncwarp();
    if (hits > kHits || candidates > kCandidates || candidates < a.top) {
      careful_warp_top(z, a.vocab, a.top, least, list.candidate);
      candidates = a.top;
    }
    for (uint32_t i = lane; i < candidates; i += 32) {
      const uint64_t key = list.candidate[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < candidates; ++j) rank += list.candidate[j] > key;
      if (rank < a.top) {
        a.top_ids[row * a.top + rank] = ~static_cast<uint32_t>(key);
        a.top_logprob[row * a.top + rank] = log_q(logit_of(key), s, a.inv_t);
      }
    }
    __syncwarp();  // the list is free for the next row
  }
}

template <typename T, int NV, bool ENTROPY>
__global__ void __launch_bounds__(kShortWarps * 32) score_backward_short_kernel(const ScoreArgs a) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_enter();
  for (size_t row = static_cast<size_t>(blockIdx.x) * kShortWarps + warp; row < a.rows;
       row += static_cast<size_t>(gridDim.x) * kShortWarps) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
    const Part p = part_of(z, a.vocab, 0, 1);
    uint4 r[NV];
    load_row<T, NV>(z, p, lane, r);
    const float loose = lane < p.loose ? to_float(z[loose_at(p, lane)]) : 0.0f;
    const float m = a.stats[2 * row], s = a.stats[2 * row + 1];
    uint32_t t = TL_NO_TOKEN;
    float gl = 0.0f, zt = 0.0f;
    if (a.d_logprob) {
      t = a.targets[row];
      if (t < a.vocab) {
        gl = a.d_logprob[row] * a.inv_t;
        zt = to_float(z[t]);
      } else {
        if (t != TL_NO_TOKEN && lane == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
        t = TL_NO_TOKEN;
      }
    }
    const float ge = ENTROPY ? a.d_entropy[row] * a.inv_t : 0.0f;
    const float entropy = ENTROPY ? a.entropy[row] : 0.0f;
    const ScoreGradient g = score_gradient(a, m, s, ge == 0.0f ? 0.0f : entropy, gl, ge);
    const auto fast = [&](float x) { return score_dz<ENTROPY>(g, a.c, x); };
    const auto careful = [&](float x) { return careful_score_dz(g, a, x); };
    __syncwarp();  // the target's logit is read: dz may be z
    if (!g.none && !g.far) {
      store_row<T, NV>(dz, p, lane, r, loose, fast);
    } else {
      for (uint32_t j = lane; j < a.vocab; j += 32)
        dz[j] = from_float<T>(g.none ? 0.0f : careful(to_float(z[j])));
    }
    __syncwarp();
    if (lane == 0 && t != TL_NO_TOKEN && !g.none)
      dz[t] = from_float<T>((g.far ? careful(zt) : fast(zt)) + gl);
  }
}

template <typename T, int NV> void launch(const ScoreArgs &a, cudaStream_t s) {
  const unsigned grid = short_grid(a.rows);
  if (a.entropy) {
    if (a.top) launch_pdl(score_short_kernel<T, NV, true, true>, grid, kShortWarps * 32, 0, s, a);
    else launch_pdl(score_short_kernel<T, NV, true, false>, grid, kShortWarps * 32, 0, s, a);
  } else {
    if (a.top) launch_pdl(score_short_kernel<T, NV, false, true>, grid, kShortWarps * 32, 0, s, a);
    else launch_pdl(score_short_kernel<T, NV, false, false>, grid, kShortWarps * 32, 0, s, a);
  }
}

template <typename T, int NV> void launch_backward(const ScoreArgs &a, cudaStream_t s) {
  const unsigned grid = short_grid(a.rows);
  if (a.d_entropy) launch_pdl(score_backward_short_kernel<T, NV, true>, grid, kShortWarps * 32, 0, s, a);
  else launch_pdl(score_backward_short_kernel<T, NV, false>, grid, kShortWarps * 32, 0, s, a);
}

}  // namespace

bool score_short(const ScoreArgs &a, int32_t type, cudaStream_t s) {
  const uint32_t nv = short_vectors(a.vocab, type_size(type));
  if (!nv || a.rows < kShortRows) return false;
#define L(T) nv == 4 ? launch<T, 4>(a, s) : launch<T, 16>(a, s)
  TL_BY_TYPE(type, L)
#undef L
  return true;
}

bool score_backward_short(const ScoreArgs &a, int32_t type, cudaStream_t s) {
  const uint32_t nv = short_vectors(a.vocab, type_size(type));
  if (!nv || a.rows < kShortRows) return false;
#define L(T) nv == 4 ? launch_backward<T, 4>(a, s) : launch_backward<T, 16>(a, s)
  TL_BY_TYPE(type, L)
#undef L
  return true;
}

}  // namespace token
}  // namespace tl
