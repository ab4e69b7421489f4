// Token scoring of many short rows: a warp per row, the row in shared memory.
#include "token_score.cuh"

namespace tl {
namespace token {
namespace {

constexpr uint32_t kCandidates = 224;  // a multiple of 32
constexpr uint32_t kHits = 224;        // a multiple of 8

// A warp's shared memory: the row, and what picks the alternatives.
template <int NV, bool TOP> struct WarpShared {
  uint4 row[NV * 32];
};
template <int NV> struct WarpShared<NV, true> {
  uint4 row[NV * 32];
  uint32_t key[kCandidates], id[kCandidates];  // 16-byte aligned
  uint32_t hits, candidates;
  uint32_t unused[2];  // warps' parts stay 16-byte aligned
  uint16_t hit[kHits];  // vectors with candidates
};

// A candidate's key, larger for what ranks first.  Of 16-bit logits it holds
// the id too (rows here are shorter than 2^16): no two are equal.
template <typename T> __device__ __forceinline__ uint32_t list_key(float x, uint32_t id);
template <> __device__ __forceinline__ uint32_t list_key<float>(float x, uint32_t) { return order_of(x); }
template <> __device__ __forceinline__ uint32_t list_key<__nv_bfloat16>(float x, uint32_t id) {
  return (order_of(x) & 0xffff0000u) | (0xffffu - id);
}
template <> __device__ __forceinline__ uint32_t list_key<__half>(float x, uint32_t id) {
  // fp16's own 16 bits in order
  const uint32_t b = __half_as_ushort(__float2half_rn(x + 0.0f));
  const uint32_t o = x != x ? 0u : b & 0x8000u ? 0xffffu & ~b : b | 0x8000u;
  return o << 16 | (0xffffu - id);
}
// The logit of a key.
template <typename T> __device__ __forceinline__ float list_logit(uint32_t key) {
  const uint32_t o = key >> 16;
  const uint16_t b = static_cast<uint16_t>(o & 0x8000u ? o ^ 0x8000u : ~o);
  return to_float(*reinterpret_cast<const T *>(&b));
}
template <> __device__ __forceinline__ float list_logit<float>(uint32_t key) {
  return logit_of(static_cast<uint64_t>(key) << 32);
}

// A value that `top` or a few more of the warp's keys (N a lane) reach,
// bisected between their least and their largest: at least `top` keys.
template <int N>
__device__ __forceinline__ uint32_t threshold(const uint32_t (&key)[N], uint32_t top) {
  uint32_t lo = key[0], hi = key[0];
#pragma unroll
  for (int i = 1; i < N; ++i) lo = min(lo, key[i]), hi = max(hi, key[i]);
  // with no more than a key a lane asked for, the least of the lanes' largest
  lo = __reduce_min_sync(0xffffffffu, top <= 32 ? hi : lo);
  hi = __reduce_max_sync(0xffffffffu, hi) + 1;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count_ge(n, key[i], mid);
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
                                              uint32_t *key, uint32_t *id) {
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
  // by id: those above lo, and as many of those at lo as there is room for
  uint32_t have = 0, room = top - count_from(lo + 1);
  for (uint32_t at = 0; at < vocab && have < top; at += 32) {
    const uint32_t j = at + lane;
    const uint32_t o = j < vocab ? order_of(to_float(z[j])) : 0;
    const bool equal = j < vocab && o == lo;
    const uint32_t equals = __ballot_sync(0xffffffffu, equal);
    const bool take = (j < vocab && o > lo) || (equal && __popc(equals & ((1u << lane) - 1)) < room);
    const uint32_t mask = __ballot_sync(0xffffffffu, take);
    const uint32_t i = have + __popc(mask & ((1u << lane) - 1));
    if (take) key[i] = list_key<T>(to_float(z[j]), j), id[i] = j;
    have += __popc(mask);
    room -= min(room, static_cast<uint32_t>(__popc(equals)));
  }
  __syncwarp();
}

// Ranks and writes out a list of up to 32 R candidates; lane l has those at
// l + 32 i.  A candidate's rank is the number of keys above its own; equal
// keys (fp32 only) rank by id, looked at where the ranks' sum tells that
// there are some.
template <typename T, int R>
__device__ __forceinline__ void rank_candidates(const ScoreArgs &a, size_t row, const RowSums &s,
                                                const uint32_t *key, const uint32_t *id, uint32_t n,
                                                uint32_t lane) {
  uint32_t mine[R], rank[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mine[r] = lane + 32 * r < n ? key[lane + 32 * r] : 0xffffffffu;
    rank[r] = 0;
  }
  const uint4 *four = reinterpret_cast<const uint4 *>(key);
  for (uint32_t j = 0; j < n; j += 4) {  // the list is filled up with 0
    const uint4 k = four[j / 4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      count_gt(rank[r], k.x, mine[r]);
      count_gt(rank[r], k.y, mine[r]);
      count_gt(rank[r], k.z, mine[r]);
      count_gt(rank[r], k.w, mine[r]);
    }
  }
  if (sizeof(T) == 4) {
    uint32_t sum = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) sum += rank[r];
    if (__reduce_add_sync(0xffffffffu, sum) != n * (n - 1) / 2) {
      for (uint32_t j = 0; j < n; ++j) {
        const uint32_t k = key[j], i = id[j];
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (lane + 32 * r < n) rank[r] += k == mine[r] && i < id[lane + 32 * r];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane + 32 * r < n && rank[r] < a.top) {
      a.top_ids[row * a.top + rank[r]] = id[lane + 32 * r];
      a.top_logprob[row * a.top + rank[r]] = log_q(list_logit<T>(mine[r]), s, a.inv_t);
    }
}

// Sums of the row in shared memory; CLAMP: safe where a logit is -inf.
template <typename T, int NV, bool ENTROPY, bool CLAMP>
__device__ __forceinline__ void sum_row(const uint4 *row, uint32_t end, uint32_t lane, float c,
                                        Pow2Sums &v) {
  constexpr int E = Vec<T>::kElems;
  const Pair c2 = pair(c, c), n2 = pair(-v.n, -v.n);
  Pair s = pair(v.s, 0.0f), h = pair(v.h, 0.0f);
  for_vectors<NV>(end, lane, [&](int, uint32_t j) {
    Pair z[E / 2];
    Vec<T>::pairs(row[j], z);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      Pair x = fma2(z[e], c2, n2);
      if (CLAMP) {
        const float2 f = halves(x);
        x = pair(max_nan(f.x, -1e4f), max_nan(f.y, -1e4f));
      }
      const Pair p = ex2_pair(x);
      s = add2(s, p);
      if (ENTROPY) h = fma2(p, x, h);
    }
  });
  const float2 a = halves(s), b = halves(h);
  v.s = warp_sum(a.x + a.y);
  if (ENTROPY) v.h = warp_sum(b.x + b.y);
}

// Alternatives: 128 groups of vectors (or every vector, for more than 32)
// give a threshold that at least `top` logits reach; the candidates in the
// vectors that reach it are ranked among one another.  12288 x 2048 fp32: 19
// us without alternatives (memory: 5.3 TB/s), 25 with one, 33.6 with 32, where
// 21 warps an SM wait for their own steps (issue slots 51 % busy, memory 35):
// 1,300 instructions a row, 530 of them without alternatives.  In registers a
// row left room for 15 warps (47 us).
template <typename T, int NV, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(kScoreWarps * 32) score_short_kernel(const ScoreArgs a) {
  extern __shared__ uint4 shared[];
  constexpr int E = Vec<T>::kElems;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  WarpShared<NV, TOP> &w = reinterpret_cast<WarpShared<NV, TOP> *>(shared)[warp];
  const size_t stride = static_cast<size_t>(gridDim.x) * kScoreWarps;
  size_t row = static_cast<size_t>(blockIdx.x) * kScoreWarps + warp;
  pdl_enter();
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  Part p{};
  float loose = 0.0f;
  const auto begin_row = [&] {
    if (row >= a.rows) return;
    z = static_cast<const T *>(a.logits) + row * a.row_stride;
    p = part_of(z, a.vocab, 0, 1);
    stage_row<T, NV>(z, p, lane, w.row);
    loose = lane < p.loose ? to_float(z[loose_at(p, lane)]) : -INFINITY;
  };
  begin_row();
  while (row < a.rows) {
    const size_t r = row;
    uint32_t t = TL_NO_TOKEN;
    if (a.targets) t = a.targets[r];
    await_row();
    const float zt = lane == 0 && t < a.vocab ? to_float(z[t]) : 0.0f;
    float most[NV];  // of each vector
#pragma unroll
    for (int i = 0; i < NV; ++i) most[i] = -INFINITY;
    for_vectors<NV>(p.end, lane, [&](int i, uint32_t j) { most[i] = Vec<T>::largest(w.row[j]); });
    float group[4] = {loose, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < NV; ++i) group[i * 4 / NV] = fmaxf(group[i * 4 / NV], most[i]);
    RowSums s;
    s.m = warp_max(fmaxf(fmaxf(group[0], group[1]), fmaxf(group[2], group[3])));
    Pow2Sums v = {shift_of(s.m, a.c), 0.0f, 0.0f};
    add_term<ENTROPY>(v, loose, a.c);
    const Pow2Sums start = v;
    sum_row<T, NV, ENTROPY, false>(w.row, p.end, lane, a.c, v);
    if (ENTROPY && v.h != v.h) {  // 0 times a masked logit's x
      v = start;
      sum_row<T, NV, ENTROPY, true>(w.row, p.end, lane, a.c, v);
    }
    s.s = sum_at(v.s, v.n, s.m, a.c);
    s.log_s = logf(s.s);
    if (ENTROPY) s.entropy = v.s == 0.0f ? 0.0f : (log2f(v.s) - v.h / v.s) * 0.6931471805599453f;
    if (far_out(s.m, a.c)) {
      Sums y = empty_sums();
      for (uint32_t j = lane; j < a.vocab; j += 32) add_logit(y, to_float(z[j]), a.c);
      y = warp_merge(y, a.c);
      s.s = y.s;
      s.log_s = logf(s.s);
      s.entropy = s.log_s - y.h * a.inv_t / y.s;
    }
    if (lane == 0) {
      if (a.targets) {
        a.logprob[r] = t < a.vocab ? log_q(zt, s, a.inv_t) : 0.0f;
        if (t >= a.vocab && t != TL_NO_TOKEN) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
      }
      if (ENTROPY) a.entropy[r] = s.entropy;
      if (a.stats) {
        a.stats[2 * r] = s.m;
        a.stats[2 * r + 1] = s.s;
      }
    }
    if constexpr (TOP) {
      uint32_t least;
      if (NV > 4 && a.top > 32) {
        uint32_t key[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = order_of_number(most[i]);
        least = threshold<NV>(key, a.top);
      } else {
        uint32_t key[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) key[i] = order_of_number(group[i]);
        least = threshold<4>(key, a.top);
      }
      const float from = logit_of(static_cast<uint64_t>(least) << 32);
      // a bit for each of the lane's vectors that hold candidates
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        mark_from(hits, most[i], from, 1u << i);
      if (lane == 0) w.hits = w.candidates = 0;
      __syncwarp();
      while (hits) {
        const uint32_t at = (__ffs(hits) - 1) * 32 + lane;
        hits &= hits - 1;
        if (at >= p.end) break;  // -inf in place of vectors that a row lacks
        const uint32_t i = atomicAdd(&w.hits, 1u);
        if (i < kHits) w.hit[i] = at;
      }
      const auto candidate = [&](float x, uint32_t id) {
        const uint32_t i = atomicAdd(&w.candidates, 1u);
        if (i < kCandidates) w.key[i] = list_key<T>(x, id), w.id[i] = id;
      };
      if (lane < p.loose && loose >= from) candidate(loose, loose_at(p, lane));
      __syncwarp();
      const uint32_t vectors = w.hits;
      if (vectors <= kHits)
        for (uint32_t i = lane; i < vectors * E; i += 32) {
          const uint32_t j = w.hit[i / E] * E + i % E;
          const float x = to_float(reinterpret_cast<const T *>(w.row)[j]);
          if (x >= from) candidate(x, p.head + j);
        }
      __syncwarp();
      uint32_t candidates = w.candidates;
      if (vectors > kHits || candidates > kCandidates || candidates < a.top) {
        careful_warp_top(z, a.vocab, a.top, least, w.key, w.id);
        candidates = a.top;
      }
      row += stride;
      begin_row();
      if (lane < 4 && candidates + lane < kCandidates) w.key[candidates + lane] = 0;
      __syncwarp();
      if (candidates <= 32) rank_candidates<T, 1>(a, r, s, w.key, w.id, candidates, lane);
      else if (candidates <= 64) rank_candidates<T, 2>(a, r, s, w.key, w.id, candidates, lane);
      else if (candidates <= 96) rank_candidates<T, 3>(a, r, s, w.key, w.id, candidates, lane);
      else if (candidates <= 128) rank_candidates<T, 4>(a, r, s, w.key, w.id, candidates, lane);
      else if (candidates <= 192) rank_candidates<T, 6>(a, r, s, w.key, w.id, candidates, lane);
      else rank_candidates<T, kCandidates / 32>(a, r, s, w.key, w.id, candidates, lane);
      __syncwarp();  // the list is free for the next row
    } else {
      __syncwarp();
      row += stride;
      begin_row();
    }
  }
}

template <typename T, int NV, bool ENTROPY>
__global__ void __launch_bounds__(kShortWarps * 32) score_backward_short_kernel(const ScoreArgs a) {
  extern __shared__ uint4 shared[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4 *buffer = shared + warp * NV * 32;
  const size_t stride = static_cast<size_t>(gridDim.x) * kShortWarps;
  size_t row = static_cast<size_t>(blockIdx.x) * kShortWarps + warp;
  pdl_enter();
  for (; row < a.rows; row += stride) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
    const Part p = part_of(z, a.vocab, 0, 1);
    stage_row<T, NV>(z, p, lane, buffer);
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
    const Pair c2 = pair(a.c, a.c);
    const auto fast = [&](float x) { return score_dz<ENTROPY>(g, a.c, x); };
    const auto fast2 = [&](Pair x) { return score_dz2<ENTROPY>(g, c2, x); };
    const auto careful = [&](float x) { return careful_score_dz(g, a, x); };
    await_row();  // and the target's logit is read: dz may be z
    if (!g.none && !g.far) {
      write_row<T, NV>(dz, p, lane, buffer, loose, fast2, fast);
    } else {
      for (uint32_t j = lane; j < a.vocab; j += 32)
        dz[j] = from_float<T>(g.none ? 0.0f : careful(to_float(z[j])));
    }
    __syncwarp();
    if (lane == 0 && t != TL_NO_TOKEN && !g.none)
      dz[t] = from_float<T>((g.far ? careful(zt) : fast(zt)) + gl);
  }
}

// Launches a kernel of CTAs of W warps that need `warp_bytes` of shared
// memory each.
template <int W, typename K> void launch_short(K kernel, const ScoreArgs &a, size_t warp_bytes, cudaStream_t s) {
  const size_t smem = warp_bytes * W;
  if (smem > 48 * 1024)  // a failure shows in the launch's status
    (void)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_pdl(kernel, short_grid(a.rows, W, smem), W * 32, smem, s, a);
}

template <typename T, int NV> void launch(const ScoreArgs &a, cudaStream_t s) {
  constexpr size_t with = sizeof(WarpShared<NV, true>), without = sizeof(WarpShared<NV, false>);
  if (a.entropy) {
    if (a.top) launch_short<kScoreWarps>(score_short_kernel<T, NV, true, true>, a, with, s);
    else launch_short<kScoreWarps>(score_short_kernel<T, NV, true, false>, a, without, s);
  } else {
    if (a.top) launch_short<kScoreWarps>(score_short_kernel<T, NV, false, true>, a, with, s);
    else launch_short<kScoreWarps>(score_short_kernel<T, NV, false, false>, a, without, s);
  }
}

template <typename T, int NV> void launch_backward(const ScoreArgs &a, cudaStream_t s) {
  if (a.d_entropy) launch_short<kShortWarps>(score_backward_short_kernel<T, NV, true>, a, NV * 512, s);
  else launch_short<kShortWarps>(score_backward_short_kernel<T, NV, false>, a, NV * 512, s);
}

}  // namespace

bool score_short(const ScoreArgs &a, int32_t type, cudaStream_t s) {
  const uint32_t nv = short_vectors(a.rows, a.vocab, type_size(type));
  if (!nv) return false;
#define L(T) nv == 4 ? launch<T, 4>(a, s) : nv == 16 ? launch<T, 16>(a, s) : launch<T, 32>(a, s)
  TL_BY_TYPE(type, L)
#undef L
  return true;
}

bool score_backward_short(const ScoreArgs &a, int32_t type, cudaStream_t s) {
  const uint32_t nv = short_vectors(a.rows, a.vocab, type_size(type));
  if (!nv) return false;
#define L(T) nv == 4 ? launch_backward<T, 4>(a, s) : nv == 16 ? launch_backward<T, 16>(a, s) : launch_backward<T, 32>(a, s)
  TL_BY_TYPE(type, L)
#undef L
  return true;
}

}  // namespace token
}  // namespace tl
