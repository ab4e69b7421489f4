// Arguments of the attention kernels over a paged cache and the plain loop
// over one row's keys (k_paged_attention*.cu).
#pragma once

#include "paged_cache.cuh"

namespace tl {
namespace paged {

constexpr uint32_t kMaxHead = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A job that is cut over several CTAs, written by the one that ends it: its
// first CTA (none: UINT32_MAX) and which rows it is.
struct Join {
  uint32_t first, sequence, head, tile;
};

struct AttentionArgs {
  tl_paged_cache cache;
  tl_head_view q, out;
  uint32_t q_heads, group;  // query heads, query heads of a key head
  uint32_t window, causal;
  uint64_t most;            // keys that a sequence can have
  float scale;
  float *lse;
  uint32_t *status;
  // shares of the work, see Share
  float *parts;       // [ctas, 2] partial results
  Join *joins;        // [ctas]
  uint32_t whole;     // jobs are not cut
};

// Keys [from, to) that the token at `position` sees.
__device__ __forceinline__ void seen(const AttentionArgs &a, uint32_t length, int64_t position, uint32_t &from,
                                     uint32_t &to) {
  from = 0;
  to = length;
  if (!a.causal && !a.window) return;
  if (a.causal) to = position < 0 ? 0u : static_cast<uint32_t>(min(static_cast<int64_t>(length), position + 1));
  if (a.window) {
    const int64_t first = position + 1 - static_cast<int64_t>(a.window);
    if (first > 0) from = static_cast<uint32_t>(min(first, static_cast<int64_t>(to)));
  }
}

// Offset of key j of sequence s in the cache (elements), or a negative number
// where its page does not exist (the flag is raised).
__device__ __forceinline__ int64_t key_offset(const AttentionArgs &a, uint32_t s, uint32_t j) {
  const tl_paged_cache &c = a.cache;
  const uint32_t block = j / c.page_size;
  const uint32_t page = c.table[static_cast<uint64_t>(s) * c.table_stride + block];
  if (page >= c.pages) {
    raise_flag(a.status, TL_FLAG_INDEX_RANGE);
    return -1;
  }
  return static_cast<int64_t>(page * c.page_stride + (j - block * c.page_size) * c.slot_stride);
}

// One query row over keys [from, to) by a warp, nothing but its own keys
// touched: 32 scores at a time, a lane each, then the lanes share the values'
// elements.  acc[i] is element lane + 32 i; m is in units of log2.
template <typename T>
__device__ __forceinline__ void row_over_keys(const AttentionArgs &a, uint32_t s, uint32_t head, const T *q,
                                              uint32_t from, uint32_t to, uint32_t lane, float &m, float &l,
                                              float (&acc)[kMaxHead / 32]) {
  const tl_paged_cache &c = a.cache;
  const T *k = static_cast<const T *>(c.k) + head * c.head_stride;
  const T *v = static_cast<const T *>(c.v) + head * c.head_stride;
  const float scale = a.scale * kLog2e;
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < static_cast<int>(kMaxHead) / 32; ++i) acc[i] = 0.0f;
  for (uint32_t j0 = from; j0 < to; j0 += 32) {
    const int64_t at = j0 + lane < to ? key_offset(a, s, j0 + lane) : -1;
    float x = -INFINITY;
    if (at >= 0) {
      x = 0.0f;
      for (uint32_t d = 0; d < c.D; ++d) x = fmaf(heads::element_of(q[d]), heads::element_of(k[at + d]), x);
      x *= scale;
    }
    float top = x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float to_m = fmaxf(m, top), base = to_m == -INFINITY ? 0.0f : to_m;
    const float p = x == -INFINITY ? 0.0f : exp2f(x - base), f = m == -INFINITY ? 0.0f : exp2f(m - base);
    l = fmaf(l, f, warp_sum(p));
    m = to_m;
#pragma unroll
    for (int i = 0; i < static_cast<int>(kMaxHead) / 32; ++i) acc[i] *= f;
    for (uint32_t i = 0; i < 32 && j0 + i < to; ++i) {
      const float w = __shfl_sync(0xffffffffu, p, i);
      const int64_t place = __shfl_sync(0xffffffffu, at, i);
      const float score = __shfl_sync(0xffffffffu, x, i);
      if (place < 0 || score == -INFINITY) continue;
#pragma unroll
      for (int e = 0; e < static_cast<int>(kMaxHead) / 32; ++e)
        if (lane + 32 * e < c.D) acc[e] = fmaf(w, heads::element_of(v[place + lane + 32 * e]), acc[e]);
    }
  }
}

// How the work is shared out.  A job is one key head's query rows of one
// sequence, `ROWS` rows at most (token by token, the group's heads of a token
// side by side), over the sequence's keys in blocks of `KEYS`.  All blocks of
// all jobs lie in one line, which is cut into equal shares; a share that starts
// or ends inside a job leaves a partial result (numerators' sum, maximum and
// sum of the softmax), and join_kernel adds those up in the order of the keys.
// Every CTA works its share out by itself from the lengths on the device, so
// that a captured call follows them.
template <uint32_t ROWS, uint32_t KEYS> struct Work {
  Sequence q;
  uint32_t first, blocks;  // the sequence's blocks, from the first that any of its rows sees
  uint64_t tiles;

  __device__ __forceinline__ void set(const AttentionArgs &a, uint32_t s) {
    q = sequence_of(a.cache, s, a.most);
    const int64_t lo = a.window ? static_cast<int64_t>(q.length) - q.count + 1 - static_cast<int64_t>(a.window) : 0;
    first = lo > 0 ? static_cast<uint32_t>(lo / KEYS) : 0;
    const uint32_t end = static_cast<uint32_t>((static_cast<uint64_t>(q.length) + KEYS - 1) / KEYS);
    blocks = end > first ? end - first : 1;
    tiles = (static_cast<uint64_t>(q.count) * a.group + ROWS - 1) / ROWS;
  }
  // places in the line
  __device__ __forceinline__ uint64_t cost(const AttentionArgs &a) const {
    return tiles * a.cache.heads * (a.whole ? 1 : blocks);
  }
};

// The sequence in which this CTA's share starts, the share's offset in it and
// its size; the line's length is cut into `ctas` shares of at least `least`.
struct Share {
  uint64_t begin, size;  // in the line
  uint64_t full;         // what every share but the last is
  uint64_t offset;       // of the share's start in its sequence
  uint32_t sequence;
  bool any;
};
template <uint32_t ROWS, uint32_t KEYS, int THREADS>
__device__ __forceinline__ Share share_of(const AttentionArgs &a, uint32_t cta, uint32_t ctas, uint32_t least) {
  constexpr int kWarps = THREADS / 32;
  __shared__ uint64_t warp_sum[kWarps + 1];
  __shared__ Share found;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid / 32, n = a.cache.sequences;
  const uint32_t per = (n + THREADS - 1) / THREADS, s0 = tid * per, s1 = min(s0 + per, n);
  Work<ROWS, KEYS> w;
  uint64_t mine = 0;
  for (uint32_t s = s0; s < s1; ++s) {
    w.set(a, s);
    if (w.q.bad && cta == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
    mine += w.cost(a);
  }
  uint64_t up = mine;  // inclusive sums over the warp, then over the CTA
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t v = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= static_cast<uint32_t>(o)) up += v;
  }
  if (lane == 31) warp_sum[warp] = up;
  if (tid == 0) found.any = false;
  __syncthreads();
  uint64_t before = up - mine, total = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (static_cast<uint32_t>(i) < warp) before += warp_sum[i];
    total += warp_sum[i];
  }
  uint64_t size = (total + ctas - 1) / ctas;
  if (size < least) size = least;
  const uint64_t begin = size * cta;
  if (begin >= before && begin < before + mine) {
    uint32_t s = s0;
    for (; s < s1; ++s) {
      w.set(a, s);
      const uint64_t c = w.cost(a);
      if (begin < before + c) break;
      before += c;
    }
    found = Share{begin, min(size, total - begin), size, begin - before, s, true};
  }
  __syncthreads();
  return found;
}


// What a call asks of a kernel family: its grid and the workspace's floats
// behind the joins.
struct Plan {
  uint32_t ctas, whole;
  uint64_t part_floats;  // of a partial result, 0 where jobs are not cut
};
inline uint64_t plan_bytes(const Plan &p) {
  return p.whole ? 0 : p.ctas * (2 * p.part_floats * sizeof(float) + sizeof(Join));
}
// Most blocks of `keys` that a job can have, and most jobs of `rows` rows.
inline uint64_t most_blocks(const AttentionArgs &a, uint32_t max_new, uint32_t keys) {
  uint64_t n = a.most;
  if (a.window && static_cast<uint64_t>(a.window) + max_new < n) n = static_cast<uint64_t>(a.window) + max_new;
  return n / keys + 2;
}
inline uint64_t most_jobs(const AttentionArgs &a, uint32_t rows) {
  return (static_cast<uint64_t>(a.cache.tokens) * a.group / rows + a.cache.sequences) * a.cache.heads;
}

Plan step_plan(const AttentionArgs &a, uint32_t max_new);
void launch_step(const AttentionArgs &a, const Plan &p, bool wide, cudaStream_t s);

}  // namespace paged
}  // namespace tl
