// Arguments of the attention kernels over a paged cache and the plain loop
// over one row's keys (k_paged_attention*.cu).
#pragma once

#include "paged_cache.cuh"

namespace tl {
namespace paged {

constexpr uint32_t kMaxHead = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttentionArgs {
  tl_paged_cache cache;
  tl_head_view q, out;
  uint32_t q_heads, group;  // query heads, query heads of a key head
  uint32_t window, causal;
  uint64_t most;            // keys that a sequence can have
  float scale;
  float *lse;
  uint32_t *status;
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

}  // namespace paged
}  // namespace tl
