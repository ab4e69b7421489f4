// What the cache's writer and its reader share (k_cache_append.cu,
// k_paged_*.cu): the check of a cache's fields and where a sequence's tokens
// and keys lie.
#pragma once

#include "heads.cuh"

namespace tl {
namespace paged {

// The descriptor's cache with its default strides filled in; `rows` of keys
// are 16-byte aligned when *aligned.
int check_cache(const char *who, tl_paged_cache &c, bool *aligned);

// One sequence of a batch as a kernel may use it: its new tokens' rows and
// its keys, clipped to what the tensors hold.
struct Sequence {
  uint32_t start, count;  // rows of its new tokens
  uint32_t length;        // keys
  uint32_t total;         // keys before they were clipped, which the positions go by
  bool bad;               // something was clipped
};
__device__ __forceinline__ Sequence sequence_of(const tl_paged_cache &c, uint32_t s, uint64_t most) {
  const uint32_t start = c.starts[s], end = c.starts[s + 1], length = c.lengths[s];
  Sequence q{start, end - start, length, length, false};
  if (end < start || end > c.tokens) {
    q.bad = true;
    q.count = 0;
  }
  if (length > most) {
    q.bad = true;
    q.length = static_cast<uint32_t>(most);
  }
  return q;
}
// keys that a row of the table can hold, 2^31 at most
__host__ __device__ __forceinline__ uint64_t table_keys(const tl_paged_cache &c) {
  const uint64_t n = static_cast<uint64_t>(c.table_stride) * c.page_size;
  return n < 1ull << 31 ? n : 1ull << 31;
}

// The last sequence that starts at or before row `token`, by a warp: 32
// places at a time.  UINT32_MAX when there is none; whether the row lies in
// that sequence is the caller's to check.
__device__ __forceinline__ uint32_t sequence_at(const tl_paged_cache &c, uint32_t token, uint32_t lane) {
  uint32_t lo = 0, hi = c.sequences;
  for (;;) {
    const uint32_t step = (hi - lo + 31) / 32, i = lo + lane * step;
    const unsigned ok = __ballot_sync(0xffffffffu, i < hi && c.starts[i] <= token);
    if (!ok) return 0xffffffffu;
    lo += (__popc(ok) - 1) * step;
    if (step == 1) return lo;
    hi = min(hi, lo + step);
  }
}

}  // namespace paged
}  // namespace tl
