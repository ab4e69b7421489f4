// Arguments of the attention kernels over a paged cache and the plain loop
// over one row's keys (k_paged_attention*.cu).
#pragma once

#include "paged_cache.cuh"

namespace tl {
namespace paged {

constexpr uint32_t kMaxHead = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 16 bytes into shared memory, zeros where they are not there
__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void await() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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

// Whether a value of the keys [from, to) is not finite, by a warp.
template <typename T>
__device__ __forceinline__ bool any_infinite(const AttentionArgs &a, uint32_t s, uint32_t head, uint32_t from, uint32_t to, uint32_t lane) {
  const T *v = static_cast<const T *>(a.cache.v) + head * a.cache.head_stride;
  bool found = false;
  for (uint32_t j = from; j < to && !found; ++j) {
    const int64_t at = key_offset(a, s, j);
    for (uint32_t d = lane; at >= 0 && d < a.cache.D; d += 32) {
      const float x = heads::element_of(v[at + d]);
      found = found || x - x != 0.0f;
    }
    found = __any_sync(0xffffffffu, found);
  }
  return found;
}

// How the work is shared out.  A job is one key head's query rows of one
// sequence, `ROWS` rows at most (a tile; token by token, the group's heads of
// a token side by side), over the keys that they see, in blocks of `KEYS`.
// The jobs lie in one line, sequence by sequence, tile by tile, head by head, each
// as long as its keys (for causal tiles an even slope, at least what they see)
// and kJob more, about what starting and ending a job costs.  With 1, 2, 3, 5 and 8
// blocks, 64 sequences of 16 to 8191 keys and a new token each took 148, 126, 112, 105
// and 108 us, 8192 tokens of one prompt 893, 736, 609, 570 and 588, 24 chunks 113, 91,
// 87, 89 and 95.  The line is cut into equal shares; a share that starts or ends
// inside a job leaves a partial result (numerators' sum, maximum and sum of
// the softmax), and join_kernel adds those up in the order of the keys.
// Every CTA works its share out by itself from the lengths on the device, so
// that a captured call follows them.
template <uint32_t ROWS, uint32_t KEYS> struct Work {
  static constexpr uint64_t kJob = 5 * KEYS;
  Sequence q;
  uint64_t tiles;
  uint64_t base, slope;  // line of tile t: base + slope t, for each head

  __device__ __forceinline__ void set(const AttentionArgs &a, uint32_t s) {
    q = sequence_of(a.cache, s, a.most);
    tiles = (static_cast<uint64_t>(q.count) * a.group + ROWS - 1) / ROWS;
    const uint32_t step = (ROWS + a.group - 1) / a.group;  // tokens of a tile
    slope = 0;
    if (a.whole) {
      base = 1;
      return;
    }
    base = q.length;
    if (a.window) base = min(base, static_cast<uint64_t>(a.window) + step + KEYS);
    else if (a.causal) {
      slope = step;
      base = (q.total > q.count ? min(q.total - q.count, q.length) : 0) + step;
    }
    base += kJob;
  }
  // the line before tile t
  __device__ __forceinline__ uint64_t before(const AttentionArgs &a, uint64_t t) const {
    return a.cache.heads * (t * base + (t ? t * (t - 1) / 2 : 0) * slope);
  }
};

// This CTA's share: its place in the line and the sequence it starts in.
struct Share {
  uint64_t begin, size;  // in the line
  uint64_t full;         // what every share but the last is
  uint64_t offset;       // of the share's start in its sequence
  uint32_t sequence;
  bool any;
};
template <uint32_t ROWS, uint32_t KEYS, int THREADS>
__device__ __forceinline__ Share share_of(const AttentionArgs &a, uint32_t cta, uint32_t ctas, uint64_t least) {
  constexpr int kWarps = THREADS / 32;
  __shared__ uint64_t warp_sum[kWarps];
  __shared__ Share found;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid / 32, n = a.cache.sequences;
  const uint32_t per = (n + THREADS - 1) / THREADS, s0 = min(tid * per, n), s1 = min(s0 + per, n);
  Work<ROWS, KEYS> w;
  uint64_t mine = 0;
  for (uint32_t s = s0; s < s1; ++s) {
    w.set(a, s);
    if (w.q.bad && cta == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
    mine += w.before(a, w.tiles);
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
      const uint64_t c = w.before(a, w.tiles);
      if (begin < before + c) break;
      before += c;
    }
    found = Share{begin, min(size, total - begin), size, begin - before, s, true};
  }
  __syncthreads();
  return found;
}

// A part of a job: what a CTA does of it.
struct Piece {
  uint32_t sequence, head, tile;
  uint32_t start;              // first row of its sequence's tokens
  uint32_t block_lo, block_hi; // blocks of the keys [block * KEYS, ..)
  bool opens, ends;            // the job's first block, its last one
  uint32_t first_cta;          // that has its first block
  uint32_t row0;               // of the tile, among the sequence's rows (fewer than 2^32)
  uint32_t last;               // its last row
  uint32_t length;             // the sequence's keys
  int64_t position0;           // of the sequence's first new token
  uint32_t from, to;           // keys that any of its rows sees
  __device__ __forceinline__ int64_t position(const AttentionArgs &a, uint32_t row) const {
    return position0 + static_cast<int64_t>((row0 + row) / a.group);
  }
};

// The pieces of a share, in order.
template <uint32_t ROWS, uint32_t KEYS> struct Walk {
  Work<ROWS, KEYS> w;
  uint64_t offset, left, at;
  uint32_t s;

  __device__ __forceinline__ void start(const AttentionArgs &a, const Share &share) {
    s = share.sequence;
    offset = share.offset;
    at = share.begin;
    left = share.any ? share.size : 0;
    if (left) w.set(a, s);
  }
  __device__ __forceinline__ bool next(const AttentionArgs &a, const Share &share, Piece &p) {
    while (left) {
      const uint64_t line = w.before(a, w.tiles);
      if (offset >= line) {  // the next sequence with any rows
        offset -= line;
        w.set(a, ++s);
        continue;
      }
      uint64_t lo = 0, hi = w.tiles;  // the last tile that starts at or before offset
      while (hi - lo > 1) {
        const uint64_t mid = (lo + hi) / 2;
        if (w.before(a, mid) <= offset) lo = mid;
        else hi = mid;
      }
      const uint64_t job = w.base + w.slope * lo, in_tile = offset - w.before(a, lo);
      const uint64_t x0 = in_tile % job, take = min(left, job - x0), x1 = x0 + take;
      p.sequence = s;
      p.head = static_cast<uint32_t>(in_tile / job);
      p.tile = static_cast<uint32_t>(lo);
      p.start = w.q.start;
      p.row0 = static_cast<uint32_t>(lo) * ROWS;
      p.last = min(ROWS, w.q.count * a.group - p.row0) - 1;
      p.length = w.q.length;
      p.position0 = static_cast<int64_t>(w.q.total) - w.q.count;
      uint32_t unused;
      seen(a, w.q.length, p.position(a, 0), p.from, unused);
      seen(a, w.q.length, p.position(a, p.last), unused, p.to);
      const uint32_t first = p.from / KEYS;
      const uint32_t end = static_cast<uint32_t>((static_cast<uint64_t>(p.to) + KEYS - 1) / KEYS);
      const uint32_t blocks = end > first ? end - first : 1;  // rows without keys are written too
      const auto block = [&](uint64_t x) {
        if (a.whole || x == job) return x ? blocks : 0u;
        return static_cast<uint32_t>(min(x > w.kJob ? (x - w.kJob) / KEYS : 0, static_cast<uint64_t>(blocks)));
      };
      const uint32_t b0 = block(x0), b1 = block(x1);
      const uint64_t job_at = at - x0;
      offset += take;
      at += take;
      left -= take;
      if (b0 == b1) continue;  // nothing but a job's overhead, or behind its keys
      p.block_lo = first + b0;
      p.block_hi = first + b1;
      p.opens = b0 == 0;
      p.ends = b1 == blocks;
      p.first_cta = static_cast<uint32_t>((job_at + w.kJob + KEYS - 1) / share.full);
      return true;
    }
    return false;
  }
};

// One row's result: the whole of it, or a part in the workspace.
__device__ __forceinline__ void put_lse(const AttentionArgs &a, uint64_t token, uint32_t h, float m, float l) {
  if (a.lse) a.lse[token * a.q_heads + h] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
}

// floats of a partial result of a tile: outputs, maxima, sums
template <uint32_t ROWS, int DP> constexpr uint32_t part_floats() { return ROWS * DP + 2 * ROWS; }

// The jobs that were cut, each where it ends: the partial results of a row are
// added up in the order of the keys, a lane DP / 32 neighbouring elements.  Large
// tiles are cut in two or three: a warp takes four rows, all their loads under
// way at once (one row after another took 22 us for 147 joins of 256 rows, so 15).
// Small ones may be cut in many: four warps share a row's parts (37 parts of 8 jobs
// of 4 rows: 40 us by one warp, so 8).  The factors of 32 parts are worked out first, a
// lane each, so that no load of outputs waits for one (19 parts of 8 jobs of 20 rows:
// 33 us where each part's factor came before its outputs, so 15).
template <typename TO, uint32_t ROWS, int DP>
__global__ void __launch_bounds__(128) join_kernel(const AttentionArgs a) {
  constexpr bool kShare = ROWS <= 16;
  constexpr int R = kShare ? 1 : 4, E = DP / 32;
  __shared__ float sums[kShare ? 4 : 1][DP];
  pdl_enter();
  const Join j = a.joins[blockIdx.x];
  if (j.first == 0xffffffffu) return;
  const uint32_t lane = threadIdx.x & 31, end = blockIdx.x;
  const Sequence q = sequence_of(a.cache, j.sequence, a.most);
  const uint32_t row0 = j.tile * ROWS, rows = min(ROWS, q.count * a.group - row0);
  const uint32_t warp = threadIdx.x / 32, r0 = kShare ? blockIdx.y : (blockIdx.y * 4 + warp) * R;
  if (r0 >= rows) return;
  const auto part = [&](uint32_t cta) {
    return a.parts + (static_cast<size_t>(cta) * 2 + (cta == j.first ? 1 : 0)) * part_floats<ROWS, DP>();
  };
  float mm[R], ll[R], acc[R][E];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mm[r] = -INFINITY;
    ll[r] = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[r][e] = 0.0f;
  }
  for (uint32_t i = j.first + lane; i <= end; i += 32)
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (r0 + r < rows) mm[r] = fmaxf(mm[r], part(i)[ROWS * DP + r0 + r]);
#pragma unroll
  for (int r = 0; r < R; ++r) mm[r] = warp_max(mm[r]);
  // 32 parts at a time: their factors, a lane each, then their outputs
  constexpr uint32_t kStep = kShare ? 4 : 1;
  for (uint32_t i0 = j.first; i0 <= end; i0 += 32) {
    const uint32_t i = i0 + lane, n = min(32u, end - i0 + 1);
    float f[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f[r] = 0.0f;
      if (r0 + r >= rows || i > end) continue;
      const float wm = part(i)[ROWS * DP + r0 + r], wl = part(i)[ROWS * DP + ROWS + r0 + r];
      f[r] = wm == -INFINITY ? 0.0f : ex2_approx(wm - mm[r]);
      ll[r] = fmaf(f[r], wl, ll[r]);
    }
#pragma unroll 4
    for (uint32_t k = kShare ? warp : 0; k < n; k += kStep) {
      const float *const p = part(i0 + k);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float by = __shfl_sync(0xffffffffu, f[r], k);
        float x[E] = {};
        if (r0 + r < rows) {
          if constexpr (E == 4) {
            const float4 y = *reinterpret_cast<const float4 *>(p + (r0 + r) * DP + lane * E);
            x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
          } else {
            const float2 y = *reinterpret_cast<const float2 *>(p + (r0 + r) * DP + lane * E);
            x[0] = y.x, x[1] = y.y;
          }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = by != 0.0f ? fmaf(by, x[e], acc[r][e]) : acc[r][e];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) ll[r] = warp_sum(ll[r]);
  if constexpr (kShare) {
#pragma unroll
    for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = acc[0][e];
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
#pragma unroll
      for (int e = 0; e < E; ++e) acc[0][e] += sums[w][lane * E + e];
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r0 + r >= rows) continue;
    const uint32_t place = row0 + r0 + r, in_sequence = place / a.group;
    const uint64_t token = q.start + static_cast<uint64_t>(in_sequence);
    const uint32_t h = j.head * a.group + (place - in_sequence * a.group);
    TO *out = static_cast<TO *>(const_cast<void *>(a.out.p)) + token * a.out.row_stride + h * a.out.head_stride;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane * E + e < a.cache.D) heads::set_element(out[lane * E + e], ll[r] == 0.0f ? 0.0f : acc[r][e] / ll[r]);
    if (lane == 0) put_lse(a, token, h, mm[r], ll[r]);
  }
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
Plan tile_plan(const AttentionArgs &a);
void launch_tile(const AttentionArgs &a, const Plan &p, bool wide, cudaStream_t s);

}  // namespace paged
}  // namespace tl
