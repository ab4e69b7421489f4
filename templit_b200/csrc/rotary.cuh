// Arguments and work shares of the rotation kernels (k_rotary.cu,
// k_rotary_backward.cu).
#pragma once

#include "heads.cuh"

namespace tl {
namespace heads {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr uint32_t kMaxCtas = kNumSMs * 4;  // one round of the SMs, at most

struct RotaryPart {
  tl_head_view x, out, d_out, dx;
  const float *weight;
  float *dweight, *partial;  // partial: [ctas, D]
  uint32_t heads, ctas;
  uint32_t chunks, run;  // a token's heads in runs of `run`, a warp each
};
struct RotaryArgs {
  RotaryPart part[2];
  uint32_t D, T, tokens, rotary, lanes;
  bool interleaved, norm, vectors;
  bool whole;  // a token's heads of both parts are one group
  float eps, inv_d, magnitude;
  const uint64_t *frequencies;
  const uint32_t *positions;
  uint32_t first_position;
};

// Where a warp is: a batch of heads of one token.  Warps stay on the SMs and
// load the next batch before they work on the one that they hold, so that
// loads are always under way (a warp a token, without: 12288 x 12 heads of 64
// fp32 20 us, norm and rotation of 16384 x 40 heads of 128 bf16 86 us).
struct Batch {
  uint64_t group;  // run of a token's heads
  uint32_t part, token, b, t, position;
  uint32_t head, end;
  bool any;
};
// A group's first batch.  Where a token's heads are one run, a group is the
// token, its queries first and then its keys; else the runs of all tokens'
// queries lie before those of the keys (apart: each part's groups by themselves).
__device__ __forceinline__ void set_batch(const RotaryArgs &a, Batch &s, uint64_t first_groups, uint64_t groups) {
  s.any = s.group < groups;
  if (!s.any) return;
  s.part = a.whole ? a.part[0].heads == 0 : s.group >= first_groups;
  const RotaryPart &p = a.part[s.part];
  const uint64_t g = !a.whole && s.part ? s.group - first_groups : s.group;
  // groups fit in 32 bits where chunks > 1 (few tokens)
  s.token = p.chunks == 1 ? static_cast<uint32_t>(g) : static_cast<uint32_t>(g) / p.chunks;
  const uint32_t chunk = p.chunks == 1 ? 0 : static_cast<uint32_t>(g) - s.token * p.chunks;
  s.b = s.token / a.T;
  s.t = s.token - s.b * a.T;
  s.position = a.positions ? a.positions[s.token] : a.first_position + s.t;
  s.head = chunk * p.run;
  s.end = min(s.head + p.run, p.heads);
}
// The batch behind s, `step` heads on; whether it is of the same run.
__device__ __forceinline__ bool next_batch(const RotaryArgs &a, Batch &s, uint32_t step, uint64_t stride, uint64_t first_groups,
                                           uint64_t groups) {
  s.head += step;
  if (s.head < s.end) return true;
  if (a.whole && s.part == 0 && a.part[1].heads) {
    s.part = 1;
    s.head = 0;
    s.end = a.part[1].heads;
  } else {
    s.group += stride;
    set_batch(a, s, first_groups, groups);
  }
  return false;
}
__device__ __forceinline__ uint64_t place(const tl_head_view &v, const Batch &s, uint32_t sub) {
  return s.b * v.batch_stride + s.t * v.row_stride + (s.head + sub) * v.head_stride;
}

// U head rows of a lane; vectors that it has none of stay 0.
template <typename T, int V, int U> struct HeadRows {
  Raw<T, V> a[U], b[U];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = b[u] = Raw<T, V>{};
  }
  // Rows `step` apart; `left` heads, `per` at a time, are there.  The others are 0
  // (EMPTY: they add to sums over heads) or keep what they held, which goes nowhere.
  template <bool EMPTY> __device__ __forceinline__ void load(const T *x, uint64_t step, const Slot &slot, uint32_t left, uint32_t per) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (EMPTY) a[u] = b[u] = Raw<T, V>{};
      if (u * per < left && slot.has_a) a[u].load(x + u * step + slot.a);
      if (u * per < left && slot.has_b) b[u].load(x + u * step + slot.b);
    }
  }
};

// Checks a descriptor and fills in everything but the shares.
int rotary_args(const char *who, const tl_rotary_desc *d, bool backward, RotaryArgs &a);
// Shares the work out over `most` CTAs, `rows` head rows a batch; the grid.
// `apart`: each CTA takes heads of one part only.
unsigned share_out(RotaryArgs &a, uint32_t rows, uint32_t most, bool apart);

}  // namespace heads
}  // namespace tl
