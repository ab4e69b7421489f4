// Arguments and work shares of the rotation kernels (k_rotary.cu,
// k_rotary_backward.cu).
#pragma once

#include "heads.cuh"

namespace tl {
namespace heads {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kBatch = 4;                   // head rows in flight a lane
constexpr uint32_t kMaxCtas = kNumSMs * 4;  // of the gradient: a row of partial weight gradients each

struct RotaryPart {
  tl_head_view x, out, d_out, dx;
  const float *weight;
  float *dweight, *partial;  // partial: [ctas, D]
  uint32_t heads, ctas;
  uint32_t chunks, steps, all_steps;  // a token's heads in runs of `steps` head rows
};
struct RotaryArgs {
  RotaryPart part[2];
  uint32_t D, T, tokens, rotary, lanes;
  bool interleaved, norm, vectors;
  float eps, inv_d, magnitude;
  const uint64_t *frequencies;
  const uint32_t *positions;
  uint32_t first_position;
};

// Checks a descriptor and fills in everything but the shares.
int rotary_args(const char *who, const tl_rotary_desc *d, bool backward, RotaryArgs &a);
// Shares the work out; the grid.
unsigned share_out(RotaryArgs &a, bool persistent);

}  // namespace heads
}  // namespace tl
