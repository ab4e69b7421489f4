// Gradient of the rotation and norm of heads (include/templit_cuda.h:
// tl_rotary_heads_backward).  With g = the incoming gradient turned back and
// x^ = x / rms:
//   dw = sum over tokens and heads of g x^
//   dx = (g w - x^ mean(g w x^)) / rms            (norm; else dx = g)
// Bound by memory: d_out and x are read once, dx is written once.  The grid
// stays on the SMs; a CTA adds its heads' weight gradients up in registers,
// then in shared memory, and leaves one row, which a second kernel sums over
// the CTAs in a fixed order.
#include "rotary.cuh"

namespace tl {
namespace heads {
namespace {

template <typename TI, typename TO, int V, int S, bool NORM, bool INTER>
__global__ void __launch_bounds__(kThreads) rotate_backward_kernel(const RotaryArgs a) {
  constexpr int U = V == 1 ? 1 : kBatch / 2;
  __shared__ float sums[kWarps][TL_HEAD_MAX_DIM];
  pdl_enter();
  const bool second = blockIdx.x >= a.part[0].ctas;
  const RotaryPart &part = a.part[second];
  const uint32_t cta = blockIdx.x - (second ? a.part[0].ctas : 0);
  const bool inter = V == 1 ? a.interleaved : INTER;
  const bool norm = V == 1 ? a.norm : NORM;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint32_t lanes = a.lanes, at = lane & (lanes - 1), sub = lane / lanes, per = 32 / lanes;

  Slot slot[S];
  float wa[S][V], wb[S][V], dwa[S][V], dwb[S][V];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    slot[s] = slot_of(at + s * lanes, V, a.D, a.rotary, inter);
    load_weights<V>(norm ? part.weight : nullptr, slot[s], wa[s], wb[s]);
#pragma unroll
    for (int i = 0; i < V; ++i) dwa[s][i] = dwb[s][i] = 0.0f;
  }
  const uint64_t items = static_cast<uint64_t>(a.tokens) * part.chunks;
  const uint64_t warps = static_cast<uint64_t>(part.ctas) * kWarps;
  for (uint64_t item = static_cast<uint64_t>(cta) * kWarps + warp; item < items; item += warps) {
    const uint32_t token = static_cast<uint32_t>(item / part.chunks), chunk = static_cast<uint32_t>(item % part.chunks);
    const uint32_t b = token / a.T, t = token % a.T;
    float cos[S][V], sin[S][V];
    angles<V, S>(a.frequencies, a.positions ? a.positions[token] : a.first_position + t, a.magnitude, at, lanes,
                 a.rotary, cos, sin);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int i = 0; i < V; ++i) sin[s][i] = -sin[s][i];
    const TI *x = static_cast<const TI *>(part.x.p) + b * part.x.batch_stride + t * part.x.row_stride;
    const TO *g = static_cast<const TO *>(part.d_out.p) + b * part.d_out.batch_stride + t * part.d_out.row_stride;
    TI *dx = static_cast<TI *>(const_cast<void *>(part.dx.p)) + b * part.dx.batch_stride + t * part.dx.row_stride;
    const uint32_t end = min((chunk + 1) * part.steps, part.all_steps);
    for (uint32_t step = chunk * part.steps; step < end; step += U) {
      Raw<TO, V> ra[U][S], rb[U][S];
      Raw<TI, V> xa[U][S], xb[U][S];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t h = (step + u) * per + sub;
        const bool there = step + u < end && h < part.heads;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          ra[u][s] = rb[u][s] = Raw<TO, V>{};
          xa[u][s] = xb[u][s] = Raw<TI, V>{};
          if (there && slot[s].has_a) {
            ra[u][s].load(g + h * part.d_out.head_stride + slot[s].a);
            if (norm) xa[u][s].load(x + h * part.x.head_stride + slot[s].a);
          }
          if (there && slot[s].has_b) {
            rb[u][s].load(g + h * part.d_out.head_stride + slot[s].b);
            if (norm) xb[u][s].load(x + h * part.x.head_stride + slot[s].b);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t h = (step + u) * per + sub;
        float ga[S][V], gb[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s) {
          ra[u][s].get(ga[s]);
          rb[u][s].get(gb[s]);
          if (slot[s].turned) turn<V>(ga[s], gb[s], cos[s], sin[s], inter);
        }
        if (norm) {
          float va[S][V], vb[S][V], squares = 0.0f;
#pragma unroll
          for (int s = 0; s < S; ++s) {
            xa[u][s].get(va[s]);
            xb[u][s].get(vb[s]);
#pragma unroll
            for (int i = 0; i < V; ++i) squares = fmaf(va[s][i], va[s][i], fmaf(vb[s][i], vb[s][i], squares));
          }
          const float r = __frsqrt_rn(head_sum(squares, lanes) * a.inv_d + a.eps);
          float dot = 0.0f;
#pragma unroll
          for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              va[s][i] *= r;
              vb[s][i] *= r;
              dwa[s][i] = fmaf(ga[s][i], va[s][i], dwa[s][i]);
              dwb[s][i] = fmaf(gb[s][i], vb[s][i], dwb[s][i]);
              ga[s][i] *= wa[s][i];
              gb[s][i] *= wb[s][i];
              dot = fmaf(ga[s][i], va[s][i], fmaf(gb[s][i], vb[s][i], dot));
            }
          dot = head_sum(dot, lanes) * a.inv_d;
#pragma unroll
          for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              ga[s][i] = fmaf(-va[s][i], dot, ga[s][i]) * r;
              gb[s][i] = fmaf(-vb[s][i], dot, gb[s][i]) * r;
            }
        }
        const bool there = step + u < end && h < part.heads;
        TI *row = dx + h * part.dx.head_stride;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          Raw<TI, V> y;
          if (there && slot[s].has_a) {
            y.set(ga[s]);
            y.store(row + slot[s].a);
          }
          if (there && slot[s].has_b) {
            y.set(gb[s]);
            y.store(row + slot[s].b);
          }
        }
      }
    }
  }
  if constexpr (V > 1 && !NORM) return;
  if (!part.dweight) return;
  // over the heads that a warp holds side by side, then over its CTA's warps
#pragma unroll
  for (int s = 0; s < S; ++s)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      for (uint32_t o = 16; o >= lanes; o >>= 1) {
        dwa[s][i] += __shfl_xor_sync(0xffffffffu, dwa[s][i], o);
        dwb[s][i] += __shfl_xor_sync(0xffffffffu, dwb[s][i], o);
      }
      if (sub == 0 && slot[s].has_a) sums[warp][slot[s].a + i] = dwa[s][i];
      if (sub == 0 && slot[s].has_b) sums[warp][slot[s].b + i] = dwb[s][i];
    }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < a.D; d += kThreads) {
    float sum = sums[0][d];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) sum += sums[w][d];
    part.partial[static_cast<size_t>(cta) * a.D + d] = sum;
  }
}

// dweight[d] = the sum of the CTAs' rows: 32 columns a CTA, a warp for every
// 32nd row, then the warps' sums in order.
__global__ void __launch_bounds__(1024) weight_gradient_kernel(const RotaryArgs a) {
  __shared__ float sums[32][33];
  pdl_enter();
  const RotaryPart &part = a.part[blockIdx.y];
  if (!part.dweight) return;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32, d = blockIdx.x * 32 + lane;
  float sum = 0.0f;
  if (d < a.D) {
#pragma unroll 8
    for (uint32_t c = warp; c < part.ctas; c += 32) sum += part.partial[static_cast<size_t>(c) * a.D + d];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  if (warp == 0 && d < a.D) {
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 32; ++w) sum += sums[w][lane];
    part.dweight[d] = sum;
  }
}

template <typename TI, typename TO> void launch_backward(RotaryArgs &a, unsigned grid, cudaStream_t s) {
  constexpr int V = sizeof(TI) == 4 && sizeof(TO) == 4 ? 4 : 8;
  if (!a.vectors) launch_pdl(rotate_backward_kernel<TI, TO, 1, 4, false, false>, grid, kThreads, 0, s, a);
  else if (a.norm) {
    if (a.interleaved) launch_pdl(rotate_backward_kernel<TI, TO, V, 1, true, true>, grid, kThreads, 0, s, a);
    else launch_pdl(rotate_backward_kernel<TI, TO, V, 1, true, false>, grid, kThreads, 0, s, a);
  } else {
    if (a.interleaved) launch_pdl(rotate_backward_kernel<TI, TO, V, 1, false, true>, grid, kThreads, 0, s, a);
    else launch_pdl(rotate_backward_kernel<TI, TO, V, 1, false, false>, grid, kThreads, 0, s, a);
  }
}

}  // namespace
}  // namespace heads
}  // namespace tl

using namespace tl;
using namespace tl::heads;

extern "C" {

size_t tl_rotary_heads_workspace_size(const tl_rotary_desc *d) {
  if (!d || d->D > TL_HEAD_MAX_DIM || (!d->q.dweight && !d->k.dweight)) return 0;
  return (kMaxCtas + 2) * static_cast<size_t>(d->D) * sizeof(float);
}

int tl_rotary_heads_backward(const tl_rotary_desc *desc, void *stream) {
  const char *who = "tl_rotary_heads_backward";
  RotaryArgs a{};
  if (int rc = rotary_args(who, desc, true, a)) return rc;
  const size_t need = tl_rotary_heads_workspace_size(desc);
  if (need && (!desc->workspace || desc->workspace_bytes < need))
    return fail(TL_ERR_INVALID, std::string(who) + ": workspace too small");
  if (reinterpret_cast<uintptr_t>(desc->workspace) % 4)
    return fail(TL_ERR_INVALID, std::string(who) + ": workspace not aligned");
  cudaStream_t s = as_stream(stream);
  if (a.tokens == 0) {
    // an empty sum
    for (const tl_rotary_part *p : {&desc->q, &desc->k})
      if (p->heads && p->dweight)
        if (int rc = check_cuda(cudaMemsetAsync(p->dweight, 0, desc->D * sizeof(float), s), who)) return rc;
    return TL_OK;
  }
  const unsigned grid = share_out(a, true);
  a.part[0].partial = static_cast<float *>(desc->workspace);
  a.part[1].partial = a.part[0].partial + static_cast<size_t>(a.part[0].ctas) * a.D;
#define L(TI, TO) launch_backward<TI, TO>(a, grid, s)
  TL_BY_TYPES(desc->type, desc->out_type, L)
#undef L
  if (int rc = launch_status(who)) return rc;
  if (!need) return TL_OK;
  launch_pdl(weight_gradient_kernel, dim3((a.D + 31) / 32, 2), 1024, 0, s, a);
  return launch_status(who);
}

}  // extern "C"
