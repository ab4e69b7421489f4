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

constexpr int kGradientRows = 2;  // head rows a lane

template <typename TI, typename TO, int V, int S, int U, bool NORM, bool INTER>
__global__ void __launch_bounds__(kThreads, NORM || V == 1 ? 3 : 4) rotate_backward_kernel(const RotaryArgs a) {
  __shared__ float sums[kWarps][TL_HEAD_MAX_DIM];
  pdl_enter();
  const bool second = blockIdx.x >= a.part[0].ctas;
  const RotaryPart &part = a.part[second];
  const uint32_t cta = blockIdx.x - (second ? a.part[0].ctas : 0);
  const bool inter = V == 1 ? a.interleaved : INTER;
  const bool norm = V == 1 ? a.norm : NORM;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint32_t lanes = a.lanes, at = lane & (lanes - 1), sub = lane / lanes, per = 32 / lanes;
  // this part's groups only
  const uint64_t first_groups = static_cast<uint64_t>(a.tokens) * a.part[0].chunks;
  const uint64_t groups = second ? first_groups + static_cast<uint64_t>(a.tokens) * a.part[1].chunks : first_groups;
  const uint64_t warps = static_cast<uint64_t>(part.ctas) * kWarps;

  Slot slot[S];
  float wa[S][V], wb[S][V], dwa[S][V], dwb[S][V];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    slot[s] = slot_of(at + s * lanes, V, a.D, a.rotary, inter);
    load_weights<V>(norm ? part.weight : nullptr, slot[s], wa[s], wb[s]);
#pragma unroll
    for (int i = 0; i < V; ++i) dwa[s][i] = dwb[s][i] = 0.0f;
  }
  struct Rows {
    HeadRows<TO, V, S, U> g;
    HeadRows<TI, V, S, U> x;
  };
  const auto load = [&](Rows &r, const Batch &s) {
    const uint32_t left = s.end > s.head + sub ? s.end - s.head - sub : 0;
    r.g.load(static_cast<const TO *>(part.d_out.p) + place(part.d_out, s, sub), per * part.d_out.head_stride, slot, left, per);
    if (norm) r.x.load(static_cast<const TI *>(part.x.p) + place(part.x, s, sub), per * part.x.head_stride, slot, left, per);
  };
  Batch s;
  s.group = (second ? first_groups : 0) + static_cast<uint64_t>(cta) * kWarps + warp;
  set_batch(a, s, first_groups, groups);
  Rows rows, next_rows;
  if (s.any) load(rows, s);
  uint64_t turned = ~0ull;
  float cos[S][V], sin[S][V];
  while (s.any) {
    Batch n = s;
    next_batch(a, n, U * per, warps, first_groups, groups);
    if (n.any) load(next_rows, n);
    if (s.group != turned) {
      turned = s.group;
      angles<V, S>(a.frequencies, s.position, a.magnitude, at, lanes, a.rotary, cos, sin);
#pragma unroll
      for (int i = 0; i < S; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) sin[i][e] = -sin[i][e];
    }
    TI *const dx = static_cast<TI *>(const_cast<void *>(part.dx.p)) + place(part.dx, s, sub);
    const uint32_t left = s.end > s.head + sub ? s.end - s.head - sub : 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float ga[S][V], gb[S][V], va[S][V], vb[S][V], both[2] = {0.0f, 0.0f};  // sum x^2, sum g w x
#pragma unroll
      for (int i = 0; i < S; ++i) {
        rows.g.a[u][i].get(ga[i]);
        rows.g.b[u][i].get(gb[i]);
        if (slot[i].turned) turn<V>(ga[i], gb[i], cos[i], sin[i], inter);
        if (norm) {
          rows.x.a[u][i].get(va[i]);
          rows.x.b[u][i].get(vb[i]);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            both[0] = fmaf(va[i][e], va[i][e], fmaf(vb[i][e], vb[i][e], both[0]));
            both[1] = fmaf(ga[i][e] * wa[i][e], va[i][e], fmaf(gb[i][e] * wb[i][e], vb[i][e], both[1]));
          }
        }
      }
      if (norm) {
        head_sums<2>(both, lanes);
        const float r = rsqrtf(fmaf(both[0], a.inv_d, a.eps)), dot = both[1] * r * a.inv_d;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            va[i][e] *= r;
            vb[i][e] *= r;
            dwa[i][e] = fmaf(ga[i][e], va[i][e], dwa[i][e]);
            dwb[i][e] = fmaf(gb[i][e], vb[i][e], dwb[i][e]);
            ga[i][e] = fmaf(-va[i][e], dot, ga[i][e] * wa[i][e]) * r;
            gb[i][e] = fmaf(-vb[i][e], dot, gb[i][e] * wb[i][e]) * r;
          }
      }
#pragma unroll
      for (int i = 0; i < S; ++i) {
        Raw<TI, V> y;
        if (u * per < left && slot[i].has_a) {
          y.set(ga[i]);
          y.store(dx + u * (per * part.dx.head_stride) + slot[i].a);
        }
        if (u * per < left && slot[i].has_b) {
          y.set(gb[i]);
          y.store(dx + u * (per * part.dx.head_stride) + slot[i].b);
        }
      }
    }
    s = n;
    rows = next_rows;
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

template <typename TI, typename TO> void launch_backward(const RotaryArgs &a, unsigned grid, cudaStream_t s) {
  constexpr int V = vector_of(sizeof(TI), sizeof(TO)), U = kGradientRows;
  if (!a.vectors) launch_pdl(rotate_backward_kernel<TI, TO, 1, 4, 1, false, false>, grid, kThreads, 0, s, a);
  else if (a.norm) {
    if (a.interleaved) launch_pdl(rotate_backward_kernel<TI, TO, V, 1, U, true, true>, grid, kThreads, 0, s, a);
    else launch_pdl(rotate_backward_kernel<TI, TO, V, 1, U, true, false>, grid, kThreads, 0, s, a);
  } else {
    if (a.interleaved) launch_pdl(rotate_backward_kernel<TI, TO, V, 1, U, false, true>, grid, kThreads, 0, s, a);
    else launch_pdl(rotate_backward_kernel<TI, TO, V, 1, U, false, false>, grid, kThreads, 0, s, a);
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
  const unsigned grid = share_out(a, a.vectors ? kGradientRows : 1, true);
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
