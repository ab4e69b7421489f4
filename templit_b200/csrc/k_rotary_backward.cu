// Gradient of the rotation and norm of heads (include/templit_cuda.h:
// tl_rotary_heads_backward).  With g = the incoming gradient turned back and
// x^ = x / rms:
//   dw = sum over tokens and heads of g x^
//   dx = (g w - x^ mean(g w x^)) / rms            (norm; else dx = g)
// Bound by memory: d_out and x are read once, dx is written once.  The grid
// stays on the SMs; a CTA adds its heads' weight gradients up in registers,
// then in shared memory, and leaves one row, which a second kernel sums over
// the CTAs in a fixed order.
//
// 16384 x 40 heads of 128 bf16: 118 us (503 MB, 4.25 TB/s); the registers of the norm's sums
// leave 12 warps an SM, too few to cover what each waits for: a warp issues every 5.8 cycles,
// of which 1.6 are its own operands, 1.0 loads and 0.6 shuffles, so that issue (48 %) and
// memory (50 %) are half busy each; the sum of the CTAs' rows is 7 us more.  The rotation alone, a quarter of each head turned, 16384 x 40 heads: 62 us.
#include "rotary.cuh"

namespace tl {
namespace heads {
namespace {

// head rows of a lane's batch, of the norm's gradient and without
constexpr int kNormRows = 1, kPlainRows = 2;
constexpr int kNormCtas = 3;      // CTAs an SM where the norm's gradient takes the registers

template <typename TI, typename TO, int V, int U, bool NORM, bool INTER>
__global__ void __launch_bounds__(kThreads, NORM ? kNormCtas : 4) rotate_backward_kernel(const RotaryArgs a) {
  __shared__ float sums[NORM ? kWarps : 1][TL_HEAD_MAX_DIM];
  pdl_enter();
  const bool second = blockIdx.x >= a.part[0].ctas;
  const RotaryPart &part = a.part[second];
  const uint32_t cta = blockIdx.x - (second ? a.part[0].ctas : 0);
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const uint32_t lanes = a.lanes, at = lane & (lanes - 1), sub = lane / lanes, per = 32 / lanes;
  // this part's groups only
  const uint64_t first_groups = static_cast<uint64_t>(a.tokens) * a.part[0].chunks;
  const uint64_t groups = second ? first_groups + static_cast<uint64_t>(a.tokens) * a.part[1].chunks : first_groups;
  const uint64_t warps = static_cast<uint64_t>(part.ctas) * kWarps;
  const Slot slot = slot_of(at, V, a.D, a.rotary, INTER);
  const uint64_t g_step = per * part.d_out.head_stride, x_step = per * part.x.head_stride, dx_step = per * part.dx.head_stride;
  const auto left_of = [&](const Batch &s) { return s.end > s.head + sub ? s.end - s.head - sub : 0u; };

  Pair wa[V / 2], wb[V / 2], dwa[V / 2], dwb[V / 2];
  {
    float fa[V], fb[V];
    load_weights<V>(NORM ? part.weight : nullptr, slot, fa, fb);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      wa[i] = pair(fa[2 * i], fa[2 * i + 1]);
      wb[i] = pair(fb[2 * i], fb[2 * i + 1]);
      dwa[i] = dwb[i] = 0;
    }
  }
  struct Rows {
    HeadRows<TO, V, U> g;
    HeadRows<TI, V, U> x;
  };
  Batch s;
  s.group = (second ? first_groups : 0) + static_cast<uint64_t>(cta) * kWarps + warp;
  set_batch(a, s, first_groups, groups);
  const TO *g = nullptr;
  const TI *x = nullptr;
  TI *dx = nullptr;
  const auto point = [&](const Batch &n) {
    g = static_cast<const TO *>(part.d_out.p) + place(part.d_out, n, sub);
    if (NORM) x = static_cast<const TI *>(part.x.p) + place(part.x, n, sub);
  };
  const auto load = [&](Rows &r, const Batch &n) {
    r.g.template load<NORM>(g, g_step, slot, left_of(n), per);
    if (NORM) r.x.template load<true>(x, x_step, slot, left_of(n), per);
  };
  Rows even, odd;
  even.g.clear();
  odd.g.clear();
  even.x.clear();
  odd.x.clear();
  if (s.any) {
    point(s);
    load(even, s);
  }
  uint64_t turned = ~0ull;
  Turn<V> turn;
  const auto work = [&](const Rows &rows, Rows &next) {
    Batch n = s;
    if (next_batch(a, n, U * per, warps, first_groups, groups)) {
      g += U * g_step;
      if (NORM) x += U * x_step;
    } else if (n.any) {
      point(n);
    }
    if (n.any) load(next, n);
    if (s.group != turned) {
      turned = s.group;
      float cos[V], sin[V];
      angles<V>(a.frequencies, s.position, a.magnitude, at, lanes, a.rotary, cos, sin);
#pragma unroll
      for (int i = 0; i < V; ++i) sin[i] = -sin[i];
      turn.set(cos, sin, INTER);
      dx = static_cast<TI *>(const_cast<void *>(part.dx.p)) + place(part.dx, s, sub);
    }
    Pair ga[U][V / 2], gb[U][V / 2];
    float both[2 * U];  // sum x^2, sum g w x
#pragma unroll
    for (int u = 0; u < U; ++u) {
      get_pairs(rows.g.a[u], ga[u]);
      get_pairs(rows.g.b[u], gb[u]);
      turn.apply(ga[u], gb[u], slot.turned, INTER);
      if (NORM) {
        Pair va[V / 2], vb[V / 2], xx = 0, gx = 0;
        get_pairs(rows.x.a[u], va);
        get_pairs(rows.x.b[u], vb);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          xx = fma2(va[i], va[i], fma2(vb[i], vb[i], xx));
          gx = fma2(mul2(ga[u][i], wa[i]), va[i], fma2(mul2(gb[u][i], wb[i]), vb[i], gx));
        }
        both[2 * u] = sum2(xx);
        both[2 * u + 1] = sum2(gx);
      }
    }
    if (NORM) head_sums<2 * U>(both, lanes);
    const uint32_t left = left_of(s);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (NORM) {
        float r = rsqrtf(fmaf(both[2 * u], a.inv_d, a.eps));
        if (s.head + sub + u * per >= s.end) r = 0.0f;  // not there: the norm of its zeros is none without an eps
        const float dot = -(both[2 * u + 1] * r * a.inv_d) * r;
        const Pair r2 = pair(r, r), dot2 = pair(dot, dot);
        Pair va[V / 2], vb[V / 2];
        get_pairs(rows.x.a[u], va);
        get_pairs(rows.x.b[u], vb);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          va[i] = mul2(va[i], r2);
          vb[i] = mul2(vb[i], r2);
          dwa[i] = fma2(ga[u][i], va[i], dwa[i]);
          dwb[i] = fma2(gb[u][i], vb[i], dwb[i]);
          // (g w - x^ mean(g w x^)) / rms
          ga[u][i] = fma2(va[i], dot2, mul2(mul2(ga[u][i], wa[i]), r2));
          gb[u][i] = fma2(vb[i], dot2, mul2(mul2(gb[u][i], wb[i]), r2));
        }
      }
      Raw<TI, V> y;
      if (u * per < left && slot.has_a) {
        set_pairs(y, ga[u]);
        y.store(dx + u * dx_step + slot.a);
      }
      if (u * per < left && slot.has_b) {
        set_pairs(y, gb[u]);
        y.store(dx + u * dx_step + slot.b);
      }
    }
    dx += U * dx_step;
    s = n;
    return n.any;
  };
  if (s.any)
    while (work(even, odd) && work(odd, even)) {
    }
  if constexpr (NORM) {
    if (!part.dweight) return;
    // over the heads that a warp holds side by side, then over its CTA's warps
    float da[V], db[V];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 p = halves(dwa[i]), q = halves(dwb[i]);
      da[2 * i] = p.x, da[2 * i + 1] = p.y, db[2 * i] = q.x, db[2 * i + 1] = q.y;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      for (uint32_t o = 16; o >= lanes; o >>= 1) {
        da[i] += __shfl_xor_sync(0xffffffffu, da[i], o);
        db[i] += __shfl_xor_sync(0xffffffffu, db[i], o);
      }
      if (sub == 0 && slot.has_a) sums[warp][slot.a + i] = da[i];
      if (sub == 0 && slot.has_b) sums[warp][slot.b + i] = db[i];
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < a.D; d += kThreads) {
      float sum = sums[0][d];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) sum += sums[w][d];
      part.partial[static_cast<size_t>(cta) * a.D + d] = sum;
    }
  }
}

// The same by single elements, a warp a head; the CTA's heads are of one part.
template <typename TI, typename TO> __global__ void __launch_bounds__(kThreads) rotate_backward_elements_kernel(const RotaryArgs a) {
  constexpr int S = TL_HEAD_MAX_DIM / 64;
  __shared__ float sums[kWarps][TL_HEAD_MAX_DIM];
  pdl_enter();
  const bool second = blockIdx.x >= a.part[0].ctas;
  const RotaryPart &part = a.part[second];
  const uint32_t cta = blockIdx.x - (second ? a.part[0].ctas : 0), lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  float dwa[S] = {}, dwb[S] = {};
  const uint64_t items = static_cast<uint64_t>(a.tokens) * part.heads, warps = static_cast<uint64_t>(part.ctas) * kWarps;
  for (uint64_t item = static_cast<uint64_t>(cta) * kWarps + warp; item < items; item += warps) {
    const uint32_t token = static_cast<uint32_t>(item / part.heads), h = static_cast<uint32_t>(item - static_cast<uint64_t>(token) * part.heads);
    const uint32_t b = token / a.T, t = token - b * a.T, position = a.positions ? a.positions[token] : a.first_position + t;
    const auto row = [&](const tl_head_view &v) { return b * v.batch_stride + t * v.row_stride + h * v.head_stride; };
    const TO *g = static_cast<const TO *>(part.d_out.p) + row(part.d_out);
    const TI *x = a.norm ? static_cast<const TI *>(part.x.p) + row(part.x) : nullptr;
    TI *dx = static_cast<TI *>(const_cast<void *>(part.dx.p)) + row(part.dx);
    float ga[S], gb[S], va[S] = {}, vb[S] = {}, both[2] = {0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const Slot slot = slot_of(lane + 32 * s, 1, a.D, a.rotary, a.interleaved);
      ga[s] = slot.has_a ? element_of(g[slot.a]) : 0.0f;
      gb[s] = slot.has_b ? element_of(g[slot.b]) : 0.0f;
      if (slot.turned) {
        float sn, cs;
        sine_cosine(position * a.frequencies[lane + 32 * s], sn, cs);
        const float c = cs * a.magnitude, n = sn * a.magnitude, u = ga[s];
        ga[s] = fmaf(u, c, gb[s] * n);
        gb[s] = fmaf(gb[s], c, -(u * n));
      }
      if (a.norm) {
        va[s] = slot.has_a ? element_of(x[slot.a]) : 0.0f;
        vb[s] = slot.has_b ? element_of(x[slot.b]) : 0.0f;
        const float w = part.weight && slot.has_a ? part.weight[slot.a] : 1.0f, v = part.weight && slot.has_b ? part.weight[slot.b] : 1.0f;
        both[0] = fmaf(va[s], va[s], fmaf(vb[s], vb[s], both[0]));
        both[1] = fmaf(ga[s] * w, va[s], fmaf(gb[s] * v, vb[s], both[1]));
      }
    }
    if (a.norm) head_sums<2>(both, 32);
    const float r = a.norm ? rsqrtf(fmaf(both[0], a.inv_d, a.eps)) : 1.0f, dot = both[1] * r * a.inv_d;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const Slot slot = slot_of(lane + 32 * s, 1, a.D, a.rotary, a.interleaved);
      if (a.norm) {
        const float w = part.weight && slot.has_a ? part.weight[slot.a] : 1.0f, v = part.weight && slot.has_b ? part.weight[slot.b] : 1.0f;
        va[s] *= r;
        vb[s] *= r;
        dwa[s] = fmaf(ga[s], va[s], dwa[s]);
        dwb[s] = fmaf(gb[s], vb[s], dwb[s]);
        ga[s] = fmaf(-va[s], dot, ga[s] * w) * r;
        gb[s] = fmaf(-vb[s], dot, gb[s] * v) * r;
      }
      if (slot.has_a) set_element(dx[slot.a], ga[s]);
      if (slot.has_b) set_element(dx[slot.b], gb[s]);
    }
  }
  if (!part.dweight) return;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const Slot slot = slot_of(lane + 32 * s, 1, a.D, a.rotary, a.interleaved);
    if (slot.has_a) sums[warp][slot.a] = dwa[s];
    if (slot.has_b) sums[warp][slot.b] = dwb[s];
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
  constexpr int V = vector_of(sizeof(TI), sizeof(TO)), U = kPlainRows, N = kNormRows;
  if (!a.vectors) launch_pdl(rotate_backward_elements_kernel<TI, TO>, grid, kThreads, 0, s, a);
  else if (a.norm) {
    if (a.interleaved) launch_pdl(rotate_backward_kernel<TI, TO, V, N, true, true>, grid, kThreads, 0, s, a);
    else launch_pdl(rotate_backward_kernel<TI, TO, V, N, true, false>, grid, kThreads, 0, s, a);
  } else {
    if (a.interleaved) launch_pdl(rotate_backward_kernel<TI, TO, V, U, false, true>, grid, kThreads, 0, s, a);
    else launch_pdl(rotate_backward_kernel<TI, TO, V, U, false, false>, grid, kThreads, 0, s, a);
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
  const unsigned grid = share_out(a, !a.vectors ? 1 : a.norm ? kNormRows : kPlainRows, kNumSMs * (a.vectors && a.norm ? kNormCtas : 4), true);
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
