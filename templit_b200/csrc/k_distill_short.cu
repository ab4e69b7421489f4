// Distillation of many short rows: a warp per row, the row in shared memory.
#include "distill_rows.cuh"

namespace tl {
namespace token {
namespace {

// A lane's slots l + 32 i: their ids and values.
__device__ __forceinline__ void read_slots(const DistillArgs &a, size_t row, uint32_t lane,
                                           uint32_t (&id)[kPerLane], SlotLane &l) {
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    id[i] = TL_NO_TOKEN;
    l.u[i] = l.z[i] = -INFINITY;
    if (i * 32 < a.top) read_slot(a, row, lane + 32 * i, id[i], l.u[i]);
    l.slot[i] = id[i] != TL_NO_TOKEN;
  }
}

// A logit of the row whose vectors are in shared memory.
template <typename T>
__device__ __forceinline__ float logit_at(const T *z, const Part &p, const uint4 *buffer, uint32_t j) {
  return to_float(j >= p.head && j < p.tail ? reinterpret_cast<const T *>(buffer)[j - p.head] : z[j]);
}

__device__ __forceinline__ uint32_t read_target(const DistillArgs &a, size_t row, uint32_t lane) {
  if (!a.targets) return TL_NO_TOKEN;
  const uint32_t t = a.targets[row];
  if (t < a.vocab) return t;
  if (t != TL_NO_TOKEN && lane == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
  return TL_NO_TOKEN;
}

// The gradient of the row in shared memory; slots and target, read before,
// are written a second time, after `next`: the buffer is free then.
template <typename T, int NV, bool DUAL, typename F>
__device__ __forceinline__ void gradient_row(const DistillArgs &a, size_t row, const T *z, const Part &p,
                                             uint32_t lane, const uint4 *buffer, float loose,
                                             const RowStats &r, const uint32_t (&id)[kPerLane],
                                             const SlotLane &l, uint32_t t, float zt, float scale,
                                             F next) {
  T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
  const DistillGradient g = distill_gradient<DUAL>(a, r, t, scale);
  const Pair c2 = pair(a.c, a.c);
  const auto fast = [&](float x) { return distill_dz<DUAL>(g, a.c, x); };
  const auto fast2 = [&](Pair x) { return distill_dz2<DUAL>(g, c2, x); };
  const auto careful = [&](float x) { return careful_distill_dz(g, r, a.c, x); };
  if (!g.none && !g.far) {
    write_row<T, NV>(dz, p, lane, buffer, loose, fast2, fast);
  } else {
    for (uint32_t j = lane; j < a.vocab; j += 32)
      dz[j] = from_float<T>(g.none ? 0.0f : careful(to_float(z[j])));
  }
  __syncwarp();
  next();
  if (g.none) return;
  if (lane == 0 && g.ce != 0.0f) dz[t] = from_float<T>((g.far ? careful(zt) : fast(zt)) - g.ce);
  __syncwarp();  // a target in a slot: the slot's value stands
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    if (i * 32 >= a.top) break;
    if (l.slot[i]) {
      const float pk = expf(l.u[i] - r.h) * r.b;
      dz[id[i]] = from_float<T>(slot_dz(g, r, a.c, pk, l.z[i], id[i] == t));
    }
  }
}

// As distill_kernel in k_distill.cu, with the row read once.  The slots'
// logits are taken out of the row in shared memory (TAIL): no marks.  12288 x
// 2048 fp32, 32 slots, tail and targets: 25 us for the loss, 42 to 44 with the
// gradient (4.7 to 4.9 TB/s; four exponentials a logit keep their unit 57 %
// busy, the rest is 24 warps an SM waiting for their own steps); in registers,
// 67 us.
template <typename T, int NV, bool TAIL, bool DUAL, bool GRAD>
__global__ void __launch_bounds__(kShortWarps * 32) distill_short_kernel(const DistillArgs a) {
  extern __shared__ uint4 shared[];
  constexpr int E = Vec<T>::kElems;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4 *buffer = shared + warp * NV * 32;
  const size_t stride = static_cast<size_t>(gridDim.x) * kShortWarps;
  const auto stage = [&](size_t row) {
    if (row >= a.rows) return;
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    stage_row<T, NV>(z, part_of(z, a.vocab, 0, 1), lane, buffer);
  };
  pdl_enter();
  size_t row = static_cast<size_t>(blockIdx.x) * kShortWarps + warp;
  stage(row);
  for (; row < a.rows; row += stride) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, 0, 1);
    float loose = lane < p.loose ? to_float(z[loose_at(p, lane)]) : -INFINITY;
    uint32_t id[kPerLane];
    SlotLane l;
    read_slots(a, row, lane, id, l);
    const uint32_t t = read_target(a, row, lane);
    const bool target = t != TL_NO_TOKEN && a.ce != 0.0f;
    const float scale = GRAD && a.row_scale ? a.row_scale[row] : 1.0f;
    await_row();
    const float zt = target ? logit_at(z, p, buffer, t) : 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (l.slot[i]) l.z[i] = logit_at(z, p, buffer, id[i]);
    if (TAIL) {
      __syncwarp();  // all of them are read
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (l.slot[i] && id[i] >= p.head && id[i] < p.tail)
          reinterpret_cast<T *>(buffer)[id[i] - p.head] = from_float<T>(-INFINITY);
      if (p.loose) {
        uint32_t taken = 0;  // a bit per loose logit
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
          if (l.slot[i] && (id[i] < p.head || id[i] >= p.tail))
            taken |= 1u << (id[i] < p.head ? id[i] : p.head + (id[i] - p.tail));
        if (__reduce_or_sync(0xffffffffu, taken) >> lane & 1u) loose = -INFINITY;
      }
      __syncwarp();
    }
    float m = loose;
    for_vectors<NV>(p.end, lane, [&](int, uint32_t j) { m = fmaxf(m, Vec<T>::largest(buffer[j])); });
    m = warp_max(m);
    Outside o = {m, 0.0f, 0.0f};
    if (far_out(m, a.c) || far_out(m, kLog2e)) {
      Sums v = empty_sums(), v1 = empty_sums();
      add_logit(v, loose, a.c);
      add_logit(v1, loose, kLog2e);
      for (uint32_t j = lane; j < p.end * E; j += 32) {
        const float x = to_float(reinterpret_cast<const T *>(buffer)[j]);
        add_logit(v, x, a.c);
        add_logit(v1, x, kLog2e);
      }
      o.s = warp_merge(v, a.c).s;
      o.s1 = warp_merge(v1, kLog2e).s;
    } else {
      Pow2Sums v = {shift_of(m, a.c), 0.0f, 0.0f}, v1 = {shift_of(m, kLog2e), 0.0f, 0.0f};
      add_term<false>(v, loose, a.c);
      if (DUAL) add_term<false>(v1, loose, kLog2e);
      const Pair c2 = pair(a.c, a.c), n2 = pair(-v.n, -v.n);
      const Pair c21 = pair(kLog2e, kLog2e), n21 = pair(-v1.n, -v1.n);
      Pair s = pair(v.s, 0.0f), s1 = pair(v1.s, 0.0f);
      for_vectors<NV>(p.end, lane, [&](int, uint32_t j) {
        Pair f[E / 2];
        Vec<T>::pairs(buffer[j], f);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          s = add2(s, ex2_pair(fma2(f[e], c2, n2)));
          if (DUAL) s1 = add2(s1, ex2_pair(fma2(f[e], c21, n21)));
        }
      });
      const float2 y = halves(s), y1 = halves(s1);
      o.s = sum_at(warp_sum(y.x + y.y), v.n, m, a.c);
      o.s1 = DUAL ? sum_at(warp_sum(y1.x + y1.y), v1.n, m, kLog2e) : o.s;
    }
    float loss, kl;
    const RowStats r = join_slots<TAIL>(a, l, o, target, zt, loss, kl);
    if (lane == 0) {
      a.loss[row] = loss;
      if (a.kl) a.kl[row] = kl;
      if (a.stats) write_stats(a.stats + row * TL_DISTILL_STATS, r);
    }
    if constexpr (GRAD) {
      gradient_row<T, NV, DUAL>(a, row, z, p, lane, buffer, loose, r, id, l, t, zt, scale,
                                [&] { stage(row + stride); });
    } else {
      __syncwarp();  // the buffer is free
      stage(row + stride);
    }
  }
}

template <typename T, int NV, bool DUAL>
__global__ void __launch_bounds__(kShortWarps * 32) distill_backward_short_kernel(const DistillArgs a) {
  extern __shared__ uint4 shared[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4 *buffer = shared + warp * NV * 32;
  const size_t stride = static_cast<size_t>(gridDim.x) * kShortWarps;
  const auto stage = [&](size_t row) {
    if (row >= a.rows) return;
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    stage_row<T, NV>(z, part_of(z, a.vocab, 0, 1), lane, buffer);
  };
  pdl_enter();
  size_t row = static_cast<size_t>(blockIdx.x) * kShortWarps + warp;
  stage(row);
  for (; row < a.rows; row += stride) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, 0, 1);
    const float loose = lane < p.loose ? to_float(z[loose_at(p, lane)]) : 0.0f;
    const float *st = a.stats + row * TL_DISTILL_STATS;
    const RowStats r = {st[0], st[1], st[2], st[3], st[4], st[5], st[6], st[7]};
    uint32_t id[kPerLane];
    SlotLane l;
    read_slots(a, row, lane, id, l);
    const uint32_t t = read_target(a, row, lane);
    const float scale = a.row_scale ? a.row_scale[row] : 1.0f;
    await_row();
    const float zt = t != TL_NO_TOKEN ? logit_at(z, p, buffer, t) : 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (l.slot[i]) l.z[i] = logit_at(z, p, buffer, id[i]);
    __syncwarp();  // loose logits among them are read: dz may be z
    gradient_row<T, NV, DUAL>(a, row, z, p, lane, buffer, loose, r, id, l, t, zt, scale,
                              [&] { stage(row + stride); });
  }
}

template <typename K> void launch_short(K kernel, const DistillArgs &a, int nv, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(nv) * 512 * kShortWarps;
  if (smem > 48 * 1024)  // a failure shows in the launch's status
    (void)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_pdl(kernel, short_grid(a.rows, kShortWarps, smem), kShortWarps * 32, smem, s, a);
}

template <typename T, int NV, bool TAIL, bool GRAD> void launch(const DistillArgs &a, cudaStream_t s) {
  if (dual(a)) launch_short(distill_short_kernel<T, NV, TAIL, true, GRAD>, a, NV, s);
  else launch_short(distill_short_kernel<T, NV, TAIL, false, GRAD>, a, NV, s);
}

template <typename T, int NV>
void launch_forward(const DistillArgs &a, bool tail, bool gradient, cudaStream_t s) {
  if (tail) gradient ? launch<T, NV, true, true>(a, s) : launch<T, NV, true, false>(a, s);
  else gradient ? launch<T, NV, false, true>(a, s) : launch<T, NV, false, false>(a, s);
}

template <typename T, int NV> void launch_backward(const DistillArgs &a, cudaStream_t s) {
  if (dual(a)) launch_short(distill_backward_short_kernel<T, NV, true>, a, NV, s);
  else launch_short(distill_backward_short_kernel<T, NV, false>, a, NV, s);
}

}  // namespace

bool distill_short(const DistillArgs &a, int32_t type, bool tail, bool gradient, cudaStream_t s) {
  const uint32_t nv = short_vectors(a.rows, a.vocab, type_size(type));
  if (!nv) return false;
#define L(T)                                            \
  nv == 4 ? launch_forward<T, 4>(a, tail, gradient, s)  \
          : nv == 16 ? launch_forward<T, 16>(a, tail, gradient, s) : launch_forward<T, 32>(a, tail, gradient, s)
  TL_BY_TYPE(type, L)
#undef L
  return true;
}

bool distill_backward_short(const DistillArgs &a, int32_t type, cudaStream_t s) {
  const uint32_t nv = short_vectors(a.rows, a.vocab, type_size(type));
  if (!nv) return false;
#define L(T) nv == 4 ? launch_backward<T, 4>(a, s) : nv == 16 ? launch_backward<T, 16>(a, s) : launch_backward<T, 32>(a, s)
  TL_BY_TYPE(type, L)
#undef L
  return true;
}

}  // namespace token
}  // namespace tl
