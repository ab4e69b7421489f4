// Distillation of many short rows: a warp per row, the row in registers.
#include "distill_rows.cuh"

namespace tl {
namespace token {
namespace {

// Words of a warp's marks: a bit per token, see vector_marks.
__host__ __device__ constexpr uint32_t mark_words(int nv, int elems) {
  return (nv * 32 * elems + 4 * elems + 31) / 32;
}

// A lane's slots l + 32 i: their ids, values and logits.
template <typename T>
__device__ __forceinline__ void read_slots(const DistillArgs &a, size_t row, const T *z, uint32_t lane,
                                           uint32_t (&id)[kPerLane], SlotLane &l) {
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    id[i] = TL_NO_TOKEN;
    l.u[i] = l.z[i] = -INFINITY;
    if (i * 32 < a.top) read_slot(a, row, lane + 32 * i, id[i], l.u[i]);
    l.slot[i] = id[i] != TL_NO_TOKEN;
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    if (l.slot[i]) l.z[i] = to_float(z[id[i]]);
}

__device__ __forceinline__ uint32_t read_target(const DistillArgs &a, size_t row, uint32_t lane) {
  if (!a.targets) return TL_NO_TOKEN;
  const uint32_t t = a.targets[row];
  if (t < a.vocab) return t;
  if (t != TL_NO_TOKEN && lane == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
  return TL_NO_TOKEN;
}

// The gradient of the row in registers; slots and target, read before, are
// written a second time.
template <typename T, int NV, bool DUAL>
__device__ __forceinline__ void gradient_row(const DistillArgs &a, size_t row, const T *z, const Part &p,
                                             uint32_t lane, const uint4 (&q)[NV], float loose,
                                             const RowStats &r, const uint32_t (&id)[kPerLane],
                                             const SlotLane &l, uint32_t t, float zt, float scale) {
  T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
  const DistillGradient g = distill_gradient<DUAL>(a, r, t, scale);
  const auto fast = [&](float x) { return distill_dz<DUAL>(g, a.c, x); };
  const auto careful = [&](float x) { return careful_distill_dz(g, r, a.c, x); };
  __syncwarp();  // the slots' logits are read: dz may be z
  if (!g.none && !g.far) {
    store_row<T, NV>(dz, p, lane, q, loose, fast);
  } else {
    for (uint32_t j = lane; j < a.vocab; j += 32)
      dz[j] = from_float<T>(g.none ? 0.0f : careful(to_float(z[j])));
  }
  __syncwarp();
  if (g.none) return;
  if (lane == 0 && g.ce != 0.0f) dz[t] = from_float<T>((g.far ? careful(zt) : fast(zt)) - g.ce);
  __syncwarp();  // a target in a slot: the slot's value stands
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    if (l.slot[i]) {
      const float pk = expf(l.u[i] - r.h) * r.b;
      dz[id[i]] = from_float<T>(slot_dz(g, r, a.c, pk, l.z[i], id[i] == t));
    }
}

// As distill_kernel in k_distill.cu, with the row read once: the gradient
// is made from the registers.
template <typename T, int NV, bool TAIL, bool DUAL, bool GRAD>
__global__ void __launch_bounds__(kShortWarps * 32) distill_short_kernel(const DistillArgs a) {
  constexpr int E = Vec<T>::kElems;
  constexpr uint32_t kWords = mark_words(NV, E);
  __shared__ uint32_t all_marks[TAIL ? kShortWarps : 1][kWords];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t *marks = all_marks[TAIL ? warp : 0];
  if (TAIL) {
    for (uint32_t w = lane; w < kWords; w += 32) marks[w] = 0;
    __syncwarp();
  }
  pdl_enter();
  for (size_t row = static_cast<size_t>(blockIdx.x) * kShortWarps + warp; row < a.rows;
       row += static_cast<size_t>(gridDim.x) * kShortWarps) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, 0, 1);
    const uint32_t first = E - p.head;
    uint4 q[NV];
    load_row<T, NV>(z, p, lane, q);
    float loose = lane < p.loose ? to_float(z[loose_at(p, lane)]) : -INFINITY;
    uint32_t id[kPerLane];
    SlotLane l;
    read_slots(a, row, z, lane, id, l);
    const uint32_t t = read_target(a, row, lane);
    const bool target = t != TL_NO_TOKEN && a.ce != 0.0f;
    const float zt = target ? to_float(z[t]) : 0.0f;
    const float scale = GRAD && a.row_scale ? a.row_scale[row] : 1.0f;
    if (TAIL) {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (l.slot[i]) atomicOr(&marks[(id[i] + first) / 32], 1u << ((id[i] + first) % 32));
      __syncwarp();
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i * 32 >= p.end) break;
        const uint32_t m = vector_marks<T>(marks, i * 32 + lane);
        if (m) Vec<T>::drop(q[i], m);
      }
      if (lane < p.loose) {
        const uint32_t j = loose_at(p, lane) + first;
        if (marks[j / 32] >> (j % 32) & 1u) loose = -INFINITY;
      }
    }
    float m = loose;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, Vec<T>::largest(q[i]));
    m = warp_max(m);
    Outside o = {m, 0.0f, 0.0f};
    if (far_out(m, a.c) || far_out(m, kLog2e)) {
      Sums v = empty_sums(), v1 = empty_sums();
      for (uint32_t j = lane; j < a.vocab; j += 32) {
        if (TAIL && marks[(j + first) / 32] >> ((j + first) % 32) & 1u) continue;
        add_logit(v, to_float(z[j]), a.c);
        add_logit(v1, to_float(z[j]), kLog2e);
      }
      o.s = warp_merge(v, a.c).s;
      o.s1 = warp_merge(v1, kLog2e).s;
    } else {
      Pow2Sums v = {shift_of(m, a.c), 0.0f, 0.0f}, v1 = {shift_of(m, kLog2e), 0.0f, 0.0f};
      add_term<false>(v, loose, a.c);
      if (DUAL) add_term<false>(v1, loose, kLog2e);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i * 32 >= p.end) break;
        float f[E];
        Vec<T>::unpack(q[i], f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          add_term<false>(v, f[e], a.c);
          if (DUAL) add_term<false>(v1, f[e], kLog2e);
        }
      }
      o.s = sum_at(warp_sum(v.s), v.n, m, a.c);
      o.s1 = DUAL ? sum_at(warp_sum(v1.s), v1.n, m, kLog2e) : o.s;
    }
    float loss, kl;
    const RowStats r = join_slots<TAIL>(a, l, o, target, zt, loss, kl);
    if (lane == 0) {
      a.loss[row] = loss;
      if (a.kl) a.kl[row] = kl;
      if (a.stats) write_stats(a.stats + row * TL_DISTILL_STATS, r);
    }
    if (TAIL) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (l.slot[i]) marks[(id[i] + first) / 32] = 0;
      __syncwarp();
    }
    if (GRAD) gradient_row<T, NV, DUAL>(a, row, z, p, lane, q, loose, r, id, l, t, zt, scale);
  }
}

template <typename T, int NV, bool DUAL>
__global__ void __launch_bounds__(kShortWarps * 32) distill_backward_short_kernel(const DistillArgs a) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_enter();
  for (size_t row = static_cast<size_t>(blockIdx.x) * kShortWarps + warp; row < a.rows;
       row += static_cast<size_t>(gridDim.x) * kShortWarps) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, 0, 1);
    uint4 q[NV];
    load_row<T, NV>(z, p, lane, q);
    const float loose = lane < p.loose ? to_float(z[loose_at(p, lane)]) : 0.0f;
    const float *st = a.stats + row * TL_DISTILL_STATS;
    const RowStats r = {st[0], st[1], st[2], st[3], st[4], st[5], st[6]};
    uint32_t id[kPerLane];
    SlotLane l;
    read_slots(a, row, z, lane, id, l);
    const uint32_t t = read_target(a, row, lane);
    const float zt = t != TL_NO_TOKEN ? to_float(z[t]) : 0.0f;
    gradient_row<T, NV, DUAL>(a, row, z, p, lane, q, loose, r, id, l, t, zt,
                              a.row_scale ? a.row_scale[row] : 1.0f);
  }
}

template <typename T, int NV, bool TAIL, bool GRAD> void launch(const DistillArgs &a, cudaStream_t s) {
  const unsigned grid = short_grid(a.rows);
  if (dual(a)) launch_pdl(distill_short_kernel<T, NV, TAIL, true, GRAD>, grid, kShortWarps * 32, 0, s, a);
  else launch_pdl(distill_short_kernel<T, NV, TAIL, false, GRAD>, grid, kShortWarps * 32, 0, s, a);
}

template <typename T, int NV>
void launch_forward(const DistillArgs &a, bool tail, bool gradient, cudaStream_t s) {
  if (tail) gradient ? launch<T, NV, true, true>(a, s) : launch<T, NV, true, false>(a, s);
  else gradient ? launch<T, NV, false, true>(a, s) : launch<T, NV, false, false>(a, s);
}

template <typename T, int NV> void launch_backward(const DistillArgs &a, cudaStream_t s) {
  const unsigned grid = short_grid(a.rows);
  if (dual(a)) launch_pdl(distill_backward_short_kernel<T, NV, true>, grid, kShortWarps * 32, 0, s, a);
  else launch_pdl(distill_backward_short_kernel<T, NV, false>, grid, kShortWarps * 32, 0, s, a);
}

}  // namespace

bool distill_short(const DistillArgs &a, int32_t type, bool tail, bool gradient, cudaStream_t s) {
  const uint32_t nv = short_vectors(a.vocab, type_size(type));
  if (!nv || a.rows < kShortRows) return false;
#define L(T) nv == 4 ? launch_forward<T, 4>(a, tail, gradient, s) : launch_forward<T, 16>(a, tail, gradient, s)
  TL_BY_TYPE(type, L)
#undef L
  return true;
}

bool distill_backward_short(const DistillArgs &a, int32_t type, cudaStream_t s) {
  const uint32_t nv = short_vectors(a.vocab, type_size(type));
  if (!nv || a.rows < kShortRows) return false;
#define L(T) nv == 4 ? launch_backward<T, 4>(a, s) : launch_backward<T, 16>(a, s)
  TL_BY_TYPE(type, L)
#undef L
  return true;
}

}  // namespace token
}  // namespace tl
