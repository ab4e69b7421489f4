// Distillation from a teacher's top tokens: loss rows, their gradient, and
// both in one call (tl_distill_rows, tl_distill_backward_rows,
// tl_distill_train_rows).
#include "distill_rows.cuh"

#include <cooperative_groups.h>

namespace tl {
namespace token {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;  // vectors of a thread in flight
// The gradient's second pass finds a row in L2 only as far as L2 holds the
// rows that all CTAs have under way (a little under half of its 126 MB, next
// to the gradients).  Above kL2Again bytes of them the pass goes backwards
// and lets go of what it touches; above kL2Wide CTAs of twice the threads
// have half as many rows under way.  Measured, bf16, 256 forwards, 256
// backwards, 512 backwards: 12000 x 32768 (39 MB under way) 336, 346, 454
// us; 10000 x 40000 (47 MB) 346, 341, 453; 8192 x 65536 (78 MB) 495, 440,
// 486; 4096 x 128000 (151 MB) 496, 461, 437.
constexpr size_t kL2Again = 44 << 20, kL2Wide = 110 << 20;

// The gradient of one row's part.  Thread k < top has slot k: id
// (TL_NO_TOKEN if empty or in another part), its p and its logit, read
// before anything is written (dlogits may be logits); `target_here` has the
// target's logit zt in the thread that writes it.  The slots and the target
// are written a second time.
template <int THREADS, bool AGAIN, bool WHOLE, bool DUAL, typename T>
__device__ __forceinline__ void gradient_part(const DistillArgs &a, size_t row, const T *z,
                                              const Part &part, const RowStats &r, uint32_t id,
                                              float p, float zk, uint32_t t, bool target_here,
                                              float zt) {
  T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
  const DistillGradient g = distill_gradient<DUAL>(a, r, t, a.row_scale ? a.row_scale[row] : 1.0f);
  const auto fast = [&](float x) { return distill_dz<DUAL>(g, a.c, x); };
  const Pair c2 = pair(a.c, a.c);
  const auto fast2 = [&](Pair x) { return distill_dz2<DUAL>(g, c2, x); };
  const auto careful = [&](float x) { return careful_distill_dz(g, r, a.c, x); };
  // before the pass over the row: fewer registers to keep through it
  const float at_slot = id != TL_NO_TOKEN ? slot_dz(g, r, a.c, p, zk, id == t) : 0.0f;
  const float at_target = target_here && g.ce != 0.0f ? (g.far ? careful(zt) : fast(zt)) - g.ce : 0.0f;
  if (g.none) write_elements<THREADS>(z, dz, part, [](float) { return 0.0f; });
  else if (g.far) write_elements<THREADS>(z, dz, part, careful);
  else write_vectors<THREADS, kBatch, AGAIN, WHOLE>(z, dz, part, fast2, fast);
  __syncthreads();
  if (g.none) return;
  if (target_here && g.ce != 0.0f) dz[t] = from_float<T>(at_target);
  __syncthreads();  // a target in a slot: the slot's value stands
  if (id != TL_NO_TOKEN) dz[id] = from_float<T>(at_slot);
}

// Slot k of a row in thread k.
__device__ __forceinline__ void read_slot(const DistillArgs &a, size_t row, uint32_t &id, float &u) {
  read_slot(a, row, threadIdx.x, id, u);
}

__device__ __forceinline__ uint32_t read_target(const DistillArgs &a, size_t row) {
  if (!a.targets) return TL_NO_TOKEN;
  const uint32_t t = a.targets[row];
  if (t < a.vocab) return t;
  if (t != TL_NO_TOKEN && threadIdx.x == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
  return TL_NO_TOKEN;
}

template <int THREADS> struct DistillShared {
  static constexpr int kWarps = THREADS / 32;
  Sums scratch[kWarps];
  Pow2Sums sums[kMaxCluster * kWarps], sums1[kMaxCluster * kWarps];
  float largest[kMaxCluster * kWarps];
  bool slot[TL_TOKEN_MAX_TOP];
  float u[TL_TOKEN_MAX_TOP], z[TL_TOKEN_MAX_TOP];
  float zt;
  RowStats r;
};

// The sums outside the slots by add_logit, for rows that Pow2Sums cannot
// hold.
template <int THREADS, bool TAIL, typename T>
__device__ __noinline__ Outside careful_outside(const T *z, uint32_t vocab, float c, bool target,
                                                const uint32_t *marks, uint32_t first, Sums *scratch) {
  Sums v = empty_sums(), v1 = empty_sums();
  for (uint32_t j = threadIdx.x; j < vocab; j += THREADS) {
    if (TAIL && marks[(j + first) / 32] >> ((j + first) % 32) & 1u) continue;
    const float x = to_float(z[j]);
    add_logit(v, x, c);
    if (target) add_logit(v1, x, kLog2e);
  }
  v = block_merge<THREADS / 32>(v, c, scratch);
  v1 = block_merge<THREADS / 32>(v1, kLog2e, scratch);
  return {v.m, v.s, v1.s};
}

// One CTA per row, or a cluster of CTAs that share a row.  The slots'
// tokens are marked by a bit each in shared memory (TAIL; a vector's bits are
// one byte to look at), one pass over the row sums the others, a warp joins
// the slots to the sums, and with GRAD a second pass, out of L2 as far as it
// holds the row (AGAIN), writes the gradient.  DUAL: the target's term has
// sums of its own, at temperature 1.  4096 x 128000 bf16, 64 slots, tail: the
// loss 188 us (5.6 TB/s; 173 for a few calls at full clock), with the
// gradient 451 us (4.7 TB/s of one read and one write, 431 at full clock; DRAM
// moves 8 % more).
template <typename T, int THREADS, bool TAIL, bool DUAL, bool GRAD, bool AGAIN, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, THREADS > kThreads ? 2 : GRAD ? 4 : 5) distill_kernel(const DistillArgs a) {
  extern __shared__ uint32_t marks[];
  __shared__ DistillShared<THREADS> sh;
  constexpr uint32_t kWarps = THREADS / 32;
  constexpr uint32_t E = Vec<T>::kElems;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts = CLUSTER ? cluster.num_blocks() : 1, part = CLUSTER ? cluster.block_rank() : 0;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const auto everyone = [&] {
    if (CLUSTER) cluster.sync();
    else __syncthreads();
  };
  if (TAIL)
    for (uint32_t w = tid; w < (a.vocab + 2 * E + 31) / 32; w += THREADS) marks[w] = 0;
  everyone();  // every CTA of the cluster runs; the marks are clear
  pdl_enter();
  for (size_t row = blockIdx.x / parts; row < a.rows; row += gridDim.x / parts) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, part, parts);
    const uint32_t first = E - p.head;
    uint32_t id;
    float u;
    read_slot(a, row, id, u);
    if (TAIL) {
      if (id != TL_NO_TOKEN) atomicOr(&marks[(id + first) / 32], 1u << ((id + first) % 32));
      __syncthreads();
    }
    const float zk = id != TL_NO_TOKEN ? to_float(z[id]) : -INFINITY;
    const uint32_t t = read_target(a, row);
    const bool target = t != TL_NO_TOKEN && a.ce != 0.0f;
    const float zt = target && tid == 0 ? to_float(z[t]) : 0.0f;
    const uint4 *vec = reinterpret_cast<const uint4 *>(z + p.head);
    Pow2Sums v = {-kFar, 0.0f, 0.0f}, v1 = v;
    float largest = -INFINITY;
    const auto add = [&](auto full, uint32_t at) {  // full: no vector of the batch is past the end
      uint4 q[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t j = at + i * THREADS + tid;
        q[i] = full || j < p.end ? vec[j] : make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
      }
      if (TAIL) {
        uint32_t m[kBatch], some = 0;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const uint32_t j = at + i * THREADS + tid;
          m[i] = full || j < p.end ? vector_marks<T>(marks, j) : 0;
          some |= m[i];
        }
        if (some) {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) Vec<T>::drop(q[i], m[i]);
        }
      }
      float most = Vec<T>::largest(q[0]);
#pragma unroll
      for (int i = 1; i < kBatch; ++i) most = fmaxf(most, Vec<T>::largest(q[i]));
      largest = fmaxf(largest, most);
      move_to<false>(v, fmaxf(v.n, shift_of(most, a.c)));
      if (DUAL) move_to<false>(v1, fmaxf(v1.n, shift_of(most, kLog2e)));
      add_terms<false, false, T>(v, q, a.c);
      if (DUAL) add_terms<false, false, T>(v1, q, kLog2e);
    };
    uint32_t at = p.begin;
    for (; at + THREADS * kBatch <= p.end; at += THREADS * kBatch) add(std::true_type{}, at);
    if (at < p.end) add(std::false_type{}, at);
    if (tid < p.loose) {
      const uint32_t j = loose_at(p, tid);
      float x = to_float(z[j]);
      if (TAIL && marks[(j + first) / 32] >> ((j + first) % 32) & 1u) x = -INFINITY;
      largest = fmaxf(largest, x);
      move_to<false>(v, fmaxf(v.n, shift_of(x, a.c)));
      add_term<false>(v, x, a.c);
      if (DUAL) {
        move_to<false>(v1, fmaxf(v1.n, shift_of(x, kLog2e)));
        add_term<false>(v1, x, kLog2e);
      }
    }
    if (tid < a.top) {
      sh.slot[tid] = id != TL_NO_TOKEN;
      sh.u[tid] = u;
      sh.z[tid] = zk;
    }
    if (tid == 0) sh.zt = zt;
    warp_join<false>(v);
    if (DUAL) warp_join<false>(v1);
    largest = warp_max(largest);
    if (lane == 0)
      for (uint32_t c = 0; c < parts; ++c) {
        DistillShared<THREADS> *to = CLUSTER ? cluster.map_shared_rank(&sh, c) : &sh;
        to->sums[part * kWarps + warp] = v;
        if (DUAL) to->sums1[part * kWarps + warp] = v1;
        to->largest[part * kWarps + warp] = largest;
      }
    everyone();
    float m = -INFINITY;
    for (uint32_t i = lane; i < parts * kWarps; i += 32) m = fmaxf(m, sh.largest[i]);
    m = warp_max(m);
    Outside o = {m, 0.0f, 0.0f};
    const bool far = far_out(m, a.c) || far_out(m, kLog2e);
    if (far) o = careful_outside<THREADS, TAIL>(z, a.vocab, a.c, target, marks, first, sh.scratch);
    if (warp == 0) {
      if (!far) {
        const float n = shift_of(m, a.c), n1 = shift_of(m, kLog2e);
        for (uint32_t i = lane; i < parts * kWarps; i += 32) {
          o.s += sh.sums[i].s * ex2_approx(sh.sums[i].n - n);
          if (DUAL) o.s1 += sh.sums1[i].s * ex2_approx(sh.sums1[i].n - n1);
        }
        o.s = sum_at(warp_sum(o.s), n, m, a.c);
        o.s1 = DUAL ? sum_at(warp_sum(o.s1), n1, m, kLog2e) : o.s;
      }
      SlotLane l;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const uint32_t j = lane + 32 * i;
        l.slot[i] = j < a.top && sh.slot[j];
        l.u[i] = l.slot[i] ? sh.u[j] : -INFINITY;
        l.z[i] = l.slot[i] ? sh.z[j] : -INFINITY;
      }
      float loss, kl;
      const RowStats r = join_slots<TAIL>(a, l, o, target, sh.zt, loss, kl);
      if (lane == 0) {
        sh.r = r;
        if (part == 0) {
          a.loss[row] = loss;
          if (a.kl) a.kl[row] = kl;
          if (a.stats) write_stats(a.stats + row * TL_DISTILL_STATS, r);
        }
      }
    }
    // the marks were read once more, and by every CTA all of the row, which
    // the gradient may overwrite
    if (far) everyone();
    if (TAIL && id != TL_NO_TOKEN) marks[(id + first) / 32] = 0;
    if (GRAD) {
      __syncthreads();
      const RowStats r = sh.r;
      const float pk = id != TL_NO_TOKEN ? expf(u - r.h) * r.b : 0.0f;
      const bool here = id != TL_NO_TOKEN && holds<T>(p, id);
      gradient_part<THREADS, AGAIN, true, DUAL>(a, row, z, p, r, here ? id : TL_NO_TOKEN, pk, zk, t,
                                                target && tid == 0 && holds<T>(p, t), zt);
    }
    everyone();  // shared memory is free for the next row
  }
}

// The gradient from the statistics that the loss kept; bound by memory: 4096
// x 65501 fp16 178 us (6.0 TB/s of reads and writes).
template <typename T, bool DUAL>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const DistillArgs a) {
  pdl_enter();
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, blockIdx.y, gridDim.y);
    const float *st = a.stats + row * TL_DISTILL_STATS;
    const RowStats r = {st[0], st[1], st[2], st[3], st[4], st[5], st[6], st[7]};
    uint32_t id;
    float u;
    read_slot(a, row, id, u);
    if (id != TL_NO_TOKEN && !holds<T>(p, id)) id = TL_NO_TOKEN;
    const float zk = id != TL_NO_TOKEN ? to_float(z[id]) : -INFINITY;
    const float pk = id != TL_NO_TOKEN ? expf(u - r.h) * r.b : 0.0f;
    const uint32_t t = read_target(a, row);
    const bool here = t != TL_NO_TOKEN && threadIdx.x == 0 && holds<T>(p, t);
    const float zt = here ? to_float(z[t]) : 0.0f;
    __syncthreads();  // every slot's logit is read
    gradient_part<kThreads, false, false, DUAL>(a, row, z, p, r, id, pk, zk, t, here, zt);
    __syncthreads();
  }
}

int bad(const char *who, const char *what) {
  return fail(TL_ERR_INVALID, std::string(who) + ": " + what);
}

bool positive(float x) { return x > 0.0f && !std::isinf(x); }

int distill_args(const char *who, const tl_distill_desc *d, DistillArgs &a) {
  if (!d) return bad(who, "null descriptor");
  a.row_stride = d->row_stride;
  if (int rc = check_rows(who, d->logits, d->type, d->rows, d->vocab, d->temperature, a.row_stride))
    return rc;
  if (!positive(d->teacher_temperature))
    return bad(who, "teacher temperature must be positive and finite");
  if (1.0 / d->teacher_temperature > FLT_MAX)
    return fail(TL_ERR_RANGE, std::string(who) + ": teacher temperature's reciprocal is beyond fp32");
  if (!std::isfinite(d->kd_weight) || !std::isfinite(d->ce_weight))
    return bad(who, "weights must be finite");
  if (d->tail != TL_DISTILL_RENORM && d->tail != TL_DISTILL_TAIL)
    return bad(who, "unknown tail mode");
  if (d->top == 0) return bad(who, "no teacher slots");
  if (d->top > TL_TOKEN_MAX_TOP)
    return fail(TL_ERR_RANGE, std::string(who) + ": more than 128 teacher slots");
  if (d->top > d->vocab) return bad(who, "more teacher slots than tokens");
  if (d->tail == TL_DISTILL_TAIL && d->vocab > TL_DISTILL_MAX_VOCAB)
    return fail(TL_ERR_RANGE, std::string(who) + ": vocabulary too long for the teacher's tail");
  if (d->rows == 0) return TL_OK;
  if (!d->teacher_ids || !d->teacher) return bad(who, "null teacher_ids or teacher");
  a.logits = d->logits;
  a.rows = d->rows;
  a.vocab = d->vocab;
  a.top = d->top;
  a.c = static_cast<float>(1.4426950408889634 / d->temperature);
  a.inv_t = static_cast<float>(1.0 / d->temperature);
  a.inv_t_low = static_cast<float>(1.0 / d->temperature - a.inv_t);
  a.u_scale = static_cast<float>(1.0 / d->teacher_temperature);
  a.kd = d->kd_weight;
  a.ce = d->ce_weight;
  a.teacher_ids = d->teacher_ids;
  a.teacher = d->teacher;
  a.targets = d->targets;
  a.loss = d->loss;
  a.kl = d->kl;
  a.stats = d->stats;
  a.row_scale = d->row_scale;
  a.dlogits = d->dlogits;
  a.d_row_stride = d->d_row_stride;
  return TL_OK;
}

// The status word, last: it needs the device.
int with_status(const char *who, DistillArgs &a) {
  a.status = device_status_ptr();
  return a.status ? TL_OK : fail(TL_ERR_CUDA, std::string(who) + ": no status word");
}

template <typename T, int THREADS, bool TAIL, bool DUAL, bool GRAD, bool AGAIN, bool CLUSTER>
int launch_team(const char *who, const DistillArgs &a, uint32_t parts, cudaStream_t s) {
  const uint32_t most = kNumSMs * 64u;
  const auto marks_bytes = [](size_t vocab) { return (vocab + 2 * Vec<T>::kElems + 31) / 32 * 4; };
  const size_t smem = TAIL ? marks_bytes(a.vocab) : 0;
  const unsigned grid = (a.rows < most ? a.rows : most) * parts;
  const auto kernel = distill_kernel<T, THREADS, TAIL, DUAL, GRAD, AGAIN, CLUSTER>;
  if (smem > 40 * 1024) {
    // the limit is the kernel's, not the call's: the same for every call, so
    // that none lowers it between another thread's two steps
    if (int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(marks_bytes(TL_DISTILL_MAX_VOCAB))),
                            who))
      return rc;
  }
  if (CLUSTER) launch_pdl_cluster(kernel, grid, THREADS, smem, s, parts, a);
  else launch_pdl(kernel, grid, THREADS, smem, s, a);
  return launch_status(who);
}

template <typename T, bool TAIL, bool DUAL, bool GRAD>
int launch_form(const char *who, const DistillArgs &a, cudaStream_t s) {
  const uint32_t parts = cluster_parts(a.rows, a.vocab / Vec<T>::kElems);
  if (parts > 1) return launch_team<T, kThreads, TAIL, DUAL, GRAD, false, true>(who, a, parts, s);
  if constexpr (GRAD) {
    const size_t rows = a.rows < 4 * kNumSMs ? a.rows : 4 * kNumSMs;
    const size_t under_way = rows * a.vocab * sizeof(T);
    if (under_way > kL2Wide) return launch_team<T, 2 * kThreads, TAIL, DUAL, true, true, false>(who, a, 1, s);
    if (under_way > kL2Again) return launch_team<T, kThreads, TAIL, DUAL, true, true, false>(who, a, 1, s);
  }
  return launch_team<T, kThreads, TAIL, DUAL, GRAD, false, false>(who, a, 1, s);
}

template <typename T, bool TAIL, bool GRAD>
int launch_distill(const char *who, const DistillArgs &a, cudaStream_t s) {
  return dual(a) ? launch_form<T, TAIL, true, GRAD>(who, a, s)
                 : launch_form<T, TAIL, false, GRAD>(who, a, s);
}

template <typename T> int launch_backward(const char *who, const DistillArgs &a, cudaStream_t s) {
  const dim3 grid = gradient_grid(a.rows, a.vocab / Vec<T>::kElems);
  if (dual(a)) launch_pdl(distill_backward_kernel<T, true>, grid, kThreads, 0, s, a);
  else launch_pdl(distill_backward_kernel<T, false>, grid, kThreads, 0, s, a);
  return launch_status(who);
}

template <bool GRAD>
int distill_forward(const char *who, const tl_distill_desc *d, DistillArgs &a, void *stream) {
  if (!a.loss) return bad(who, "null loss");
  if (int rc = with_status(who, a)) return rc;
  cudaStream_t s = as_stream(stream);
  const bool tail = d->tail == TL_DISTILL_TAIL;
  if (distill_short(a, d->type, tail, GRAD, s)) return launch_status(who);
  switch (d->type) {
    case TL_FLOAT32:
      return tail ? launch_distill<float, true, GRAD>(who, a, s)
                  : launch_distill<float, false, GRAD>(who, a, s);
    case TL_FLOAT16:
      return tail ? launch_distill<__half, true, GRAD>(who, a, s)
                  : launch_distill<__half, false, GRAD>(who, a, s);
    default:
      return tail ? launch_distill<__nv_bfloat16, true, GRAD>(who, a, s)
                  : launch_distill<__nv_bfloat16, false, GRAD>(who, a, s);
  }
}

}  // namespace
}  // namespace token
}  // namespace tl

using namespace tl;
using namespace tl::token;

extern "C" {

int tl_distill_rows(const tl_distill_desc *desc, void *stream) {
  const char *who = "tl_distill_rows";
  DistillArgs a{};
  if (int rc = distill_args(who, desc, a)) return rc;
  if (a.rows == 0) return TL_OK;
  return distill_forward<false>(who, desc, a, stream);
}

int tl_distill_train_rows(const tl_distill_desc *desc, void *stream) {
  const char *who = "tl_distill_train_rows";
  DistillArgs a{};
  if (int rc = distill_args(who, desc, a)) return rc;
  if (a.rows == 0) return TL_OK;
  if (int rc = check_gradient(who, a.logits, a.row_stride, a.dlogits, desc->type, a.rows, a.vocab,
                              a.d_row_stride))
    return rc;
  return distill_forward<true>(who, desc, a, stream);
}

int tl_distill_backward_rows(const tl_distill_desc *desc, void *stream) {
  const char *who = "tl_distill_backward_rows";
  DistillArgs a{};
  if (int rc = distill_args(who, desc, a)) return rc;
  if (a.rows == 0) return TL_OK;
  if (int rc = check_gradient(who, a.logits, a.row_stride, a.dlogits, desc->type, a.rows, a.vocab,
                              a.d_row_stride))
    return rc;
  if (!a.stats) return bad(who, "null stats");
  if (int rc = with_status(who, a)) return rc;
  cudaStream_t s = as_stream(stream);
  if (distill_backward_short(a, desc->type, s)) return launch_status(who);
  switch (desc->type) {
    case TL_FLOAT32: return launch_backward<float>(who, a, s);
    case TL_FLOAT16: return launch_backward<__half>(who, a, s);
    default: return launch_backward<__nv_bfloat16>(who, a, s);
  }
}

}  // extern "C"
