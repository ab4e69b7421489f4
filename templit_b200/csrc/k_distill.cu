// Distillation from a teacher's top tokens: loss rows, their gradient, and
// both in one call (tl_distill_rows, tl_distill_backward_rows,
// tl_distill_train_rows).
//
// With the student's q = softmax(z / tau) and the teacher's p over the slots
// (and p_r over the tokens outside, TL_DISTILL_TAIL), the gradient of
// KL(p || q) is (q_j - p_j) / tau in a slot and, outside the slots, q_j (1 -
// p_r / q_r) / tau.  The second is evaluated as e^((z_j - g) / tau) a / tau
// with g the largest logit outside the slots, s_r the sum there and a =
// (q_r - p_r) / s_r: neither q_r nor q_j / q_r can leave the range of fp32,
// however small the student's mass outside the slots is.
#include "token_rows.cuh"

#include <cooperative_groups.h>

namespace tl {
namespace token {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;  // vectors of a thread in flight
constexpr int kPerLane = TL_TOKEN_MAX_TOP / 32;

struct DistillArgs {
  const void *logits;
  uint64_t row_stride;
  uint32_t rows, vocab, top;
  float c, inv_t;   // log2(e) / temperature, 1 / temperature
  float u_scale;    // 1 / teacher_temperature
  float kd, ce;
  const uint32_t *teacher_ids;
  const float *teacher;
  const uint32_t *targets;
  float *loss, *kl, *stats;
  const float *row_scale;
  void *dlogits;
  uint64_t d_row_stride;
  uint32_t *status;
};

// What the gradient of a row needs.
struct RowStats {
  float m, s, s1;  // largest logit, sums at the temperature and at 1
  float g, a;      // outside the slots
  float h, b;      // the slots' p
};

// Whether the row's logits are outside what whole powers of two hold.
__device__ __forceinline__ bool row_far(const RowStats &r, float c) {
  return far_out(r.m, c) || far_out(r.g, c) || far_out(r.m, kLog2e);
}

// The gradient of one row's part.  Thread k < top has slot k: id
// (TL_NO_TOKEN if empty or in another part), its p and its logit, read
// before anything is written (dlogits may be logits); t is the target (or
// TL_NO_TOKEN), `target_here` its logit zt in the thread that writes it.
// Outside the slots dz = kd/tau a e^((z - g) / tau) + ce e^(z - m) / s1; with
// a temperature of 1 (not DUAL) both are one exponential.  The slots and
// the target are written a second time.
template <typename T, bool DUAL>
__device__ __forceinline__ void gradient_part(const DistillArgs &a, size_t row, const Part &part,
                                              const RowStats &r, uint32_t id, float p, float zk,
                                              uint32_t t, bool target_here, float zt) {
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
  const float scale = a.row_scale ? a.row_scale[row] : 1.0f;
  const bool none = scale == 0.0f || r.s == 0.0f;
  const float kd = a.kd * a.inv_t * scale, ce = t == TL_NO_TOKEN ? 0.0f : a.ce * scale;
  const float coef = kd * r.a, coef1 = ce == 0.0f ? 0.0f : ce / r.s1;
  const bool far = row_far(r, a.c);
  // e^((z - g) / tau) = 2^(z c - n) 2^(n - g c), n whole: see Pow2Sums
  const float n = shift_of(r.g, a.c), n1 = shift_of(r.m, kLog2e);
  float k = coef * ex2_approx(-fmaf(r.g, a.c, -n));
  const float k1 = coef1 == 0.0f ? 0.0f : coef1 * ex2_approx(-fmaf(r.m, kLog2e, DUAL ? -n1 : -n));
  if (!DUAL) k += k1;
  const auto fast = [&](float x) {
    float g = k * ex2_approx(fmaf(x, a.c, -n));
    if (DUAL) g = fmaf(k1, ex2_approx(fmaf(x, kLog2e, -n1)), g);
    return g;
  };
  const auto careful = [&](float x) {
    const float g = coef * ex2_approx((x - r.g) * a.c);
    return coef1 == 0.0f ? g : fmaf(coef1, ex2_approx((x - r.m) * kLog2e), g);
  };
  if (none) write_elements<kThreads>(z, dz, part, [](float) { return 0.0f; });
  else if (far) write_elements<kThreads>(z, dz, part, careful);
  else write_vectors<kThreads, kBatch>(z, dz, part, fast);
  __syncthreads();
  if (none) return;
  if (target_here && ce != 0.0f) dz[t] = from_float<T>((far ? careful(zt) : fast(zt)) - ce);
  __syncthreads();  // a target in a slot: the slot's value stands
  if (id != TL_NO_TOKEN) {
    float g = kd * (ex2_approx((zk - r.m) * a.c) / r.s - p);
    if (ce != 0.0f) g += fmaf(coef1, ex2_approx((zk - r.m) * kLog2e), id == t ? -ce : 0.0f);
    dz[id] = from_float<T>(g);
  }
}

// Slot k of a row in thread k: its id and value, empty ones as TL_NO_TOKEN.
__device__ __forceinline__ void read_slot(const DistillArgs &a, size_t row, uint32_t &id, float &u) {
  id = TL_NO_TOKEN;
  u = -INFINITY;
  if (threadIdx.x >= a.top) return;
  id = a.teacher_ids[row * a.top + threadIdx.x];
  u = a.teacher[row * a.top + threadIdx.x] * a.u_scale;
  if (id >= a.vocab) {
    if (id != TL_NO_TOKEN) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
    id = TL_NO_TOKEN;
  }
  if (u == -INFINITY) id = TL_NO_TOKEN;
  if (id == TL_NO_TOKEN) u = -INFINITY;
}

__device__ __forceinline__ uint32_t read_target(const DistillArgs &a, size_t row) {
  if (!a.targets) return TL_NO_TOKEN;
  const uint32_t t = a.targets[row];
  if (t < a.vocab) return t;
  if (t != TL_NO_TOKEN && threadIdx.x == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
  return TL_NO_TOKEN;
}

// What a warp makes of a row's slots and of the sums over the logits
// outside them (TAIL) or over all of them: lane l holds slots l + 32 i.
struct SlotLane {
  bool slot[kPerLane];
  float u[kPerLane], z[kPerLane];
};

// Relative to its largest logit m: s = sum of e^((z - m) / tau), s1 = sum of
// e^(z - m).
struct Outside {
  float m, s, s1;
};

template <bool TAIL>
__device__ __forceinline__ RowStats join_slots(const DistillArgs &a, const SlotLane &l,
                                               const Outside &o, bool target, float zt, float &loss,
                                               float &kl) {
  RowStats r;
  uint32_t slots = 0;
  float u_max = -INFINITY, z_max = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    slots += l.slot[i];
    if (l.slot[i]) u_max = fmaxf(u_max, l.u[i]), z_max = fmaxf(z_max, l.z[i]);
  }
  slots = __reduce_add_sync(0xffffffffu, slots);
  r.m = o.m, r.s = o.s, r.s1 = o.s1;
  if (TAIL) {
    // the whole row: the sums outside the slots and the slots' terms
    r.m = fmaxf(o.m, warp_max(z_max));
    float s = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (l.slot[i] && l.z[i] != -INFINITY) {
        s += ex2_approx((l.z[i] - r.m) * a.c);
        if (target) s1 += ex2_approx((l.z[i] - r.m) * kLog2e);
      }
    r.s = o.s * rescale(o.m, r.m, a.c) + warp_sum(s);
    if (target) r.s1 = o.s1 * rescale(o.m, r.m, kLog2e) + warp_sum(s1);
  }
  if (!target) r.s1 = 0.0f;
  // the teacher's p.  Their sum is taken in 64 bits: what is left of 1 may
  // be far smaller than the sum
  r.h = 0.0f, r.b = slots ? 1.0f : 0.0f;
  float p[kPerLane], log_sum = 0.0f, rest = 0.0f;
  if (!TAIL) r.h = slots ? warp_max(u_max) : 0.0f;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    p[i] = l.slot[i] ? expf(l.u[i] - r.h) : 0.0f;
    sum += p[i];
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (TAIL) {
    rest = slots ? fmaxf(0.0f, static_cast<float>(1.0 - sum)) : 0.0f;
  } else if (slots) {
    r.b = static_cast<float>(1.0 / sum);
    log_sum = logf(static_cast<float>(sum));
  }
  const float log_s = logf(r.s);
  kl = 0.0f;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    p[i] *= r.b;
    if (p[i] != p[i]) {
      kl = p[i];
    } else if (l.slot[i] && p[i] > 0.0f) {
      // a row of -inf has q = 0 everywhere
      const float log_q = r.s == 0.0f ? -INFINITY : (l.z[i] - r.m) * a.inv_t - log_s;
      kl += p[i] * ((l.u[i] - r.h) - log_sum - log_q);
    }
  }
  kl = warp_sum(kl);
  if (TAIL) {
    r.g = o.m == -INFINITY ? 0.0f : o.m;
    r.a = 0.0f;
    if (o.m != -INFINITY) {
      const float log_left = (o.m - r.m) * a.inv_t + logf(o.s) - log_s;  // log q_r
      if (rest > 0.0f) kl += rest * (logf(rest) - log_left);
      r.a = slots ? (expf(log_left) - rest) / o.s : 0.0f;
    }
  } else {
    r.g = r.m == -INFINITY ? 0.0f : r.m;
    r.a = slots && r.s != 0.0f ? 1.0f / r.s : 0.0f;
  }
  loss = a.kd == 0.0f ? 0.0f : a.kd * kl;  // a KL of +inf without weight
  if (target) {
    const float log_q1 = r.s1 == 0.0f ? -INFINITY : (zt - r.m) - logf(r.s1);
    loss -= a.ce * log_q1;
  }
  return r;
}

struct DistillShared {
  Sums scratch[kWarps];
  Pow2Sums sums[kMaxCluster * kWarps], sums1[kMaxCluster * kWarps];
  float largest[kMaxCluster * kWarps];
  bool slot[TL_TOKEN_MAX_TOP];
  float u[TL_TOKEN_MAX_TOP], z[TL_TOKEN_MAX_TOP];
  float zt;
  uint32_t t;
  RowStats r;
};

// Bits of the tokens in slots, so placed that a vector's are whole bytes
// (or half bytes): element j of a row at bit j + elements of a vector -
// head.
template <typename T> __device__ __forceinline__ uint32_t vector_marks(const uint32_t *marks, uint32_t v) {
  const uint8_t *b = reinterpret_cast<const uint8_t *>(marks);
  if (Vec<T>::kElems == 8) return b[v + 1];
  return b[(v + 1) / 2] >> (4 * ((v + 1) & 1)) & 15u;
}

// The sums outside the slots by add_logit, for rows that Pow2Sums cannot
// hold.
template <typename T, bool TAIL>
__device__ __noinline__ Outside careful_outside(const T *z, uint32_t vocab, float c, bool target,
                                                const uint32_t *marks, uint32_t first, Sums *scratch) {
  Sums v = empty_sums(), v1 = empty_sums();
  for (uint32_t j = threadIdx.x; j < vocab; j += kThreads) {
    if (TAIL && marks[(j + first) / 32] >> ((j + first) % 32) & 1u) continue;
    const float x = to_float(z[j]);
    add_logit(v, x, c);
    if (target) add_logit(v1, x, kLog2e);
  }
  v = block_merge<kWarps>(v, c, scratch);
  v1 = block_merge<kWarps>(v1, kLog2e, scratch);
  return {v.m, v.s, v1.s};
}

// One CTA per row, or a cluster of CTAs that share a row.  The slots'
// tokens are marked by a bit each in shared memory (TAIL), one pass over
// the row sums the others, a warp joins the slots to the sums, and with
// GRAD a second pass (out of L2: the CTA's part of the row is the last
// thing it read) writes the gradient.  DUAL: the target's term has sums of
// its own, at temperature 1.
template <typename T, bool TAIL, bool DUAL, bool GRAD, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 4) distill_kernel(const DistillArgs a) {
  extern __shared__ uint32_t marks[];
  __shared__ DistillShared sh;
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
    for (uint32_t w = tid; w < (a.vocab + 2 * E + 31) / 32; w += kThreads) marks[w] = 0;
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
    for (uint32_t at = p.begin; at < p.end; at += kThreads * kBatch) {
      uint4 q[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const uint32_t j = at + i * kThreads + tid;
        q[i] = j < p.end ? vec[j] : make_uint4(Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone, Vec<T>::kNone);
      }
      if (TAIL) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const uint32_t j = at + i * kThreads + tid;
          const uint32_t m = j < p.end ? vector_marks<T>(marks, j) : 0;
          if (m) Vec<T>::drop(q[i], m);
        }
      }
      float most = Vec<T>::largest(q[0]);
#pragma unroll
      for (int i = 1; i < kBatch; ++i) most = fmaxf(most, Vec<T>::largest(q[i]));
      largest = fmaxf(largest, most);
      move_to<false>(v, fmaxf(v.n, shift_of(most, a.c)));
      if (DUAL) move_to<false>(v1, fmaxf(v1.n, shift_of(most, kLog2e)));
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        float f[E];
        Vec<T>::unpack(q[i], f);
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
          add_term<false>(v, f[e], a.c);
          if (DUAL) add_term<false>(v1, f[e], kLog2e);
        }
      }
    }
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
        DistillShared *to = CLUSTER ? cluster.map_shared_rank(&sh, c) : &sh;
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
    if (far) o = careful_outside<T, TAIL>(z, a.vocab, a.c, target, marks, first, sh.scratch);
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
          if (a.stats) {
            float *st = a.stats + row * TL_DISTILL_STATS;
            st[0] = r.m, st[1] = r.s, st[2] = r.s1, st[3] = r.g;
            st[4] = r.a, st[5] = r.h, st[6] = r.b, st[7] = 0.0f;
          }
        }
      }
    }
    if (far) __syncthreads();  // the marks were read once more
    if (TAIL && id != TL_NO_TOKEN) marks[(id + first) / 32] = 0;
    if (GRAD) {
      __syncthreads();
      const RowStats r = sh.r;
      const float pk = id != TL_NO_TOKEN ? expf(u - r.h) * r.b : 0.0f;
      const bool here = id != TL_NO_TOKEN && holds<T>(p, id);
      gradient_part<T, DUAL>(a, row, p, r, here ? id : TL_NO_TOKEN, pk, zk, t,
                             target && tid == 0 && holds<T>(p, t), zt);
    }
    everyone();  // shared memory is free for the next row
  }
}

template <typename T, bool DUAL>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const DistillArgs a) {
  pdl_enter();
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Part p = part_of(z, a.vocab, blockIdx.y, gridDim.y);
    const float *st = a.stats + row * TL_DISTILL_STATS;
    const RowStats r = {st[0], st[1], st[2], st[3], st[4], st[5], st[6]};
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
    gradient_part<T, DUAL>(a, row, p, r, id, pk, zk, t, here, zt);
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

template <typename T, bool TAIL, bool DUAL, bool GRAD>
int launch_form(const char *who, const DistillArgs &a, cudaStream_t s) {
  const uint32_t vecs = a.vocab / Vec<T>::kElems;
  const uint32_t parts = cluster_parts(a.rows, vecs), most = kNumSMs * 64u;
  const size_t smem = TAIL ? (static_cast<size_t>(a.vocab) + 2 * Vec<T>::kElems + 31) / 32 * 4 : 0;
  const unsigned teams = a.rows < most ? a.rows : most;
  const auto kernel = parts == 1 ? distill_kernel<T, TAIL, DUAL, GRAD, false>
                                 : distill_kernel<T, TAIL, DUAL, GRAD, true>;
  if (smem > 40 * 1024) {
    if (int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem)),
                            who))
      return rc;
  }
  if (parts == 1) launch_pdl(kernel, teams, kThreads, smem, s, a);
  else launch_pdl_cluster(kernel, teams * parts, kThreads, smem, s, parts, a);
  return launch_status(who);
}

// Whether the target's term needs exponentials of its own.
bool dual(const DistillArgs &a) { return a.targets && a.ce != 0.0f && a.inv_t != 1.0f; }

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
  switch (desc->type) {
    case TL_FLOAT32: return launch_backward<float>(who, a, s);
    case TL_FLOAT16: return launch_backward<__half>(who, a, s);
    default: return launch_backward<__nv_bfloat16>(who, a, s);
  }
}

}  // extern "C"
