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

namespace tl {
namespace token {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

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

__device__ __forceinline__ float block_sum(float v, float *scratch) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v += scratch[w];
  return v;
}

__device__ __forceinline__ float block_max(float v, float *scratch) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v = fmaxf(v, scratch[w]);
  return v;
}

// The gradient of one row.  Thread k < top has slot k: id (TL_NO_TOKEN if
// empty), its p and its logit, read before anything is written (dlogits may
// be logits); t is the target or TL_NO_TOKEN, zt its logit.
template <typename T>
__device__ __forceinline__ void gradient_row(const DistillArgs &a, size_t row, const RowStats &r,
                                             uint32_t id, float p, float zk, uint32_t t, float zt) {
  const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
  T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
  const float scale = a.row_scale ? a.row_scale[row] : 1.0f;
  const bool none = scale == 0.0f || r.s == 0.0f;
  const float kd = a.kd * a.inv_t * scale, ce = t == TL_NO_TOKEN ? 0.0f : a.ce * scale;
  const float coef = kd * r.a, coef1 = ce == 0.0f ? 0.0f : ce / r.s1;
  const bool hard = ce != 0.0f;
  for (uint32_t j = threadIdx.x; j < a.vocab; j += kThreads) {
    float g = 0.0f;
    if (!none) {
      const float x = to_float(z[j]);
      g = coef * ex2_approx((x - r.g) * a.c);
      if (hard) g = fmaf(coef1, ex2_approx((x - r.m) * kLog2e), g);
    }
    dz[j] = from_float<T>(g);
  }
  __syncthreads();  // the slots and the target are written over
  if (none) return;
  const float inv_s = 1.0f / r.s;
  if (threadIdx.x == 0 && hard) {
    const float g = coef * ex2_approx((zt - r.g) * a.c) +
                    fmaf(coef1, ex2_approx((zt - r.m) * kLog2e), -ce);
    dz[t] = from_float<T>(g);
  }
  __syncthreads();  // a target in a slot: the slot's value stands
  if (threadIdx.x < a.top && id != TL_NO_TOKEN) {
    float g = kd * (ex2_approx((zk - r.m) * a.c) * inv_s - p);
    if (hard) g += fmaf(coef1, ex2_approx((zk - r.m) * kLog2e), id == t ? -ce : 0.0f);
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

// One CTA per row: the slots, the sums outside them (TL_DISTILL_TAIL: a bit
// per token in shared memory marks the slots), the loss, and with GRAD the
// gradient in a second pass over the row.
template <typename T, bool TAIL, bool GRAD>
__global__ void __launch_bounds__(kThreads) distill_kernel(const DistillArgs a) {
  extern __shared__ uint32_t marked[];
  __shared__ Sums scratch[kWarps];
  __shared__ float fscratch[kWarps];
  pdl_enter();
  if (TAIL) {
    for (uint32_t w = threadIdx.x; w < (a.vocab + 31) / 32; w += kThreads) marked[w] = 0;
    __syncthreads();
  }
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    uint32_t id;
    float u;
    read_slot(a, row, id, u);
    const bool slot = id != TL_NO_TOKEN;
    const float zk = slot ? to_float(z[id]) : -INFINITY;
    const uint32_t t = read_target(a, row);
    const float zt = t != TL_NO_TOKEN ? to_float(z[t]) : 0.0f;
    if (TAIL) {
      if (slot) atomicOr(&marked[id / 32], 1u << (id % 32));
      __syncthreads();
    }
    Sums v = empty_sums(), v1 = empty_sums();
    for (uint32_t j = threadIdx.x; j < a.vocab; j += kThreads) {
      const float x = to_float(z[j]);
      if (t != TL_NO_TOKEN) add_logit(v1, x, kLog2e);
      if (!TAIL || !(marked[j / 32] >> (j % 32) & 1u)) add_logit(v, x, a.c);
    }
    v = block_merge<kWarps>(v, a.c, scratch);
    v1 = block_merge<kWarps>(v1, kLog2e, scratch);
    RowStats r;
    Sums all = v;
    if (TAIL) {
      Sums mine = empty_sums();
      if (slot) add_logit(mine, zk, a.c);
      all = merge(v, block_merge<kWarps>(mine, a.c, scratch), a.c);
      if (slot) marked[id / 32] = 0;
    }
    const uint32_t slots = __syncthreads_count(slot);
    r.m = all.m;
    r.s = all.s;
    r.s1 = t != TL_NO_TOKEN ? v1.s : 0.0f;
    // the teacher's p
    float p = 0.0f, log_p = 0.0f, rest = 0.0f;
    if (TAIL) {
      r.h = 0.0f;
      r.b = slots ? 1.0f : 0.0f;
      if (slot) p = expf(u), log_p = u;
      rest = fmaxf(0.0f, 1.0f - block_sum(p, fscratch));
      if (slots == 0) rest = 0.0f;
    } else {
      r.h = block_max(u, fscratch);
      const float sum = block_sum(slot ? expf(u - r.h) : 0.0f, fscratch);
      r.b = slots ? 1.0f / sum : 0.0f;
      if (!slots) r.h = 0.0f;
      if (slot) {
        p = expf(u - r.h) * r.b;
        log_p = (u - r.h) - logf(sum);
      }
    }
    const float log_s = logf(r.s);
    float term = 0.0f;
    if (slot && p > 0.0f) {
      // an empty student row has q = 0 everywhere
      const float lq = r.s == 0.0f ? -INFINITY : (zk - r.m) * a.inv_t - log_s;
      term = p * (log_p - lq);
    } else if (p != p) {
      term = p;
    }
    float kl = block_sum(term, fscratch);
    if (TAIL) {
      r.g = v.m;
      r.a = 0.0f;
      if (v.m == -INFINITY) {
        r.g = 0.0f;
      } else {
        const float lq_r = (v.m - r.m) * a.inv_t + logf(v.s) - log_s;
        if (rest > 0.0f) kl += rest * (logf(rest) - lq_r);
        r.a = slots ? (expf(lq_r) - rest) / v.s : 0.0f;
      }
    } else {
      r.g = r.m == -INFINITY ? 0.0f : r.m;
      r.a = slots && r.s != 0.0f ? 1.0f / r.s : 0.0f;
    }
    if (threadIdx.x == 0) {
      float loss = a.kd == 0.0f ? 0.0f : a.kd * kl;  // a KL of +inf without weight
      if (t != TL_NO_TOKEN && a.ce != 0.0f) {
        const float lq1 = r.s1 == 0.0f ? -INFINITY : (zt - r.m) - logf(r.s1);
        loss -= a.ce * lq1;
      }
      a.loss[row] = loss;
      if (a.kl) a.kl[row] = kl;
      if (a.stats) {
        float *st = a.stats + row * TL_DISTILL_STATS;
        st[0] = r.m, st[1] = r.s, st[2] = r.s1, st[3] = r.g;
        st[4] = r.a, st[5] = r.h, st[6] = r.b, st[7] = 0.0f;
      }
    }
    if (GRAD) {
      gradient_row<T>(a, row, r, id, p, zk, t, zt);
      __syncthreads();
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const DistillArgs a) {
  pdl_enter();
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    const float *st = a.stats + row * TL_DISTILL_STATS;
    const RowStats r = {st[0], st[1], st[2], st[3], st[4], st[5], st[6]};
    uint32_t id;
    float u;
    read_slot(a, row, id, u);
    const bool slot = id != TL_NO_TOKEN;
    const float zk = slot ? to_float(z[id]) : -INFINITY;
    const float p = slot ? expf(u - r.h) * r.b : 0.0f;
    const uint32_t t = read_target(a, row);
    const float zt = t != TL_NO_TOKEN ? to_float(z[t]) : 0.0f;
    __syncthreads();  // every slot's logit is read
    gradient_row<T>(a, row, r, id, p, zk, t, zt);
    __syncthreads();
  }
}

unsigned grid_of(uint32_t rows) {
  const uint32_t most = kNumSMs * 64u;
  return rows < most ? rows : most;
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

template <typename T, bool TAIL, bool GRAD>
int launch_distill(const char *who, const DistillArgs &a, cudaStream_t s) {
  const size_t smem = TAIL ? (static_cast<size_t>(a.vocab) + 31) / 32 * 4 : 0;
  if (smem > 48 * 1024) {
    if (int rc = check_cuda(cudaFuncSetAttribute(distill_kernel<T, TAIL, GRAD>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(smem)),
                            who))
      return rc;
  }
  launch_pdl(distill_kernel<T, TAIL, GRAD>, grid_of(a.rows), kThreads, smem, s, a);
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
    case TL_FLOAT32: launch_pdl(distill_backward_kernel<float>, grid_of(a.rows), kThreads, 0, s, a); break;
    case TL_FLOAT16: launch_pdl(distill_backward_kernel<__half>, grid_of(a.rows), kThreads, 0, s, a); break;
    default: launch_pdl(distill_backward_kernel<__nv_bfloat16>, grid_of(a.rows), kThreads, 0, s, a); break;
  }
  return launch_status(who);
}

}  // extern "C"
