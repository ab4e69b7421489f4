// Distillation rows: what the kernels share (k_distill.cu for a CTA or a
// cluster per row, k_distill_short.cu for a warp per row).
//
// With the student's q = softmax(z / tau) and the teacher's p over the slots
// (and p_r over the tokens outside, TL_DISTILL_TAIL), the gradient of
// KL(p || q) is (P q_j - p_j) / tau in a slot and, outside the slots, q_j (P -
// p_r / q_r) / tau, P the masses that the divergence counts: sum p_k + p_r, or
// sum p_k where the student has no token outside.  P is 1 unless p_r was held
// at 0 (slots of more than 1 together) or dropped.  The second is evaluated as
// e^((z_j - g) / tau) a / tau with g the largest logit outside the slots, s_r
// the sum there and a = (P q_r - p_r) / s_r: neither q_r nor q_j / q_r can
// leave the range of fp32, however small the student's mass outside the slots
// is.
#pragma once

#include "token_rows.cuh"

namespace tl {
namespace token {

constexpr int kPerLane = TL_TOKEN_MAX_TOP / 32;  // slots of a lane where a warp has them all

struct DistillArgs {
  const void *logits;
  uint64_t row_stride;
  uint32_t rows, vocab, top;
  float c, inv_t;   // log2(e) / temperature, 1 / temperature
  float u_scale;    // 1 / teacher_temperature
  float inv_t_low;  // 1 / temperature is inv_t + inv_t_low
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
  float e;         // P - 1
};

// Slot k of a row: its id and value, empty ones as TL_NO_TOKEN.
__device__ __forceinline__ void read_slot(const DistillArgs &a, size_t row, uint32_t k, uint32_t &id,
                                          float &u) {
  id = TL_NO_TOKEN;
  u = -INFINITY;
  if (k >= a.top) return;
  id = a.teacher_ids[row * a.top + k];
  u = a.teacher[row * a.top + k] * a.u_scale;
  if (id >= a.vocab) {
    if (id != TL_NO_TOKEN) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
    id = TL_NO_TOKEN;
  }
  if (u == -INFINITY) id = TL_NO_TOKEN;
  if (id == TL_NO_TOKEN) u = -INFINITY;
}

// The coefficients of a row's gradient.
struct DistillGradient {
  float k, n, k1, n1;            // dz = k 2^(z c - n) + k1 2^(z log2(e) - n1)
  float coef, coef1, kd, ce;     // the weights with the row's scale
  bool none, far;                // no gradient; outside Pow2Sums' range
};

// Outside the slots dz = kd/tau a e^((z - g) / tau) + ce e^(z - m) / s1, by
// whole powers of two n: e^((z - g) / tau) = 2^(z c - n) 2^(n - g c).  At a
// temperature of 1 (not DUAL) both terms are one exponential.
template <bool DUAL>
__device__ __forceinline__ DistillGradient distill_gradient(const DistillArgs &a, const RowStats &r,
                                                            uint32_t t, float scale) {
  DistillGradient g;
  g.none = scale == 0.0f || r.s == 0.0f;
  g.far = far_out(r.m, a.c) || far_out(r.g, a.c) || far_out(r.m, kLog2e);
  g.kd = a.kd * a.inv_t * scale;
  g.ce = t == TL_NO_TOKEN ? 0.0f : a.ce * scale;
  g.coef = g.kd * r.a;
  g.coef1 = g.ce == 0.0f ? 0.0f : g.ce / r.s1;
  g.n = shift_of(r.g, a.c);
  g.n1 = shift_of(r.m, kLog2e);
  g.k = g.coef * ex2_approx(-fmaf(r.g, a.c, -g.n));
  g.k1 = g.coef1 == 0.0f ? 0.0f : g.coef1 * ex2_approx(-fmaf(r.m, kLog2e, DUAL ? -g.n1 : -g.n));
  if (!DUAL) g.k += g.k1;
  return g;
}

template <bool DUAL>
__device__ __forceinline__ float distill_dz(const DistillGradient &g, float c, float z) {
  const float d = g.k * ex2_approx(fmaf(z, c, -g.n));
  return DUAL ? fmaf(g.k1, ex2_approx(fmaf(z, kLog2e, -g.n1)), d) : d;
}

template <bool DUAL>
__device__ __forceinline__ Pair distill_dz2(const DistillGradient &g, Pair c, Pair z) {
  const Pair d = mul2(pair(g.k, g.k), ex2_pair(fma2(z, c, pair(-g.n, -g.n))));
  if (!DUAL) return d;
  return fma2(pair(g.k1, g.k1), ex2_pair(fma2(z, pair(kLog2e, kLog2e), pair(-g.n1, -g.n1))), d);
}

// The same for rows far out.
__device__ __forceinline__ float careful_distill_dz(const DistillGradient &g, const RowStats &r,
                                                    float c, float z) {
  const float d = g.coef * ex2_approx((z - r.g) * c);
  return g.coef1 == 0.0f ? d : fmaf(g.coef1, ex2_approx((z - r.m) * kLog2e), d);
}

// In a slot with the teacher's p and the student's logit z: P q - p.
__device__ __forceinline__ float slot_dz(const DistillGradient &g, const RowStats &r, float c, float p,
                                         float z, bool target) {
  const float q = ex2_approx((z - r.m) * c) / r.s;
  const float d = g.kd * (fmaf(r.e, q, q) - p);
  return g.ce == 0.0f ? d : d + fmaf(g.coef1, ex2_approx((z - r.m) * kLog2e), target ? -g.ce : 0.0f);
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

// log x = e ln 2 + l, |l| < 0.41: only l is rounded (3e-8).
struct Log {
  float e, l;
};
__device__ __forceinline__ Log log_parts(float x) {
  if (!(x > 1e-37f && x < 1e37f)) return {0.0f, logf(x)};  // 0, inf, NaN
  const int32_t b = __float_as_int(x), up = (b & 0x7fffff) >= 0x400000;
  return {static_cast<float>((b >> 23) - 127 + up),
          logf(__int_as_float((b & 0x7fffff) | (up ? 0x3f000000 : 0x3f800000)))};
}
// x + (e ln 2 + l), of which x and e ln 2 nearly cancel: ln 2 in two parts,
// the first of 12 bits, whose multiples are exact.
__device__ __forceinline__ float add_log(float x, float e, float l) {
  return fmaf(e, 0.693115234375f, x) + fmaf(e, 3.1946184945309e-5f, l);
}

// The divergence is summed in units of 2^16, which changes no bit of it: one
// beyond fp32 (masks of the type's lowest value) may have a weight that brings
// the loss back.
constexpr float kUnit = 65536.0f;

template <bool TAIL>
__device__ __forceinline__ RowStats join_slots(const DistillArgs &a, const SlotLane &l,
                                               const Outside &o, bool target, float zt, float &loss,
                                               float &kl) {
  RowStats r;
  uint32_t slots = 0;
  float u_max = -INFINITY, z_max = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    if (i * 32 >= a.top) break;
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
    for (int i = 0; i < kPerLane; ++i) {
      if (i * 32 >= a.top) break;
      if (l.slot[i] && l.z[i] != -INFINITY) {
        s += ex2_approx((l.z[i] - r.m) * a.c);
        if (target) s1 += ex2_approx((l.z[i] - r.m) * kLog2e);
      }
    }
    r.s = o.s * rescale(o.m, r.m, a.c) + warp_sum(s);
    if (target) r.s1 = o.s1 * rescale(o.m, r.m, kLog2e) + warp_sum(s1);
  }
  if (!target) r.s1 = 0.0f;
  // the teacher's p.  Their sum is taken in 64 bits: what is left of 1 may
  // be far smaller than the sum
  r.h = 0.0f, r.b = slots ? 1.0f : 0.0f, r.e = 0.0f;
  float p[kPerLane], rest = 0.0f;
  Log log_sum = {0.0f, 0.0f};
  if (!TAIL) r.h = slots ? warp_max(u_max) : 0.0f;
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    if (i * 32 >= a.top) break;
    p[i] = l.slot[i] ? expf(l.u[i] - r.h) : 0.0f;
    sum += p[i];
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (TAIL) {
    const float left = slots ? static_cast<float>(1.0 - sum) : 0.0f;
    rest = fmaxf(0.0f, left);
    // P - 1, not P: of a P near 1 no bits are lost
    r.e = left >= 0.0f && o.m != -INFINITY ? 0.0f : -left;
  } else if (slots) {
    r.b = static_cast<float>(1.0 / sum);
    log_sum = log_parts(static_cast<float>(sum));
  }
  // The divergence is a small difference of logarithms of size 10, whose
  // roundings alone would be 1e-6 of a divergence of 0.1: u - x, x = (z - m)
  // / tau with its rounding, cancels against log s up to what is left.
  const Log log_s = log_parts(r.s);
  const auto term = [&](float p, float u, float z, float e, float l) {  // p (u - (z - r.m) / tau + e ln 2 + l) / kUnit
    const float d = z - r.m, x = d * a.inv_t;
    // beyond fp32 (such masks at a temperature below 1) nothing else counts
    // (but a NaN), and p may be small enough for p times it to be a number
    if (isinf(x)) return fmaf(p, l, (r.m / kUnit - z / kUnit) * p * a.inv_t);
    return p * (add_log((u - x) - fmaf(d, a.inv_t, -x) - d * a.inv_t_low, e, l) * (1.0f / kUnit));
  };
  kl = 0.0f;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    if (i * 32 >= a.top) break;
    p[i] *= r.b;
    if (p[i] != p[i]) {
      kl = p[i];
    } else if (l.slot[i] && p[i] > 0.0f) {
      // a row of -inf has q = 0 everywhere, as has a logit of -inf
      const bool some = r.s != 0.0f && l.z[i] != -INFINITY;
      kl += some ? term(p[i], l.u[i] - r.h, l.z[i], log_s.e - log_sum.e, log_s.l - log_sum.l) : INFINITY;
    }
  }
  kl = warp_sum(kl);
  if (TAIL) {
    // nothing outside: the target's term still needs a shift that follows
    // the row (from 0, e^(-m) is infinite below -88)
    r.g = o.m != -INFINITY ? o.m : r.m == -INFINITY ? 0.0f : r.m;
    r.a = 0.0f;
    if (o.m != -INFINITY) {
      const Log log_o = log_parts(o.s), log_r = log_parts(rest);
      // log rest - log q_r, q_r = o.s e^((o.m - m) / tau) / s
      if (rest > 0.0f)
        kl += term(rest, 0.0f, o.m, log_r.e - log_o.e + log_s.e, log_r.l - log_o.l + log_s.l);
      const float left = o.s * rescale(o.m, r.m, a.c) / r.s;
      r.a = slots ? (fmaf(r.e, left, left) - rest) / o.s : 0.0f;
    }
  } else {
    r.g = r.m == -INFINITY ? 0.0f : r.m;
    r.a = slots && r.s != 0.0f ? 1.0f / r.s : 0.0f;
  }
  loss = a.kd == 0.0f ? 0.0f : a.kd * kl * kUnit;  // a KL of +inf without weight
  kl *= kUnit;
  if (target) {
    const float log_q1 = r.s1 == 0.0f ? -INFINITY : (zt - r.m) - logf(r.s1);
    loss -= a.ce * log_q1;
  }
  return r;
}

// Bits of the tokens in slots, so placed that a vector's are whole bytes
// (or half bytes): element j of a row at bit j + elements of a vector -
// head.
template <typename T> __device__ __forceinline__ uint32_t vector_marks(const uint32_t *marks, uint32_t v) {
  const uint8_t *b = reinterpret_cast<const uint8_t *>(marks);
  if (Vec<T>::kElems == 8) return b[v + 1];
  return b[(v + 1) / 2] >> (4 * ((v + 1) & 1)) & 15u;
}

__device__ __forceinline__ void write_stats(float *st, const RowStats &r) {
  st[0] = r.m, st[1] = r.s, st[2] = r.s1, st[3] = r.g;
  st[4] = r.a, st[5] = r.h, st[6] = r.b, st[7] = r.e;
}

// Whether the target's term needs exponentials of its own.
inline bool dual(const DistillArgs &a) { return a.targets && a.ce != 0.0f && a.inv_t != 1.0f; }

// Launch the warp-per-row kernels for rows that suit them (false: not
// launched).
bool distill_short(const DistillArgs &a, int32_t type, bool tail, bool gradient, cudaStream_t s);
bool distill_backward_short(const DistillArgs &a, int32_t type, cudaStream_t s);

}  // namespace token
}  // namespace tl
