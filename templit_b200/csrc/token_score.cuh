// Token scoring: what its kernels share (k_token_logprob.cu for a CTA or a
// cluster per row, k_token_logprob_short.cu for a warp per row).
#pragma once

#include "token_rows.cuh"

namespace tl {
namespace token {

struct ScoreArgs {
  const void *logits;
  uint64_t row_stride;
  uint32_t rows, vocab, top;
  float c;      // log2(e) / temperature
  float inv_t;  // 1 / temperature
  const uint32_t *targets;
  float *logprob, *entropy, *stats, *top_logprob;
  uint32_t *top_ids;
  const float *d_logprob, *d_entropy;
  void *dlogits;
  uint64_t d_row_stride;
  uint32_t segment_shift;  // a segment is 2^shift batches of a thread's vectors
  uint32_t *status;
};

// A row's statistics.
struct RowSums {
  float m, s;       // largest logit, sum of e^((z - m) / temperature)
  float log_s, entropy;
};

// log q of a logit; -inf in a row of -inf.
__device__ __forceinline__ float log_q(float z, const RowSums &r, float inv_t) {
  if (r.m == -INFINITY) return r.s != r.s ? r.s : -INFINITY;
  return (z - r.m) * inv_t - r.log_s;
}

__device__ __forceinline__ uint64_t key_of(float z, uint32_t id) {
  return (static_cast<uint64_t>(order_of(z)) << 32) | ~id;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

// The coefficients of a row's gradient (score_gradient).
struct ScoreGradient {
  float A, B, n;               // dz = -e (A + B x), e = 2^x, x = z c - n
  float m, inv_s, base, gl, ge;
  bool none, far;              // nothing comes in; outside Pow2Sums' range
};

// With n a whole number at the row's largest logit, q = e k and log q = x ln
// 2 + const fold into A and B.
__device__ __forceinline__ ScoreGradient score_gradient(const ScoreArgs &a, float m, float s,
                                                        float entropy, float gl, float ge) {
  ScoreGradient g;
  g.m = m, g.gl = gl, g.ge = ge;
  g.none = s == 0.0f || (gl == 0.0f && ge == 0.0f);
  g.far = far_out(m, a.c);
  g.inv_s = 1.0f / s;
  g.base = entropy - logf(s);
  g.n = rintf(m * a.c);
  const float off = fmaf(m, a.c, -g.n);  // x of the largest logit
  const float k = ex2_approx(-off) * g.inv_s;
  g.B = k * ge * 0.6931471805599453f;
  g.A = k * fmaf(ge, fmaf(-off, 0.6931471805599453f, g.base), gl);
  return g;
}

template <bool ENTROPY>
__device__ __forceinline__ float score_dz(const ScoreGradient &g, float c, float z) {
  float x = fmaf(z, c, -g.n);
  if (ENTROPY) x = max_nan(x, -1e4f);  // -inf: 0 times a number
  return -ex2_approx(x) * (ENTROPY ? fmaf(g.B, x, g.A) : g.A);
}

template <bool ENTROPY>
__device__ __forceinline__ Pair score_dz2(const ScoreGradient &g, Pair c, Pair z) {
  Pair x = fma2(z, c, pair(-g.n, -g.n));
  if (ENTROPY) {
    const float2 f = halves(x);
    x = pair(max_nan(f.x, -1e4f), max_nan(f.y, -1e4f));
  }
  const Pair f = ENTROPY ? fma2(pair(-g.B, -g.B), x, pair(-g.A, -g.A)) : pair(-g.A, -g.A);
  return mul2(ex2_pair(x), f);
}

// The same for rows far out.
__device__ __forceinline__ float careful_score_dz(const ScoreGradient &g, const ScoreArgs &a, float z) {
  const float d = z - g.m, q = ex2_approx(d * a.c) * g.inv_s;
  return q == 0.0f ? 0.0f : -q * fmaf(g.ge, fmaf(d, a.inv_t, g.base), g.gl);
}

// Launches the warp-per-row kernels for rows that suit them (false: not
// launched).
bool score_short(const ScoreArgs &a, int32_t type, cudaStream_t s);
bool score_backward_short(const ScoreArgs &a, int32_t type, cudaStream_t s);

}  // namespace token
}  // namespace tl
