// Shared parts of the operators on rows of next-token logits
// (k_token_logprob.cu, k_distill.cu): logit types, ordering keys, block
// reductions and the checks of a descriptor's common fields.
#pragma once

#include "tl_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>

namespace tl {
namespace token {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// The one rounding of a gradient to the logits' type (to nearest even).
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// A logit as a whole number with the logits' order: -0 and 0 alike, NaN
// (0) below everything else.
__device__ __forceinline__ uint32_t order_of(float z) {
  if (z != z) return 0u;
  const uint32_t b = __float_as_uint(z + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Running softmax sums of one thread or row: largest logit m, s = sum of
// 2^((z - m) c), optionally h = sum of 2^((z - m) c) (z - m) (entropy).
// -inf adds nothing; NaN reaches s through its exponential.
struct Sums {
  float m, s, h;
};

__device__ __forceinline__ Sums empty_sums() { return {-INFINITY, 0.0f, 0.0f}; }

// Factor that takes sums relative to `from` to sums relative to `to` >=
// `from` (1 for two equal infinities).
__device__ __forceinline__ float rescale(float from, float to, float c) {
  return from == to ? 1.0f : ex2_approx((from - to) * c);
}

// h relative to `to`: sum e (z - to) = f (h + (from - to) s).  Sums that a
// factor of 0 wipes out are not multiplied by a difference that overflows
// (logits of the type's lowest value as masks).
__device__ __forceinline__ float rescale_h(const Sums &a, float to, float f) {
  return f == 0.0f || a.m == -INFINITY ? 0.0f : f * fmaf(a.m - to, a.s, a.h);
}

__device__ __forceinline__ Sums merge(const Sums &a, const Sums &b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float fa = rescale(a.m, m, c), fb = rescale(b.m, m, c);
  return {m, a.s * fa + b.s * fb, rescale_h(a, m, fa) + rescale_h(b, m, fb)};
}

__device__ __forceinline__ void add_logit(Sums &a, float z, float c) {
  if (z == -INFINITY) return;
  if (z > a.m) {
    const float f = rescale(a.m, z, c);
    a.h = rescale_h(a, z, f);
    a.s *= f;
    a.m = z;
  }
  const float d = z - a.m, e = ex2_approx(d * c);
  a.s += e;
  if (e != 0.0f) a.h = fmaf(e, d, a.h);
}

__device__ __forceinline__ Sums warp_merge(Sums v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums w = {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o),
                    __shfl_xor_sync(0xffffffffu, v.h, o)};
    v = merge(v, w, c);
  }
  return v;
}

// The CTA's sums in every thread; `scratch` holds one entry per warp.
template <int WARPS>
__device__ __forceinline__ Sums block_merge(Sums v, float c, Sums *scratch) {
  v = warp_merge(v, c);
  __syncthreads();  // the last use of scratch is over
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) v = merge(v, scratch[w], c);
  return v;
}

inline size_t type_size(int32_t type) { return type == TL_FLOAT32 ? 4 : 2; }

// Checks the fields that both descriptors have; fills in the default
// strides.  TL_OK, or the status that the entry point returns.
int check_rows(const char *who, const void *logits, int32_t type, uint32_t rows, uint32_t vocab,
               float temperature, uint64_t &row_stride);
// The same for the gradient of a backward call.
int check_gradient(const char *who, const void *logits, uint64_t row_stride, void *dlogits,
                   int32_t type, uint32_t rows, uint32_t vocab, uint64_t &d_row_stride);

}  // namespace token
}  // namespace tl
