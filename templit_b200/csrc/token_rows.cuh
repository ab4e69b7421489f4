// Shared parts of the operators on rows of next-token logits
// (k_token_logprob*.cu, k_distill*.cu): logit types, ordering keys, softmax
// sums, the gradients' passes over a row and the checks of a descriptor's
// common fields.
#pragma once

#include "tl_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <climits>
#include <type_traits>

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

// order_of for a number that is not NaN.
__device__ __forceinline__ uint32_t order_of_number(float z) {
  const int32_t b = __float_as_int(z + 0.0f);
  return static_cast<uint32_t>(b ^ ((b >> 31) | static_cast<int32_t>(0x80000000u)));
}

// n += a > b and n += a >= b in two instructions (the compiler's own takes
// four or five where many are added up).
__device__ __forceinline__ void count_gt(uint32_t &n, uint32_t a, uint32_t b) {
  asm("{ .reg .pred p; setp.gt.u32 p, %1, %2; @p add.u32 %0, %0, 1; }" : "+r"(n) : "r"(a), "r"(b));
}
__device__ __forceinline__ void count_ge(uint32_t &n, uint32_t a, uint32_t b) {
  asm("{ .reg .pred p; setp.ge.u32 p, %1, %2; @p add.u32 %0, %0, 1; }" : "+r"(n) : "r"(a), "r"(b));
}

// bits |= bit where a >= b
__device__ __forceinline__ void mark_from(uint32_t &bits, float a, float b, uint32_t bit) {
  asm("{ .reg .pred p; setp.ge.f32 p, %1, %2; @p or.b32 %0, %0, %3; }"
      : "+r"(bits)
      : "f"(a), "f"(b), "r"(bit));
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

// Two fp32 in a register pair: Blackwell's packed arithmetic does both in
// one issued instruction.
typedef unsigned long long Pair;
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ float2 halves(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair ex2_pair(Pair x) {
  const float2 f = halves(x);
  return pair(ex2_approx(f.x), ex2_approx(f.y));
}

// 16 bytes of logits.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int kElems = 4;
  static constexpr uint32_t kNone = 0xff800000u;  // -inf
  static __device__ __forceinline__ void unpack(const uint4 &v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ void pairs(const uint4 &v, Pair (&f)[2]) {
    f[0] = pair(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = pair(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ uint4 pack_pairs(const Pair (&f)[2]) {
    const float2 a = halves(f[0]), b = halves(f[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x),
                      __float_as_uint(b.y));
  }
  // makes the elements whose bit is set in m -inf
  static __device__ __forceinline__ void drop(uint4 &v, uint32_t m) {
    if (m & 1) v.x = kNone;
    if (m & 2) v.y = kNone;
    if (m & 4) v.z = kNone;
    if (m & 8) v.w = kNone;
  }
  // largest element (NaN ignored)
  static __device__ __forceinline__ float largest(const uint4 &v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                 fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
};
template <> struct Vec<__half> {
  static constexpr int kElems = 8;
  static constexpr uint32_t kNone = 0xfc00fc00u;
  static __device__ __forceinline__ void unpack(const uint4 &v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ void drop(uint4 &v, uint32_t m) {
    v.x = drop_pair(v.x, m), v.y = drop_pair(v.y, m >> 2);
    v.z = drop_pair(v.z, m >> 4), v.w = drop_pair(v.w, m >> 6);
  }
  static __device__ __forceinline__ uint32_t drop_pair(uint32_t w, uint32_t m) {
    if (m & 1) w = (w & 0xffff0000u) | (kNone & 0xffffu);
    if (m & 2) w = (w & 0xffffu) | (kNone & 0xffff0000u);
    return w;
  }
  static __device__ __forceinline__ float largest(const uint4 &v) {
    const __half2 *p = reinterpret_cast<const __half2 *>(&v);
    const __half2 a = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(__low2float(a), __high2float(a));
  }
  static __device__ __forceinline__ void pairs(const uint4 &v, Pair (&f)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
      f[i] = pair(p.x, p.y);
    }
  }
  static __device__ __forceinline__ uint4 pack_pairs(const Pair (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 p = __float22half2_rn(halves(f[i]));
      w[i] = *reinterpret_cast<const uint32_t *>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int kElems = 8;
  static constexpr uint32_t kNone = 0xff80ff80u;
  static __device__ __forceinline__ void unpack(const uint4 &v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void drop(uint4 &v, uint32_t m) {
    v.x = drop_pair(v.x, m), v.y = drop_pair(v.y, m >> 2);
    v.z = drop_pair(v.z, m >> 4), v.w = drop_pair(v.w, m >> 6);
  }
  static __device__ __forceinline__ uint32_t drop_pair(uint32_t w, uint32_t m) {
    if (m & 1) w = (w & 0xffff0000u) | (kNone & 0xffffu);
    if (m & 2) w = (w & 0xffffu) | (kNone & 0xffff0000u);
    return w;
  }
  static __device__ __forceinline__ float largest(const uint4 &v) {
    const __nv_bfloat162 *p = reinterpret_cast<const __nv_bfloat162 *>(&v);
    const __nv_bfloat162 a = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(__low2float(a), __high2float(a));
  }
  static __device__ __forceinline__ void pairs(const uint4 &v, Pair (&f)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 pack_pairs(const Pair (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 p = __float22bfloat162_rn(halves(f[i]));
      w[i] = *reinterpret_cast<const uint32_t *>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// ---- rows in 16-byte vectors -------------------------------------------
// A CTA reads its part of a row (the whole row, or its slice of one that
// several CTAs share) as aligned 16-byte vectors; the elements before the
// first and after the last vector (fewer than two vectors' worth) belong to
// the first part and take one thread each.

// One CTA's part of a row: vectors [begin, end) of those that start at
// element `head`, and in the first part the elements outside the vectors.
struct Part {
  uint32_t head, begin, end, tail;  // tail: first element after the vectors
  uint32_t loose;                   // elements outside the vectors (first part)
};

template <typename T>
__device__ __forceinline__ Part part_of(const T *row, uint32_t vocab, uint32_t part, uint32_t parts) {
  constexpr uint32_t E = Vec<T>::kElems;
  const uint32_t past = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T);
  const uint32_t head = min(vocab, (E - past) % E);
  const uint32_t vecs = (vocab - head) / E;
  const uint32_t each = (vecs + parts - 1) / parts;
  Part p;
  p.head = head;
  p.begin = min(vecs, part * each);
  p.end = min(vecs, p.begin + each);
  p.tail = head + vecs * E;
  p.loose = part == 0 ? head + (vocab - p.tail) : 0;
  return p;
}

// Element of loose index i (< part.loose), and whether a part holds element j.
__device__ __forceinline__ uint32_t loose_at(const Part &p, uint32_t i) {
  return i < p.head ? i : p.tail + (i - p.head);
}
template <typename T> __device__ __forceinline__ bool holds(const Part &p, uint32_t j) {
  constexpr uint32_t E = Vec<T>::kElems;
  if (j < p.head || j >= p.tail) return p.loose != 0;
  const uint32_t v = (j - p.head) / E;
  return v >= p.begin && v < p.end;
}

// dz_j = f(z_j) over a CTA's part, element by element.
template <int THREADS, typename T, typename F>
__device__ __forceinline__ void write_elements(const T *z, T *dz, const Part &p, F f) {
  constexpr uint32_t E = Vec<T>::kElems;
  for (uint32_t j = p.head + p.begin * E + threadIdx.x; j < p.head + p.end * E; j += THREADS)
    dz[j] = from_float<T>(f(to_float(z[j])));
  if (threadIdx.x < p.loose) {
    const uint32_t j = loose_at(p, threadIdx.x);
    dz[j] = from_float<T>(f(to_float(z[j])));
  }
}

// The same by vectors, BATCH of a thread's in flight, where logits and
// gradient are aligned alike: two(pair) for the vectors' logits, one(z) for
// the others.  dz may be z: a thread reads what it writes.  AGAIN: the CTA
// has just read the row, and L2 does not hold the rows of all CTAs; the
// last batches come first, and neither they nor the gradient need to stay.
// WHOLE: whole batches have a loop without conditions (the gradient beside
// its loss: 447 -> 427 us on 4096 x 128000 bf16; by itself it is bound by
// memory, and with two coefficients more out of registers: 136 -> 150 us).
template <int THREADS, int BATCH, bool AGAIN, bool WHOLE, typename T, typename F, typename G>
__device__ __forceinline__ void write_vectors(const T *z, T *dz, const Part &p, F two, G one) {
  constexpr uint32_t E = Vec<T>::kElems, kStep = THREADS * BATCH;
  if ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15u)
    return write_elements<THREADS>(z, dz, p, one);
  const uint4 *vec = reinterpret_cast<const uint4 *>(z + p.head);
  uint4 *out = reinterpret_cast<uint4 *>(dz + p.head);
  const auto batch = [&](auto full, uint32_t at) {  // full: no vector is past the end
    uint4 r[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const uint32_t i = at + u * THREADS + threadIdx.x;
      if (full || i < p.end) r[u] = AGAIN ? __ldcs(vec + i) : vec[i];
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const uint32_t i = at + u * THREADS + threadIdx.x;
      if (!full && i >= p.end) continue;
      Pair x[E / 2];
      Vec<T>::pairs(r[u], x);
#pragma unroll
      for (uint32_t e = 0; e < E / 2; ++e) x[e] = two(x[e]);
      if (AGAIN) __stcs(out + i, Vec<T>::pack_pairs(x));
      else out[i] = Vec<T>::pack_pairs(x);
    }
  };
  if (WHOLE) {
    const uint32_t whole = (p.end - p.begin) / kStep, rest = p.begin + whole * kStep;
    if (AGAIN && rest < p.end) batch(std::false_type{}, rest);
    for (uint32_t k = 0; k < whole; ++k)
      batch(std::true_type{}, p.begin + (AGAIN ? whole - 1 - k : k) * kStep);
    if (!AGAIN && rest < p.end) batch(std::false_type{}, rest);
  } else {
    for (uint32_t at = p.begin; at < p.end; at += kStep) batch(std::false_type{}, at);
  }
  if (threadIdx.x < p.loose) {
    const uint32_t j = loose_at(p, threadIdx.x);
    dz[j] = from_float<T>(one(to_float(z[j])));
  }
}

// x or lo, whichever is larger; NaN stays.
__device__ __forceinline__ float max_nan(float x, float lo) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(lo));
  return y;
}

// ---- sums in powers of two ---------------------------------------------
// The streaming form of the sums: the shift is a whole number n of powers
// of two, so that z c - n is one rounded operation (no error from a rounded
// shift, which would scale one thread's terms against another's), and sums
// with different shifts join by exact factors.  h = sum of e x with x = z c
// - n.  n never leaves +-kFar; a row whose largest logit does (all logits
// masked by a finite value, or a very small temperature) is summed by
// add_logit instead.  n is the rounded product: at the largest logit x is what
// the rounding left, up to half a unit of the product's last place.  Within
// 2^27 that is 4, and e at most 16; from 2^32 on it would be 128 and more, e
// infinite, and its product with a joining factor of 0 a NaN.
constexpr float kFar = 1 << 27;

struct Pow2Sums {
  float n, s, h;
};

__device__ __forceinline__ float shift_of(float max, float c) {
  return fminf(fmaxf(rintf(max * c), -kFar), kFar);
}

template <bool ENTROPY>
__device__ __forceinline__ void move_to(Pow2Sums &a, float n) {
  const float f = ex2_approx(a.n - n);
  if (ENTROPY) a.h = f * fmaf(a.n - n, a.s, a.h);
  a.s *= f;
  a.n = n;
}

template <bool ENTROPY>
__device__ __forceinline__ void add_term(Pow2Sums &a, float z, float c) {
  float x = fmaf(z, c, -a.n);
  if (ENTROPY) x = max_nan(x, -1e4f);  // -inf: 0 times a number
  const float e = ex2_approx(x);
  a.s += e;
  if (ENTROPY) a.h = fmaf(e, x, a.h);
}

// Adds the terms of B vectors (shift a.n at their largest logit or above).
// With ENTROPY a masked logit's 0 times -inf shows as NaN in h: from the
// first batch of a warp that has one on (`masked`), x is held above -1e4;
// rows without masks are spared that instruction, one of 8 per pair.
template <bool ENTROPY, bool HOLD, typename T, int B>
__device__ __forceinline__ float add_terms(Pow2Sums &a, const uint4 (&r)[B], float c) {
  constexpr int E = Vec<T>::kElems;
  const Pair c2 = pair(c, c), n2 = pair(-a.n, -a.n);
  Pair s = pair(a.s, 0.0f), h = pair(0.0f, 0.0f);
#pragma unroll
  for (int u = 0; u < B; ++u) {
    Pair z[E / 2];
    Vec<T>::pairs(r[u], z);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      Pair x = fma2(z[e], c2, n2);
      if (HOLD) {
        const float2 f = halves(x);
        x = pair(max_nan(f.x, -1e4f), max_nan(f.y, -1e4f));
      }
      const Pair p = ex2_pair(x);
      s = add2(s, p);
      if (ENTROPY) h = fma2(p, x, h);
    }
  }
  const float2 f = halves(s), g = halves(h);
  a.s = f.x + f.y;
  return g.x + g.y;
}
template <bool ENTROPY, typename T, int B>
__device__ __forceinline__ void add_batch(Pow2Sums &a, const uint4 (&r)[B], float c, bool &masked) {
  if (!ENTROPY) {
    add_terms<false, false, T>(a, r, c);
    return;
  }
  if (!masked) {
    const float s = a.s, h = add_terms<true, false, T>(a, r, c);
    masked = __any_sync(0xffffffffu, h != h);
    if (!masked) {
      a.h += h;
      return;
    }
    a.s = s;
  }
  a.h += add_terms<true, true, T>(a, r, c);
}

// The warp's sums, in every lane.
template <bool ENTROPY>
__device__ __forceinline__ void warp_join(Pow2Sums &a) {
  move_to<ENTROPY>(a, warp_max(a.n));
  a.s = warp_sum(a.s);
  if (ENTROPY) a.h = warp_sum(a.h);
}

// Whether a row of largest logit m is outside what Pow2Sums hold.
__device__ __forceinline__ bool far_out(float m, float c) {
  return m != -INFINITY && !(fabsf(m * c) < kFar);
}

// Sums relative to the largest logit itself.
__device__ __forceinline__ float sum_at(float s, float n, float m, float c) {
  return m == -INFINITY ? s : s * ex2_approx(-fmaf(m, c, -n));
}

// Fewest rows that take a warp each: fewer are a wave of CTAs of three an SM.
// Vocabulary 2048, a warp and a CTA per row: scoring with 32 alternatives,
// 300 rows 6.6 and 4.8 us, 450 rows 6.9 and 7.2, 900 rows 7.4 and 10.8;
// distillation loss and gradient 5.7 and 6.3, 5.8 and 6.9, 6.7 and 11.7.
// Rows above 8 KB leave room for half the warps and need twice the rows
// (8000 bf16: loss and gradient, 600 rows 13.0 and 14.7 us, 800 rows 13.5 and
// 16.0, 1000 rows 14.3 and 17.1, 6000 rows 59 and 85; scoring with 20
// alternatives 11.2 and 10.0, 11.7 and 10.9, 13.6 and 14.1, 42 and 61; the
// gradient of scoring 8.3 and 7.2, 9.0 and 8.1, 9.8 and 11.2; distillation
// loss 8.1 and 6.1, 8.5 and 9.5, 8.9 and 10.2).
constexpr uint32_t kShortRows = 3 * kNumSMs, kShortRowsWide = 6 * kNumSMs;

// ---- short rows: a warp holds a row in shared memory -----------------------
// A row's vectors go to shared memory by cp.async, the next row's while the
// warp finishes the last one; lane l works on vectors l + 32 i, i < NV.
// Shared memory, not registers: 20 and more rows are in flight on an SM, and
// single logits can be looked up and taken out.
constexpr int kShortWarps = 4;  // warps (rows in flight) of a CTA, 6 CTAs an SM
constexpr int kScoreWarps = 3;  // for scoring: 7 CTAs an SM with the lists of alternatives, 9 without

// Vectors of a lane for a row: 4, 16, 32, or 0 where rows are too long or too
// few for a warp each.
inline uint32_t short_vectors(uint32_t rows, uint32_t vocab, size_t type_bytes) {
  const uint64_t vecs = static_cast<uint64_t>(vocab) * type_bytes / 16;
  if (rows < (vecs <= 16 * 32 ? kShortRows : kShortRowsWide)) return 0;
  return vecs <= 4 * 32 ? 4 : vecs <= 16 * 32 ? 16 : vecs <= 32 * 32 ? 32 : 0;
}
// CTAs that fill the SMs, given the shared memory of one (each takes 1 KB
// more): a second, short wave would double the time.
inline unsigned short_grid(uint32_t rows, uint32_t warps, size_t smem) {
  const uint32_t ctas = (rows + warps - 1) / warps;
  size_t per_sm = (227 * 1024) / (smem + 1024);
  if (per_sm > 9) per_sm = 9;
  const uint32_t most = kNumSMs * static_cast<uint32_t>(per_sm);
  return ctas < most ? ctas : most;
}

// f(i, v) for the vectors v = l + 32 i of a lane; rows that fill all NV have
// a loop without conditions.
template <int NV, typename F>
__device__ __forceinline__ void for_vectors(uint32_t end, uint32_t lane, F f) {
  if (end == NV * 32) {
#pragma unroll
    for (int i = 0; i < NV; ++i) f(i, i * 32 + lane);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * 32 + lane < end) f(i, i * 32 + lane);
  }
}

template <typename T, int NV>
__device__ __forceinline__ void stage_row(const T *z, const Part &p, uint32_t lane, uint4 *buffer) {
  const uint4 *vec = reinterpret_cast<const uint4 *>(z + p.head);
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(buffer));
  for_vectors<NV>(p.end, lane, [&](int, uint32_t j) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + j * 16), "l"(vec + j) : "memory");
  });
}
// The staged row is in shared memory, for every lane.
__device__ __forceinline__ void await_row() {
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
}

// dz_j = f(z_j) for the row in shared memory, by pairs; the lane's loose
// element by `one`.
template <typename T, int NV, typename F, typename G>
__device__ __forceinline__ void write_row(T *dz, const Part &p, uint32_t lane, const uint4 *buffer,
                                          float loose, F two, G one) {
  constexpr int E = Vec<T>::kElems;
  const bool aligned = aligned16(dz + p.head);
  const auto values = [&](uint32_t j, Pair (&x)[E / 2]) {
    Vec<T>::pairs(buffer[j], x);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) x[e] = two(x[e]);
  };
  if (aligned) {
    uint4 *out = reinterpret_cast<uint4 *>(dz + p.head);
    for_vectors<NV>(p.end, lane, [&](int, uint32_t j) {
      Pair x[E / 2];
      values(j, x);
      out[j] = Vec<T>::pack_pairs(x);
    });
  } else {
    for (uint32_t j = lane; j < p.end; j += 32) {
      Pair x[E / 2];
      values(j, x);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const float2 y = halves(x[e]);
        dz[p.head + j * E + 2 * e] = from_float<T>(y.x);
        dz[p.head + j * E + 2 * e + 1] = from_float<T>(y.y);
      }
    }
  }
  if (lane < p.loose) dz[loose_at(p, lane)] = from_float<T>(one(loose));
}

inline size_t type_size(int32_t type) { return type == TL_FLOAT32 ? 4 : 2; }

// Checks the fields that both descriptors have; fills in the default
// strides.  TL_OK, or the status that the entry point returns.
int check_rows(const char *who, const void *logits, int32_t type, uint32_t rows, uint32_t vocab,
               float temperature, uint64_t &row_stride);
// The same for the gradient of a backward call.
int check_gradient(const char *who, const void *logits, uint64_t row_stride, void *dlogits,
                   int32_t type, uint32_t rows, uint32_t vocab, uint64_t &d_row_stride);

// CTAs of 256 (a cluster) that share a row: more than one where the rows
// would leave half of the SMs idle and one CTA would have more than four
// vectors a thread.  A cluster costs about 2.5 us over a CTA (64 x 8192
// bf16, 20 alternatives: 6.6 us in clusters of 2, 4.3 us without; 8 x
// 50001: 6.8 and 8.6 us; 128 x 50001: 10.0 and 8.8 us).
constexpr uint32_t kMaxCluster = 8;
uint32_t cluster_parts(uint32_t rows, uint32_t vecs);
// Grid of a gradient without a reduction, CTAs of 256: rows x parts, more
// than one part where the rows alone are fewer than 16 CTAs an SM (two rounds)
// and a part keeps more than eight vectors a thread.  Gradient of scoring,
// bf16, vocabulary 50001, with parts and without: 64 rows 6.8 and 11.5 us, 148
// rows 9.1 and 12.9, 300 rows 14.3 and 16.2, 1200 rows 44.5 and 45.6, 2300
// rows 80.2 and 78.7; fp16, 130000: 300 rows 28.5 and 34.0, 1200 rows 105 and
// 110, 2300 rows 196 and 202; of distillation, bf16, 50001: 148 rows 8.7 and
// 12.1, 600 rows 26.3 and 23.8, 1800 rows 65.4 and 64.1.  Parts up to 4 CTAs an
// SM only: 600 x 130000 59.4 against 54.1; up to 64: 4 % either way.
dim3 gradient_grid(uint32_t rows, uint32_t vecs);

}  // namespace token
}  // namespace tl

#define TL_BY_TYPE(TYPE, LAUNCH)                   \
  switch (TYPE) {                                  \
    case TL_FLOAT32: LAUNCH(float); break;         \
    case TL_FLOAT16: LAUNCH(__half); break;        \
    default: LAUNCH(__nv_bfloat16); break;         \
  }
