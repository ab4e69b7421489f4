// Rows of attention heads in registers: vector loads and stores of fp32, fp16
// and bf16, angles from 64-bit turns, the rotation of pairs and the norm of a
// head (k_rotary*.cu, k_cache_append.cu).
//
// A head of D elements belongs to `lanes` neighbouring lanes of a warp (a
// power of two), each with a slot of two vectors of V elements: slot p holds
// the V pairs p V .. p V + V - 1 while those are turned, or 2 V elements
// behind the turned ones.  So a rotation needs no exchange between lanes in
// either layout, and the norm one sum over the head's lanes.  Heads that vectors do
// not fit go by single elements (scalar_head).
#pragma once

#include "tl_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace tl {
namespace heads {

inline size_t type_size(int32_t type) { return type == TL_FLOAT32 ? 4 : 2; }
// Elements of a vector: 16 bytes of each, and of the smaller where the types
// differ 8 (12288 x 12 heads of 64 fp32 with 8 elements a vector 37 us, with 4 25).
constexpr int vector_of(size_t in, size_t out) { return in == 2 && out == 2 ? 8 : 4; }
inline int vector_for(int32_t in, int32_t out) { return vector_of(type_size(in), type_size(out)); }
inline bool known_type(int32_t type) { return type >= TL_FLOAT32 && type <= TL_BFLOAT16; }

// V elements of T as they lie in memory, in words of 8 or 16 bytes.
template <typename T, int V> struct Raw {
  using Word = typename std::conditional<V * sizeof(T) % 16 == 0, uint4, uint2>::type;
  static constexpr int kWords = V * sizeof(T) / sizeof(Word);
  Word r[kWords];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) r[i] = reinterpret_cast<const Word *>(p)[i];
  }
  __device__ __forceinline__ void store(T *p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<Word *>(p)[i] = r[i];
  }
  __device__ __forceinline__ void get(float (&x)[V]) const {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(r);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        float2 f;
        if constexpr (std::is_same<T, __half>::value) f = __half22float2(reinterpret_cast<const __half2 &>(w[i]));
        else f = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162 &>(w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  // the one rounding of a result (to nearest even)
  __device__ __forceinline__ void set(const float (&x)[V]) {
    uint32_t *w = reinterpret_cast<uint32_t *>(r);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if constexpr (std::is_same<T, __half>::value)
          reinterpret_cast<__half2 &>(w[i]) = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        else
          reinterpret_cast<__nv_bfloat162 &>(w[i]) = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      }
    }
  }
};
// Two fp32 in a register pair: one issued instruction for both.
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
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float sum2(Pair p) {
  const float2 f = halves(p);
  return f.x + f.y;
}
template <typename T, int V> __device__ __forceinline__ void get_pairs(const Raw<T, V> &r, Pair (&x)[V / 2]) {
  float f[V];
  r.get(f);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) x[i] = pair(f[2 * i], f[2 * i + 1]);
}
template <typename T, int V> __device__ __forceinline__ void set_pairs(Raw<T, V> &r, const Pair (&x)[V / 2]) {
  float f[V];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 h = halves(x[i]);
    f[2 * i] = h.x;
    f[2 * i + 1] = h.y;
  }
  r.set(f);
}
__device__ __forceinline__ float element_of(float x) { return x; }
__device__ __forceinline__ float element_of(__half x) { return __half2float(x); }
__device__ __forceinline__ float element_of(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void set_element(float &y, float x) { y = x; }
__device__ __forceinline__ void set_element(__half &y, float x) { y = __float2half_rn(x); }
__device__ __forceinline__ void set_element(__nv_bfloat16 &y, float x) { y = __float2bfloat16_rn(x); }
// Sine and cosine of `turns` / 2^64 of a full turn.  The quarter turn is split
// off exactly in whole numbers; what is left, |x| <= pi / 4, goes through the
// Taylor series, whose first terms left out are x^11 / 11! < 1.8e-9 and
// x^10 / 10! < 2.5e-8 (a quarter of fp32's unit at cos x > 0.7).
__device__ __forceinline__ void sine_cosine(uint64_t turns, float &s, float &c) {
  const uint32_t quarter = static_cast<uint32_t>((turns + (1ull << 61)) >> 62);
  const int64_t rest = static_cast<int64_t>(turns - (static_cast<uint64_t>(quarter) << 62));
  const float x = __ll2float_rn(rest) * 3.4061215800304e-19f;  // 2 pi / 2^64
  const float y = x * x;
  float a = fmaf(y, 2.7557319e-6f, -1.9841270e-4f);  // 1/9!, -1/7!
  a = fmaf(y, a, 8.3333333e-3f);                      // 1/5!
  a = fmaf(y, a, -1.6666667e-1f);                     // -1/3!
  a = fmaf(x * y, a, x);
  float b = fmaf(y, 2.4801587e-5f, -1.3888889e-3f);  // 1/8!, -1/6!
  b = fmaf(y, b, 4.1666667e-2f);                      // 1/4!
  b = fmaf(y, b, -0.5f);
  b = fmaf(y, b, 1.0f);
  const bool swap = quarter & 1u;
  s = swap ? b : a;
  c = swap ? a : b;
  if (quarter & 2u) s = -s;
  if ((quarter + 1u) & 2u) c = -c;
}

// Where a lane's slot lies in a head.
struct Slot {
  uint32_t a, b;  // first element of its two vectors
  bool turned, has_a, has_b;
};
__device__ __forceinline__ Slot slot_of(uint32_t p, uint32_t V, uint32_t D, uint32_t rotary, bool interleaved) {
  Slot s;
  s.turned = 2 * p * V < rotary;
  s.a = s.turned && !interleaved ? p * V : 2 * p * V;
  s.b = s.turned && !interleaved ? rotary / 2 + p * V : 2 * p * V + V;
  s.has_a = s.a < D && 2 * p * V < D;
  s.has_b = s.has_a && s.b < D;
  return s;
}

// A lane's slot turned, in register pairs (the gradient, which has more to do
// for an element than memory gives it time).  HALF: elements i of a and of b are a
// pair; INTERLEAVED: neighbours are.
template <int V> struct Turn {
  Pair a1[V / 2], a2[V / 2], b1[V / 2], b2[V / 2];
  __device__ __forceinline__ void set(const float (&cos)[V], const float (&sin)[V], bool interleaved) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if (!interleaved) {  // a' = a a1 + b a2, b' = a b1 + b b2
        a1[i] = b2[i] = pair(cos[2 * i], cos[2 * i + 1]);
        a2[i] = pair(-sin[2 * i], -sin[2 * i + 1]);
        b1[i] = pair(sin[2 * i], sin[2 * i + 1]);
      } else {  // (a0, a1)' = (a0, a1) a1 + (a1, a0) a2, likewise b
        const int j = V / 2 + i;
        a1[i] = pair(cos[i], cos[i]);
        a2[i] = pair(-sin[i], sin[i]);
        b1[i] = pair(cos[j], cos[j]);
        b2[i] = pair(-sin[j], sin[j]);
      }
    }
  }
  // (elements behind the turned ones stay apart: 0 times a neighbour's NaN is NaN)
  __device__ __forceinline__ void apply(Pair (&a)[V / 2], Pair (&b)[V / 2], bool turned, bool interleaved) const {
    if (!turned) return;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if (!interleaved) {
        const Pair x = a[i], y = b[i];
        a[i] = fma2(x, a1[i], mul2(y, a2[i]));
        b[i] = fma2(x, b1[i], mul2(y, b2[i]));
      } else {
        const float2 x = halves(a[i]), y = halves(b[i]);
        a[i] = fma2(a[i], a1[i], mul2(pair(x.y, x.x), a2[i]));
        b[i] = fma2(b[i], b1[i], mul2(pair(y.y, y.x), b2[i]));
      }
    }
  }
};

// Angles of a lane's slot p0 at one position, `magnitude` included; cosine 1
// and sine 0 behind the turned elements.  The `PER` lanes at one place of the heads
// that lie side by side in a warp share the work.
template <int V, int PER>
__device__ __forceinline__ void shared_angles(const uint64_t *frequencies, uint32_t position, float magnitude, uint32_t p0,
                                              uint32_t lanes, uint32_t rotary, float (&cos)[V], float (&sin)[V]) {
  constexpr int N = V > PER ? V / PER : 1;  // a lane's: pairs sub, sub + PER, ..
  const uint32_t sub = (threadIdx.x & 31) / lanes;
  const bool turned = 2 * p0 * V < rotary;
  float cs[N], sn[N];
#pragma unroll
  for (int r = 0; r < N; ++r) {
    cs[r] = 1.0f;
    sn[r] = 0.0f;
    const uint32_t i = r * PER + sub;
    if (i < V && turned) {
      sine_cosine(position * frequencies[p0 * V + i], sn[r], cs[r]);
      cs[r] *= magnitude;
      sn[r] *= magnitude;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    cos[i] = PER == 1 ? cs[i % N] : __shfl_sync(0xffffffffu, cs[i / PER], p0 + lanes * (i % PER));
    sin[i] = PER == 1 ? sn[i % N] : __shfl_sync(0xffffffffu, sn[i / PER], p0 + lanes * (i % PER));
  }
}
template <int V>
__device__ __forceinline__ void angles(const uint64_t *frequencies, uint32_t position, float magnitude, uint32_t p0,
                                       uint32_t lanes, uint32_t rotary, float (&cos)[V], float (&sin)[V]) {
  if (lanes == 8) shared_angles<V, 4>(frequencies, position, magnitude, p0, lanes, rotary, cos, sin);
  else if (lanes <= 4) shared_angles<V, 8>(frequencies, position, magnitude, p0, lanes, rotary, cos, sin);
  else if (lanes == 16) shared_angles<V, 2>(frequencies, position, magnitude, p0, lanes, rotary, cos, sin);
  else shared_angles<V, 1>(frequencies, position, magnitude, p0, lanes, rotary, cos, sin);
}

// The norm's weights of a lane's slot: 1 without any.
template <int V>
__device__ __forceinline__ void load_weights(const float *w, const Slot &s, float (&a)[V], float (&b)[V]) {
  if (w && aligned16(w)) {  // slots begin at whole vectors
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 one = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
      const float4 x = s.has_a ? *reinterpret_cast<const float4 *>(w + s.a + i) : one;
      const float4 y = s.has_b ? *reinterpret_cast<const float4 *>(w + s.b + i) : one;
      a[i] = x.x, a[i + 1] = x.y, a[i + 2] = x.z, a[i + 3] = x.w;
      b[i] = y.x, b[i + 1] = y.y, b[i + 2] = y.z, b[i + 3] = y.w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    a[i] = w && s.has_a ? w[s.a + i] : 1.0f;
    b[i] = w && s.has_b ? w[s.b + i] : 1.0f;
  }
}

// Sums over the `lanes` lanes of a head (a power of two), in each of them; all
// of them step by step together, so that one's shuffles cover the others'.
template <int N> __device__ __forceinline__ void head_sums(float (&x)[N], uint32_t lanes) {
#pragma unroll
  for (uint32_t o = 1; o < 32; o <<= 1) {
    if (o >= lanes) break;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
  }
}

// A lane's part of a head: normed (f the norm's factor), turned, rounded.
template <typename TI, typename TO, int V>
__device__ __forceinline__ void finish_head(const Raw<TI, V> &ra, const Raw<TI, V> &rb, const Slot &slot, const float (&cos)[V],
                                            const float (&sin)[V], const float (&wa)[V], const float (&wb)[V], float f, bool norm,
                                            bool inter, bool there, TO *row) {
  float a[V], b[V];
  ra.get(a);
  rb.get(b);
  if (norm) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      a[i] *= f * wa[i];
      b[i] *= f * wb[i];
    }
  }
  if (slot.turned) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      // pair i: elements i of both vectors, or neighbours in one
      float &u = !inter ? a[i] : i < V / 2 ? a[2 * i] : b[2 * i - V], &w = !inter ? b[i] : i < V / 2 ? a[2 * i + 1] : b[2 * i + 1 - V];
      const float u0 = u, w0 = w;
      u = fmaf(u0, cos[i], -(w0 * sin[i]));
      w = fmaf(u0, sin[i], w0 * cos[i]);
    }
  }
  Raw<TO, V> y;
  if (there && slot.has_a) {
    y.set(a);
    y.store(row + slot.a);
  }
  if (there && slot.has_b) {
    y.set(b);
    y.store(row + slot.b);
  }
}
template <typename T, int V> __device__ __forceinline__ float squares(const Raw<T, V> &ra, const Raw<T, V> &rb) {
  float a[V], b[V], sum = 0.0f;
  ra.get(a);
  rb.get(b);
#pragma unroll
  for (int i = 0; i < V; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
  return sum;
}

// One head by single elements, a warp, lane + 32 s the slots of two elements:
// any size, alignment and type.
template <typename TI, typename TO>
__device__ __forceinline__ void scalar_head(const TI *x, TO *out, uint32_t D, uint32_t rotary, const uint64_t *frequencies,
                                            uint32_t position, float magnitude, const float *weight, bool norm, bool inter,
                                            float inv_d, float eps) {
  constexpr int S = TL_HEAD_MAX_DIM / 64;
  const uint32_t lane = threadIdx.x & 31;
  float a[S], b[S], sum[1] = {0.0f};
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const Slot slot = slot_of(lane + 32 * s, 1, D, rotary, inter);
    a[s] = slot.has_a ? element_of(x[slot.a]) : 0.0f;
    b[s] = slot.has_b ? element_of(x[slot.b]) : 0.0f;
    sum[0] = fmaf(a[s], a[s], fmaf(b[s], b[s], sum[0]));
  }
  float f = 1.0f;
  if (norm) {
    head_sums<1>(sum, 32);
    f = rsqrtf(fmaf(sum[0], inv_d, eps));
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const Slot slot = slot_of(lane + 32 * s, 1, D, rotary, inter);
    float u = a[s], w = b[s];
    if (norm) {
      u *= f * (weight && slot.has_a ? weight[slot.a] : 1.0f);
      w *= f * (weight && slot.has_b ? weight[slot.b] : 1.0f);
    }
    if (slot.turned) {
      float sn, cs;
      sine_cosine(position * frequencies[lane + 32 * s], sn, cs);
      const float c = cs * magnitude, n = sn * magnitude, u0 = u;
      u = fmaf(u, c, -(w * n));
      w = fmaf(u0, n, w * c);
    }
    if (slot.has_a) set_element(out[slot.a], u);
    if (slot.has_b) set_element(out[slot.b], w);
  }
}

// The lanes a head takes and the vectors that may be used for it.
struct Shape {
  uint32_t lanes;
  bool vectors;
};
// Vectors of V elements; rotated pairs and the rest have to come in whole ones.
inline Shape shape_for(uint32_t D, uint32_t rotary, uint32_t V, bool aligned) {
  Shape s{32, aligned && D % V == 0 && (rotary / 2) % V == 0 && (D - rotary) % V == 0};
  if (s.vectors) {
    s.lanes = 1;
    while (s.lanes * 2 * V < D) s.lanes *= 2;
  }
  return s;
}
// Whether every row of a view starts on the boundary that its words of up to 16
// bytes ask for, of vectors of V elements.
inline bool aligned_view(const tl_head_view &v, int32_t type, bool batches, uint32_t V) {
  const uint64_t bytes = V * type_size(type) < 16 ? V * type_size(type) : 16, e = bytes / type_size(type);
  return reinterpret_cast<uintptr_t>(v.p) % bytes == 0 && (!batches || v.batch_stride % e == 0) && v.head_stride % e == 0 &&
         v.row_stride % e == 0;
}

// Checks that the rotation's fields of several descriptors share.
int check_turn(const char *who, uint32_t D, uint32_t rotary_dim, int32_t layout, int32_t norm, float eps,
               float magnitude, const uint64_t *frequencies);
// A view of [batches, rows, heads, D] of `type`: pointer, alignment, extent;
// no stride of one that is written is 0 or below D (whether larger ones meet is not
// worked out: a caller's).
int check_view(const char *who, const char *name, const tl_head_view &v, int32_t type, uint64_t batches,
               uint64_t rows, uint64_t heads, uint32_t D, bool written);
// In place or apart: one pointer means one layout and one type.
inline bool half_in_place(const tl_head_view &a, int32_t ta, const tl_head_view &b, int32_t tb, bool batches) {
  return a.p == b.p && (ta != tb || a.head_stride != b.head_stride || a.row_stride != b.row_stride ||
                        (batches && a.batch_stride != b.batch_stride));
}

// LAUNCH(TI, TO) for the pairs of types that the entry points take.
#define TL_BY_TYPES(IN, OUT, LAUNCH)                                             \
  switch ((IN) * 3 + (OUT)) {                                                    \
    case 0: LAUNCH(float, float); break;                                         \
    case 1: LAUNCH(float, __half); break;                                        \
    case 2: LAUNCH(float, __nv_bfloat16); break;                                 \
    case 3: LAUNCH(__half, float); break;                                        \
    case 4: LAUNCH(__half, __half); break;                                       \
    case 6: LAUNCH(__nv_bfloat16, float); break;                                 \
    default: LAUNCH(__nv_bfloat16, __nv_bfloat16); break;                        \
  }
inline bool mixed_halves(int32_t in, int32_t out) { return in != out && in != TL_FLOAT32 && out != TL_FLOAT32; }

}  // namespace heads
}  // namespace tl
