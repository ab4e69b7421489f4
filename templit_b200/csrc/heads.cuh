// Rows of attention heads in registers: vector loads and stores of fp32, fp16
// and bf16, angles from 64-bit turns, the rotation of pairs and the norm of a
// head (k_rotary*.cu, k_cache_append.cu).
//
// A head of D elements belongs to `lanes` neighbouring lanes of a warp (a
// power of two), each with S slots of two vectors of V elements: slot p holds
// the V pairs p V .. p V + V - 1 while those are turned, or 2 V elements
// behind the turned ones.  So a rotation needs no exchange between lanes in
// either layout, and the norm one sum over the head's lanes.
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

// V elements of T as they lie in memory, in words of 8 or 16 bytes (V = 1: one
// element).
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
  __device__ __forceinline__ float squares() const {
    float x[V], sum = 0.0f;
    get(x);
#pragma unroll
    for (int i = 0; i < V; ++i) sum = fmaf(x[i], x[i], sum);
    return sum;
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
__device__ __forceinline__ float element_of(float x) { return x; }
__device__ __forceinline__ float element_of(__half x) { return __half2float(x); }
__device__ __forceinline__ float element_of(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void set_element(float &y, float x) { y = x; }
__device__ __forceinline__ void set_element(__half &y, float x) { y = __float2half_rn(x); }
__device__ __forceinline__ void set_element(__nv_bfloat16 &y, float x) { y = __float2bfloat16_rn(x); }
template <typename T> struct Raw<T, 1> {
  T r;
  __device__ __forceinline__ void load(const T *p) { r = *p; }
  __device__ __forceinline__ void store(T *p) const { *p = r; }
  __device__ __forceinline__ void get(float (&x)[1]) const { x[0] = element_of(r); }
  __device__ __forceinline__ float squares() const { return element_of(r) * element_of(r); }
  __device__ __forceinline__ void set(const float (&x)[1]) { set_element(r, x[0]); }
};

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

// Pair i of a slot's two vectors.
template <int V> __device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float (&cos)[V],
                                                      const float (&sin)[V], bool interleaved) {
  if (V == 1 || !interleaved) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float u = a[i], w = b[i];
      a[i] = fmaf(u, cos[i], -(w * sin[i]));
      b[i] = fmaf(u, sin[i], w * cos[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float u = a[2 * i], w = a[2 * i + 1];
      a[2 * i] = fmaf(u, cos[i], -(w * sin[i]));
      a[2 * i + 1] = fmaf(u, sin[i], w * cos[i]);
      const float u2 = b[2 * i], w2 = b[2 * i + 1];
      b[2 * i] = fmaf(u2, cos[V / 2 + i], -(w2 * sin[V / 2 + i]));
      b[2 * i + 1] = fmaf(u2, sin[V / 2 + i], w2 * cos[V / 2 + i]);
    }
  }
}

// Angles of a lane's slots at one position, `magnitude` included; cosine 1
// and sine 0 behind the turned elements.  The lanes at one place of the heads
// that lie side by side in a warp share the work.
template <int V, int S>
__device__ __forceinline__ void angles(const uint64_t *frequencies, uint32_t position, float magnitude,
                                       uint32_t p0, uint32_t lanes, uint32_t rotary, float (&cos)[S][V],
                                       float (&sin)[S][V]) {
  const uint32_t per = 32 / lanes, sub = (threadIdx.x & 31) / lanes;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const uint32_t p = p0 + s * lanes;
    const bool turned = 2 * p * V < rotary;
    float cs[V], sn[V];  // pairs sub, sub + per, ..
#pragma unroll
    for (int r = 0; r < V; ++r) {
      cs[r] = 1.0f;
      sn[r] = 0.0f;
      const uint32_t i = r * per + sub;
      if (r * per < V && i < V && turned) {
        sine_cosine(position * frequencies[p * V + i], sn[r], cs[r]);
        cs[r] *= magnitude;
        sn[r] *= magnitude;
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t from = p0 + lanes * (i & (per - 1));
      // pair i is the (i / per)-th of that lane
      const float c = per == 1 ? cs[i] : per == 2 ? cs[i / 2] : per == 4 ? cs[i / 4] : cs[0];
      const float n = per == 1 ? sn[i] : per == 2 ? sn[i / 2] : per == 4 ? sn[i / 4] : sn[0];
      cos[s][i] = __shfl_sync(0xffffffffu, c, from);
      sin[s][i] = __shfl_sync(0xffffffffu, n, from);
    }
  }
}

// The norm's weights of a lane's slot: 1 without any.
template <int V>
__device__ __forceinline__ void load_weights(const float *w, const Slot &s, float (&a)[V], float (&b)[V]) {
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

// Heads [first, end) of one token from x to out: the norm of each where
// `norm`, the turn of its first `rotary` elements where `turned`.  U head rows
// a lane are loaded before the first is used, the first ones before `angles`
// works out cos and sin.
template <typename TI, typename TO, int V, int S, int U, typename Angles>
__device__ __forceinline__ void run_heads(const TI *x, uint64_t x_stride, TO *out, uint64_t out_stride,
                                          uint32_t first, uint32_t end, uint32_t lanes, uint32_t sub,
                                          const Slot (&slot)[S], const float (&wa)[S][V], const float (&wb)[S][V],
                                          Angles angles, bool norm, bool turned, bool inter, float inv_d, float eps) {
  const uint32_t per = 32 / lanes;
  const uint64_t x_step = per * x_stride, out_step = per * out_stride;
  x += (first + sub) * x_stride;
  out += (first + sub) * out_stride;
  Raw<TI, V> ra[U][S], rb[U][S];
  const auto load = [&](uint32_t h0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = h0 + u * per + sub < end;
      const TI *row = x + u * x_step;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        ra[u][s] = rb[u][s] = Raw<TI, V>{};
        if (there && slot[s].has_a) ra[u][s].load(row + slot[s].a);
        if (there && slot[s].has_b) rb[u][s].load(row + slot[s].b);
      }
    }
    x += U * x_step;
  };
  load(first);
  float cos[S][V], sin[S][V];
  angles(cos, sin);
  for (uint32_t h0 = first; h0 < end; h0 += U * per) {
    if (h0 != first) load(h0);
    float r[U];
    if (norm) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        r[u] = 0.0f;
#pragma unroll
        for (int s = 0; s < S; ++s) r[u] += ra[u][s].squares() + rb[u][s].squares();
      }
      head_sums<U>(r, lanes);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool there = h0 + u * per + sub < end;
      float va[S][V], vb[S][V];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        ra[u][s].get(va[s]);
        rb[u][s].get(vb[s]);
      }
      if (norm) {
        const float f = rsqrtf(fmaf(r[u], inv_d, eps));
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            va[s][i] *= f * wa[s][i];
            vb[s][i] *= f * wb[s][i];
          }
      }
      TO *row = out + u * out_step;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (turned && slot[s].turned) turn<V>(va[s], vb[s], cos[s], sin[s], inter);
        Raw<TO, V> y;
        if (there && slot[s].has_a) {
          y.set(va[s]);
          y.store(row + slot[s].a);
        }
        if (there && slot[s].has_b) {
          y.set(vb[s]);
          y.store(row + slot[s].b);
        }
      }
    }
    out += U * out_step;
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
// one that is written has no two rows in one place.
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
