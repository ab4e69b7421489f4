// Attention over a paged cache for few query rows a key head (single tokens
// and short runs of them, any type; include/templit_cuda.h:
// tl_paged_attention).
//
// Bound by memory: every key and value is read once for up to 16 query rows
// (a token's heads that share a key head lie side by side), so the rows' own
// arithmetic is small and mma.sync (fp32: the CUDA cores) is enough.  A warp works
// alone: it brings 16 keys and values (8 of 32 bits) at a time into its own ring in
// shared memory by cp.async, several steps ahead, multiplies and keeps its rows'
// maxima, sums and outputs in registers; no barrier but the warp's own until its
// share of a job is done, when the CTA's warps join in shared memory.  Shares
// of the keys and their joining: paged_attention.cuh.
//
// 8 key heads of 128 bf16, 4 query heads each: one token over 200003 keys 135 us
// (819 MB, 6.1 TB/s); 64 sequences of 16 to 8191 keys 92 us (5.0 TB/s), where a CTA's
// jobs' starts and ends, between which its loads pause, are what is left.  Chunks in fp32 read
// a sequence's keys once for 16 rows: 64 sequences of 192 tokens, 6 heads of 64: 433 us; one
// prompt of 2048: 508 us (6.4 TFLOP/s).
#include "paged_attention.cuh"

namespace tl {
namespace paged {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr uint32_t kRows = 16;
// Blocks of a share, where there is that much: one token over 1023 keys 17, 20 and 34 us
// with 1, 4 and 16, 512 sequences of 16 to 511 keys 150, 147 and 147.
constexpr uint32_t kLeast = 4;

// Keys of a warp's step.
template <typename T> constexpr uint32_t step_keys() { return sizeof(T) == 2 ? 16 : 8; }

constexpr int kStages = 3;
template <typename T, int DP> constexpr uint32_t stage_bytes() { return 2 * step_keys<T>() * DP * sizeof(T); }
// fp32: the queries and the warps' probabilities too
template <typename T, int DP> constexpr size_t smem_bytes() {
  return static_cast<size_t>(kWarps) * kStages * stage_bytes<T, DP>() +
         (sizeof(T) == 4 ? (kRows * DP + kWarps * kRows * 8) * sizeof(float) : 0);
}

__device__ __forceinline__ void load_matrices(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_transposed(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ float4 load_vector(uint32_t at) {
  float4 x;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
  return x;
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// What a row of the tile sees.
struct Bounds {
  uint32_t from[kRows], to[kRows];
};

// A warp's rows of 16-bit types, m16n8k16: lane i holds rows i / 4 and i / 4 + 8.
template <typename T, int DP> struct Lane {
  static constexpr int KS = DP / 16;
  static constexpr uint32_t N = 16, kHalf = N * DP * 2;
  // Numerators are at most 2^kShift, so that fp16's small ones keep their bits
  // (normal down to 2^-28 of the largest).
  static constexpr float kShift = std::is_same<T, __half>::value ? 14.0f : 0.0f;
  uint32_t q[KS][4];  // the first product's left operand
  float m[2], l[2], o[DP / 8][4];

  static __device__ __forceinline__ uint32_t spot(uint32_t row, uint32_t ch) { return row * (DP * 2) + ((ch ^ (row & 7)) << 4); }

  __device__ __forceinline__ void begin(const AttentionArgs &a, const Piece &w, float *) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t row = lane / 4 + 8 * i;
      const uint32_t place = w.row0 + row;
      const T *p = static_cast<const T *>(a.q.p) + (w.start + static_cast<uint64_t>(place / a.group)) * a.q.row_stride +
                   (w.head * a.group + place % a.group) * a.q.head_stride;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t d = k * 16 + j * 8 + (lane & 3) * 2;
          q[k][i + 2 * j] = row <= w.last && d < a.cache.D ? *reinterpret_cast<const uint32_t *>(p + d) : 0u;
        }
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  }

  __device__ __forceinline__ void step(const AttentionArgs &a, uint32_t from, uint32_t key, unsigned good, bool full,
                                       uint32_t, const Bounds &bounds, float *) {
    const uint32_t lane = threadIdx.x & 31;
    const float scale = a.scale * kLog2e;
    float x[2][4] = {};
    {
      const uint32_t row = (lane >> 4) * 8 + (lane & 7), ch = (lane >> 3) & 1;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t b[4];
        load_matrices(from + spot(row, k * 2 + ch), b);
        mma16<T>(x[0], q[k], b[0], b[1]);
        mma16<T>(x[1], q[k], b[2], b[3]);
      }
    }
    // element e of x[n]: row lane / 4 + 8 (e / 2), key 8 n + 2 (lane & 3) + (e & 1)
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[n][e] *= scale;
        if (!full) {
          const uint32_t i = n * 8 + (lane & 3) * 2 + (e & 1), j = key + i, row = lane / 4 + 8 * (e >> 1);
          if (!(good >> i & 1) || j < bounds.from[row] || j >= bounds.to[row]) x[n][e] = -INFINITY;
        }
        top[e >> 1] = fmaxf(top[e >> 1], x[n][e]);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2)) - kShift;
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float now = fmaxf(m[i], top[i]);
        const float f = now == m[i] ? 1.0f : ex2_approx(m[i] - now);
        m[i] = now;
        l[i] *= f;
#pragma unroll
        for (int d = 0; d < DP / 8; ++d) {
          o[d][2 * i] *= f;
          o[d][2 * i + 1] *= f;
        }
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
    for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[n][e] = ex2_approx(x[n][e] - base[e >> 1]);
        l[e >> 1] += x[n][e];
      }
    // the numerators' rounding to the type, which the matrix instructions ask for;
    // their sum stays in fp32
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = x[i >> 1][(i & 1) * 2], hi = x[i >> 1][(i & 1) * 2 + 1];
      if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2 &>(p[i]) = __floats2half2_rn(lo, hi);
      else reinterpret_cast<__nv_bfloat162 &>(p[i]) = __floats2bfloat162_rn(lo, hi);
    }
    const uint32_t row = lane & 15, ch = lane >> 4;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      uint32_t b[4];
      load_transposed(from + kHalf + spot(row, d * 2 + ch), b);
      mma16<T>(o[2 * d], p, b[0], b[1]);
      mma16<T>(o[2 * d + 1], p, b[2], b[3]);
    }
  }

  // outs: [row][DP]
  __device__ __forceinline__ void leave(uint32_t, float *outs, float *ms, float *ls) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t row = lane / 4 + 8 * i;
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
        *reinterpret_cast<float2 *>(outs + row * DP + d * 8 + (lane & 3) * 2) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
      if ((lane & 3) == 0) {
        ms[row] = m[i];
        ls[row] = l[i];
      }
    }
  }
};

// fp32 on the CUDA cores (split into tf32 parts on the tensor cores the
// output was 1.0e-6 from the exact one where this is at 2e-7): four lanes a
// key for the scores, every lane a few elements of all rows for the output.
template <int DP> struct Lane<float, DP> {
  static constexpr uint32_t N = 8, kHalf = N * DP * 4;
  static constexpr int V = DP / 16;  // vectors of a lane's part of a key
  static constexpr int E = DP / 32;  // elements of the output that a lane has
  float m[kRows], l[kRows], o[kRows][E];

  // lanes 0..7 read two keys at once
  static __device__ __forceinline__ uint32_t spot(uint32_t row, uint32_t ch) { return row * (DP * 4) + ((ch ^ ((row & 1) << 2)) << 4); }

  // shared: the queries, negated where the scale is negative, then each warp's probabilities
  __device__ __forceinline__ void begin(const AttentionArgs &a, const Piece &w, float *shared) {
    const float sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
    for (uint32_t i = threadIdx.x; i < kRows * DP; i += kThreads) {
      const uint32_t row = i / DP, d = i % DP;
      const uint32_t place = w.row0 + row;
      float x = 0.0f;
      if (row <= w.last && d < a.cache.D)
        x = sign * (static_cast<const float *>(a.q.p) + (w.start + static_cast<uint64_t>(place / a.group)) * a.q.row_stride +
                    (w.head * a.group + place % a.group) * a.q.head_stride)[d];
      shared[i] = x;
    }
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[r][e] = 0.0f;
    }
  }

  __device__ __forceinline__ void step(const AttentionArgs &a, uint32_t from, uint32_t key, unsigned good, bool full,
                                       uint32_t last, const Bounds &bounds, float *shared) {
    const uint32_t lane = threadIdx.x & 31, k = lane >> 2, part = lane & 3;
    const float c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * kLog2e;
    const uint32_t queries = static_cast<uint32_t>(__cvta_generic_to_shared(shared));
    float *const p = shared + kRows * DP + threadIdx.x / 32 * kRows * 8;
    float4 x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = load_vector(from + spot(k, i * 4 + part));
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
      if (r > last) break;
      float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float4 q = load_vector(queries + (r * DP + (i * 4 + part) * 4) * 4);
        s0 = fmaf(x[i].x, q.x, s0);
        s1 = fmaf(x[i].y, q.y, s1);
        s2 = fmaf(x[i].z, q.z, s2);
        s3 = fmaf(x[i].w, q.w, s3);
      }
      float s = (s0 + s1) + (s2 + s3);
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      if (!full && (!(good >> k & 1) || key + k < bounds.from[r] || key + k >= bounds.to[r])) s = -INFINITY;
      float top = s;
#pragma unroll
      for (int i = 4; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
      top *= c;
      if (top > m[r]) {
        const float f = ex2_approx(m[r] - top);
        m[r] = top;
        l[r] *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[r][e] *= f;
      }
      const float e = ex2_approx(fmaf(s, c, m[r] == -INFINITY ? 0.0f : -m[r]));
      l[r] += e;
      if (part == 0) p[r * 8 + k] = e;
    }
    __syncwarp();
    float v[N][E];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
      const uint32_t at = from + kHalf + spot(i, lane * E / 4) + lane * E % 4 * 4;
      if constexpr (E == 4) {
        const float4 y = load_vector(at);
        v[i][0] = y.x, v[i][1] = y.y, v[i][2] = y.z, v[i][3] = y.w;
      } else {
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[i][0]), "=f"(v[i][1]) : "r"(at) : "memory");
      }
    }
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
      if (r > last) break;
      const float4 p0 = reinterpret_cast<const float4 *>(p + r * 8)[0], p1 = reinterpret_cast<const float4 *>(p + r * 8)[1];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float y = fmaf(p0.x, v[0][e], o[r][e]);
        y = fmaf(p0.y, v[1][e], y);
        y = fmaf(p0.z, v[2][e], y);
        y = fmaf(p0.w, v[3][e], y);
        y = fmaf(p1.x, v[4][e], y);
        y = fmaf(p1.y, v[5][e], y);
        y = fmaf(p1.z, v[6][e], y);
        o[r][e] = fmaf(p1.w, v[7][e], y);
      }
    }
  }

  __device__ __forceinline__ void leave(uint32_t last, float *outs, float *ms, float *ls) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
      if (r > last) break;
#pragma unroll
      for (int i = 4; i < 32; i <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], i);
#pragma unroll
      for (int e = 0; e < E; ++e) outs[r * DP + lane * E + e] = o[r][e];
      if (lane == 0) {
        ms[r] = m[r];
        ls[r] = l[r];
      }
    }
  }
};

template <typename T, typename TO, int DP>
__global__ void __launch_bounds__(kThreads, 2) step_kernel(const AttentionArgs a) {
  using L = Lane<T, DP>;
  constexpr uint32_t N = L::N;                 // keys of a warp's step
  constexpr uint32_t KEYS = N * kWarps;        // of a block
  constexpr uint32_t E = 16 / sizeof(T);       // elements of a vector
  constexpr uint32_t CH = DP / E;              // vectors of a row
  constexpr uint32_t kHalf = L::kHalf;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows];
  __shared__ Bounds bounds;
  float *const shared = reinterpret_cast<float *>(smem + kWarps * kStages * 2 * kHalf);
  pdl_enter();
  const tl_paged_cache &c = a.cache;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const Share share = share_of<kRows, KEYS, kThreads>(a, blockIdx.x, gridDim.x, a.whole ? 1 : kLeast * KEYS);
  Join join{0xffffffffu, 0, 0, 0};
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kStages * 2 * kHalf;

  Walk<kRows, KEYS> walk;
  Piece w;
  walk.start(a, share);
  while (walk.next(a, share, w)) {
    // rows
    const uint32_t head = w.head, last = w.last;
    const uint32_t row0 = w.row0;
    uint32_t all_from = w.from, all_to = w.to, most_from, least_to, f, t;
    seen(a, w.length, w.position(a, 0), f, least_to);
    seen(a, w.length, w.position(a, last), most_from, t);
    const bool uneven = all_from != most_from || all_to != least_to;
    if (threadIdx.x < kRows) {
      uint32_t from = 0, to = 0;
      if (threadIdx.x <= last) seen(a, w.length, w.position(a, threadIdx.x), from, to);
      bounds.from[threadIdx.x] = from;
      bounds.to[threadIdx.x] = to;
    }
    const uint32_t key_hi = static_cast<uint32_t>(min(static_cast<uint64_t>(w.block_hi) * KEYS, static_cast<uint64_t>(all_to)));
    // this warp's steps: keys first_key + i KEYS
    const uint32_t first_key = w.block_lo * KEYS + warp * N;
    const uint32_t steps = first_key < key_hi ? (key_hi - first_key + KEYS - 1) / KEYS : 0;

    L rows;
    rows.begin(a, w, shared);
    __syncthreads();
    const T *kp = static_cast<const T *>(c.k) + head * c.head_stride;
    const T *vp = static_cast<const T *>(c.v) + head * c.head_stride;
    // where lane i's key of a step lies, -1 where there is none
    const auto offset_of = [&](uint32_t step) -> int64_t {
      const uint32_t j = first_key + step * KEYS + lane;
      return step < steps && lane < N && j >= all_from && j < key_hi ? key_offset(a, w.sequence, j) : -1;
    };
    const auto bring = [&](uint32_t step, int64_t from) {
      const uint32_t to = ring + (step % kStages) * 2 * kHalf;
#pragma unroll
      for (uint32_t i = 0; i < N * CH / 32; ++i) {
        const uint32_t row = (lane + 32 * i) / CH, ch = (lane + 32 * i) % CH;
        const int64_t place = __shfl_sync(0xffffffffu, from, row);
        const bool there = place >= 0 && ch * E < c.D;
        // (a copy of nothing gets an address that exists too)
        const T *const k_from = there ? kp + place + ch * E : static_cast<const T *>(a.q.p);
        const T *const v_from = there ? vp + place + ch * E : static_cast<const T *>(a.q.p);
        const uint32_t spot = to + L::spot(row, ch);
        copy16(spot, k_from, there);
        copy16(spot + kHalf, v_from, there);
      }
    };
    unsigned good[kStages];  // a bit for every key that is there
    int64_t next = offset_of(0);
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      good[i] = __ballot_sync(0xffffffffu, next >= 0);
      if (static_cast<uint32_t>(i) < steps) bring(i, next);
      commit();
      next = offset_of(i + 1);
    }
    for (uint32_t step0 = 0; step0 < steps; step0 += kStages) {
#pragma unroll
      for (int u = 0; u < kStages; ++u) {
        const uint32_t step = step0 + u;
        if (step >= steps) break;
        good[(u + kStages - 1) % kStages] = __ballot_sync(0xffffffffu, next >= 0);
        if (step + kStages - 1 < steps) bring(step + kStages - 1, next);
        commit();
        next = offset_of(step + kStages);
        await<kStages - 1>();
        __syncwarp();
        const uint32_t from = ring + u * 2 * kHalf, key = first_key + step * KEYS;
        const bool full = good[u] == (1u << N) - 1 && key >= most_from && key + N <= least_to;
        rows.step(a, from, key, good[u], full, last, bounds, shared);
        __syncwarp();
      }
    }
    await<0>();
    // the CTA's warps into one: outputs through the ring, a row's four warps by one warp
    __syncthreads();
    float *const outs = reinterpret_cast<float *>(smem);  // [warp][row][DP]
    rows.leave(last, outs + warp * kRows * DP, sm_m[warp], sm_l[warp]);
    __syncthreads();
    float *const part = a.parts + (static_cast<size_t>(blockIdx.x) * 2 + (w.opens ? 1 : 0)) * part_floats<kRows, DP>();
    for (uint32_t row = warp; row <= last; row += kWarps) {
      float mm = sm_m[0][row], ll = 0.0f, acc[DP / 32];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) mm = fmaxf(mm, sm_m[i][row]);
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) acc[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        // nothing seen: a sum of 0 (a maximum passes NaN by: of nothing else it is -inf too)
        const float wl = sm_l[i][row];
        if (wl == 0.0f) continue;
        const float f = ex2_approx(sm_m[i][row] - mm);
        ll = fmaf(f, wl, ll);
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) acc[e] = fmaf(f, outs[(i * kRows + row) * DP + lane + 32 * e], acc[e]);
      }
      const uint32_t place = row0 + row, h = head * a.group + place % a.group;
      const uint64_t token = w.start + static_cast<uint64_t>(place / a.group);
      bool nan = false;
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) nan = nan || (lane + 32 * e < c.D && acc[e] != acc[e]);
      if (uneven && ll == ll && __any_sync(0xffffffffu, nan)) {
        // Where a value that other rows of the tile see, and this one does not, is not
        // finite (0 times it is NaN): the row's own keys one by one.
        const uint32_t lo = max(all_from, w.block_lo * KEYS);
        seen(a, w.length, w.position(a, row), f, t);
        if (any_infinite<T>(a, w.sequence, head, lo, min(f, key_hi), lane) ||
            any_infinite<T>(a, w.sequence, head, max(t, lo), key_hi, lane)) {
          float again[kMaxHead / 32];
          const T *q = static_cast<const T *>(a.q.p) + token * a.q.row_stride + h * a.q.head_stride;
          row_over_keys<T>(a, w.sequence, head, q, max(f, lo), min(t, key_hi), lane, mm, ll, again);
#pragma unroll
          for (int e = 0; e < DP / 32; ++e) acc[e] = again[e];
        }
      }
      if (w.opens && w.ends) {
        TO *out = static_cast<TO *>(const_cast<void *>(a.out.p)) + token * a.out.row_stride + h * a.out.head_stride;
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
          if (lane + 32 * e < c.D) heads::set_element(out[lane + 32 * e], ll == 0.0f ? 0.0f : acc[e] / ll);
        if (lane == 0) put_lse(a, token, h, mm, ll);
      } else {
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) part[row * DP + lane + 32 * e] = acc[e];
        if (lane == 0) {
          part[kRows * DP + row] = mm;
          part[kRows * DP + kRows + row] = ll;
        }
      }
    }
    if (!w.opens && w.ends) join = Join{w.first_cta, w.sequence, head, w.tile};
    __syncthreads();  // the ring is free again
  }
  if (!a.whole && threadIdx.x == 0) a.joins[blockIdx.x] = join;
}

template <typename T, typename TO, int DP> void launch(const AttentionArgs &a, const Plan &p, cudaStream_t s) {
  constexpr size_t smem = smem_bytes<T, DP>();
  (void)cudaFuncSetAttribute(step_kernel<T, TO, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_pdl(step_kernel<T, TO, DP>, p.ctas, kThreads, smem, s, a);
  if (!p.whole) launch_pdl(join_kernel<TO, kRows, DP>, dim3(p.ctas, kRows), 128, 0, s, a);
}

}  // namespace

Plan step_plan(const AttentionArgs &a, uint32_t max_new) {
  const uint32_t keys = kWarps * (a.cache.type == TL_FLOAT32 ? step_keys<float>() : step_keys<__half>());
  const uint32_t dp = a.cache.D > 64 ? 128 : 64;
  Plan p{};
  // Jobs of few blocks are not cut, and nothing is joined.  64 sequences of up to 192 and
  // 511 keys: 24.6 and 28.7 us whole, 27.7 and 33.8 cut; one sequence of 192 keys 14.3 and
  // 17.4, of 1023 keys 30.7 and 19.5.
  p.whole = most_blocks(a, max_new, keys) <= 8;
  const uint64_t jobs = most_jobs(a, kRows);
  const uint64_t most = p.whole ? kNumSMs * 16 : kNumSMs * 2;
  p.ctas = static_cast<uint32_t>(p.whole && jobs < most ? jobs : most);
  p.part_floats = kRows * dp + 2 * kRows;
  return p;
}

void launch_step(const AttentionArgs &a, const Plan &p, bool wide, cudaStream_t s) {
  const bool narrow = a.cache.D <= 64;
#define L(T, TO) narrow ? launch<T, TO, 64>(a, p, s) : launch<T, TO, 128>(a, p, s)
  if (a.cache.type == TL_FLOAT32) L(float, float);
  else if (a.cache.type == TL_FLOAT16) { if (wide) L(__half, float); else L(__half, __half); }
  else if (wide) L(__nv_bfloat16, float);
  else L(__nv_bfloat16, __nv_bfloat16);
#undef L
}

}  // namespace paged
}  // namespace tl
