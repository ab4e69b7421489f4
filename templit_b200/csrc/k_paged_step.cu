// Attention over a paged cache for few query rows a key head (single tokens
// and short runs of them, any type; include/templit_cuda.h:
// tl_paged_attention).
//
// Bound by memory: every key and value is read once for up to 16 query rows
// (a token's heads that share a key head lie side by side), so the rows' own
// arithmetic is small and mma.sync is enough.  A warp works alone: it brings 16
// keys and values (8 of 32 bits) at a time into its own ring in shared memory
// by cp.async, several steps ahead, multiplies and keeps its rows' maxima,
// sums and outputs in registers; no barrier but the warp's own until its
// share of a job is done, when the CTA's warps join in shared memory.  Shares
// of the keys and their joining: paged_attention.cuh.
#include "paged_attention.cuh"

namespace tl {
namespace paged {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr uint32_t kRows = 16;

template <typename T> struct Step;
// 16-bit types: m16n8k16, 16 keys a step.  Numerators are at most 2^kShift, so
// that fp16's small ones keep their bits (normal down to 2^-28 of the largest).
template <> struct Step<__nv_bfloat16> {
  static constexpr uint32_t kKeys = 16;
  static constexpr float kShift = 0.0f;
};
template <> struct Step<__half> {
  static constexpr uint32_t kKeys = 16;
  static constexpr float kShift = 14.0f;
};
// fp32: m16n8k8 of operands split into two tf32 parts, 8 keys a step.
template <> struct Step<float> {
  static constexpr uint32_t kKeys = 8;
  static constexpr float kShift = 0.0f;
};

constexpr int kStages = 3;
template <typename T, int DP> constexpr uint32_t stage_bytes() { return 2 * Step<T>::kKeys * DP * sizeof(T); }
template <typename T, int DP> constexpr size_t smem_bytes() {
  return static_cast<size_t>(kWarps) * kStages * stage_bytes<T, DP>() + (sizeof(T) == 4 ? DP / 8 * 32 * 2 * sizeof(uint4) : 0);
}
// floats of a partial result: outputs, maxima, sums
template <int DP> constexpr uint32_t part_floats() { return kRows * DP + 2 * kRows; }

__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void await() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
__device__ __forceinline__ float load_word(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
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
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = big + small to 2^-22 of x, both of tf32's 11 bits (rounded to nearest)
__device__ __forceinline__ void split(float x, uint32_t &big, uint32_t &small) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(big) : "f"(x));
  const float rest = x - __uint_as_float(big);
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(small) : "f"(rest));
}

// Rows of a job that a lane holds (its two of 16): keys [from, to) of each.
struct Rows {
  uint32_t from[2], to[2];
};

template <typename T, typename TO, int DP>
__global__ void __launch_bounds__(kThreads, 2) step_kernel(const AttentionArgs a) {
  constexpr uint32_t N = Step<T>::kKeys;       // keys of a warp's step
  constexpr uint32_t KEYS = N * kWarps;        // of a block
  constexpr uint32_t E = 16 / sizeof(T);       // elements of a vector
  constexpr uint32_t CH = DP / E;              // vectors of a row
  constexpr int KS = DP / (sizeof(T) == 2 ? 16 : 8);  // steps of the first product
  constexpr uint32_t kHalf = N * DP * sizeof(T);
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows];
  pdl_enter();
  const tl_paged_cache &c = a.cache;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const Share share = share_of<kRows, KEYS, kThreads>(a, blockIdx.x, gridDim.x, a.whole ? 1 : 4);
  Join join{0xffffffffu, 0, 0, 0};
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * kStages * 2 * kHalf;
  const float scale = a.scale * kLog2e;

  uint32_t s = share.sequence;
  uint64_t offset = share.offset, left = share.any ? share.size : 0, at = share.begin;
  Work<kRows, KEYS> w;
  if (left) w.set(a, s);
  while (left) {
    const uint64_t line = w.cost(a);
    if (offset >= line) {  // the next sequence with any rows
      offset -= line;
      ++s;
      w.set(a, s);
      continue;
    }
    // this job, and the part of its blocks that is ours
    const uint32_t span = a.whole ? 1 : w.blocks;
    const uint32_t job = static_cast<uint32_t>(offset / span), block0 = static_cast<uint32_t>(offset % span);
    const uint32_t tile = job / c.heads, head = job % c.heads;
    const uint32_t take = static_cast<uint32_t>(min(left, static_cast<uint64_t>(span - block0)));
    const bool opens = block0 == 0, ends = block0 + take == span;
    const uint32_t b_lo = w.first + (a.whole ? 0 : block0), b_hi = w.first + (a.whole ? w.blocks : block0 + take);

    // rows
    const uint64_t row0 = static_cast<uint64_t>(tile) * kRows, rows = static_cast<uint64_t>(w.q.count) * a.group;
    const int64_t position0 = static_cast<int64_t>(w.q.length) - w.q.count;
    const uint32_t last = static_cast<uint32_t>(min(row0 + kRows, rows) - 1 - row0);
    uint32_t all_from, all_to, f, t;
    seen(a, w.q.length, position0 + static_cast<int64_t>(row0 / a.group), all_from, t);
    uint32_t least_to = t;
    seen(a, w.q.length, position0 + static_cast<int64_t>((row0 + last) / a.group), f, all_to);
    const uint32_t most_from = f;
    const bool uneven = all_from != most_from || all_to != least_to;
    Rows r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t row = lane / 4 + 8 * i;
      r.from[i] = r.to[i] = 0;
      if (row <= last) seen(a, w.q.length, position0 + static_cast<int64_t>((row0 + row) / a.group), r.from[i], r.to[i]);
    }
    const uint32_t key_lo = max(b_lo * KEYS, all_from / N * N);
    const uint32_t key_hi = static_cast<uint32_t>(min(static_cast<uint64_t>(b_hi) * KEYS, static_cast<uint64_t>(all_to)));
    // this warp's steps: keys first_key + i KEYS
    const uint32_t skip = key_lo > b_lo * KEYS ? (key_lo - b_lo * KEYS) / KEYS : 0;
    const uint32_t first_key = b_lo * KEYS + skip * KEYS + warp * N;
    const uint32_t steps = first_key < key_hi ? (key_hi - first_key + KEYS - 1) / KEYS : 0;

    // queries as the first product's left operand
    // (fp32: split, in shared memory, as 128 registers a lane would not be left)
    uint32_t qa[sizeof(T) == 2 ? KS : 1][4];
    uint4 *const halves = reinterpret_cast<uint4 *>(smem + kWarps * kStages * 2 * kHalf) + lane;
    if constexpr (sizeof(T) == 4) {
      for (uint32_t k = warp; k < KS; k += kWarps) {
        uint32_t big[4], small[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t row = lane / 4 + 8 * i;
          const uint64_t place = row0 + row;
          const T *p = static_cast<const T *>(a.q.p) + (w.q.start + place / a.group) * a.q.row_stride +
                       (head * a.group + place % a.group) * a.q.head_stride;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t d = k * 8 + j * 4 + (lane & 3);
            split(row <= last && d < c.D ? heads::element_of(p[d]) : 0.0f, big[i + 2 * j], small[i + 2 * j]);
          }
        }
        halves[k * 64] = make_uint4(big[0], big[1], big[2], big[3]);
        halves[k * 64 + 32] = make_uint4(small[0], small[1], small[2], small[3]);
      }
      __syncthreads();
    } else {
      const T *q = static_cast<const T *>(a.q.p);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t row = lane / 4 + 8 * i;
        const uint64_t place = row0 + row;
        const T *p = q + (w.q.start + place / a.group) * a.q.row_stride + (head * a.group + place % a.group) * a.q.head_stride;
        const bool there = row <= last;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t d = k * 16 + j * 8 + (lane & 3) * 2;
            qa[k][i + 2 * j] = there && d < c.D ? *reinterpret_cast<const uint32_t *>(p + d) : 0u;
          }
      }
    }

    const T *kp = static_cast<const T *>(c.k) + head * c.head_stride;
    const T *vp = static_cast<const T *>(c.v) + head * c.head_stride;
    // where lane i's key of a step lies, -1 where there is none
    const auto offset_of = [&](uint32_t step) -> int64_t {
      const uint32_t j = first_key + step * KEYS + lane;
      return step < steps && lane < N && j >= all_from && j < key_hi ? key_offset(a, s, j) : -1;
    };
    const auto bring = [&](uint32_t step, int64_t from) {
      const uint32_t to = ring + (step % kStages) * 2 * kHalf;
#pragma unroll
      for (uint32_t i = 0; i < N * CH / 32; ++i) {
        const uint32_t row = (lane + 32 * i) / CH, ch = (lane + 32 * i) % CH;
        const int64_t place = __shfl_sync(0xffffffffu, from, row);
        const bool there = place >= 0 && ch * E < c.D;
        const uint64_t e = there ? place + ch * E : 0;
        const uint32_t spot = to + row * (DP * sizeof(T)) + ((ch ^ (row & 7)) << 4);
        copy16(spot, kp + e, there);
        copy16(spot + kHalf, vp + e, there);
      }
    };
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
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
        float x[N / 8][4];
#pragma unroll
        for (uint32_t n = 0; n < N / 8; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
        if constexpr (sizeof(T) == 2) {
          const uint32_t row = (lane >> 4) * 8 + (lane & 7), ch = (lane >> 3) & 1;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t b[4];
            load_matrices(from + row * (DP * 2) + (((k * 2 + ch) ^ (row & 7)) << 4), b);
            mma16<T>(x[0], qa[k], b[0], b[1]);
            mma16<T>(x[1], qa[k], b[2], b[3]);
          }
        } else {
          const uint32_t row = lane >> 2;
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t b0, b1, s0, s1;
            split(load_word(from + row * (DP * 4) + (((k * 2) ^ row) << 4) + (lane & 3) * 4), b0, s0);
            split(load_word(from + row * (DP * 4) + (((k * 2 + 1) ^ row) << 4) + (lane & 3) * 4), b1, s1);
            const uint4 qb = halves[k * 64], qs = halves[k * 64 + 32];
            const uint32_t big[4] = {qb.x, qb.y, qb.z, qb.w}, small[4] = {qs.x, qs.y, qs.z, qs.w};
            mma8(x[0], small, b0, b1);
            mma8(x[0], big, s0, s1);
            mma8(x[0], big, b0, b1);
          }
        }
        // element e of x[n]: row lane / 4 + 8 (e / 2), key 8 n + 2 (lane & 3) + (e & 1)
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (uint32_t n = 0; n < N / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[n][e] *= scale;
            if (!full) {
              const uint32_t i = n * 8 + (lane & 3) * 2 + (e & 1), j = key + i;
              if (!(good[u] >> i & 1) || j < r.from[e >> 1] || j >= r.to[e >> 1]) x[n][e] = -INFINITY;
            }
            top[e >> 1] = fmaxf(top[e >> 1], x[n][e]);
          }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2)) - Step<T>::kShift;
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
        for (uint32_t n = 0; n < N / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[n][e] = ex2_approx(x[n][e] - base[e >> 1]);
            l[e >> 1] += x[n][e];
          }
        const uint32_t values = from + kHalf;
        if constexpr (sizeof(T) == 2) {
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
            load_transposed(values + row * (DP * 2) + (((d * 2 + ch) ^ (row & 7)) << 4), b);
            mma16<T>(o[2 * d], p, b[0], b[1]);
            mma16<T>(o[2 * d + 1], p, b[2], b[3]);
          }
        } else {
          // The left operand's column j (and j + 4) of a lane is key 2 j (2 j + 1), as the
          // scores lie, so the values' rows are taken in the same order.
          uint32_t p[4], ps[4];
          split(x[0][0], p[0], ps[0]);
          split(x[0][2], p[1], ps[1]);
          split(x[0][1], p[2], ps[2]);
          split(x[0][3], p[3], ps[3]);
          const uint32_t k0 = (lane & 3) * 2, n = lane >> 2;
#pragma unroll
          for (int d = 0; d < DP / 8; ++d) {
            uint32_t b0, b1, s0, s1;
            const uint32_t ch = d * 2 + (n >> 2);
            split(load_word(values + k0 * (DP * 4) + ((ch ^ k0) << 4) + (n & 3) * 4), b0, s0);
            split(load_word(values + (k0 + 1) * (DP * 4) + ((ch ^ (k0 + 1)) << 4) + (n & 3) * 4), b1, s1);
            mma8(o[d], ps, b0, b1);
            mma8(o[d], p, s0, s1);
            mma8(o[d], p, b0, b1);
          }
        }
        __syncwarp();
      }
    }
    await<0>();
    // the CTA's warps into one: outputs through the ring, a row's four warps by one warp
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    __syncthreads();
    float *const outs = reinterpret_cast<float *>(smem);  // [warp][row][DP]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t row = lane / 4 + 8 * i;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d)
        *reinterpret_cast<float2 *>(outs + (warp * kRows + row) * DP + d * 8 + (lane & 3) * 2) =
            make_float2(o[d][2 * i], o[d][2 * i + 1]);
      if ((lane & 3) == 0) {
        sm_m[warp][row] = m[i];
        sm_l[warp][row] = l[i];
      }
    }
    __syncthreads();
    float *const part = a.parts + (static_cast<size_t>(blockIdx.x) * 2 + (opens ? 1 : 0)) * part_floats<DP>();
    for (uint32_t row = warp; row <= last; row += kWarps) {
      float mm = sm_m[0][row], ll = 0.0f, acc[DP / 32];
#pragma unroll
      for (int i = 1; i < kWarps; ++i) mm = fmaxf(mm, sm_m[i][row]);
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) acc[e] = 0.0f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const float wm = sm_m[i][row];
        if (wm == -INFINITY) continue;
        const float f = ex2_approx(wm - mm);
        ll = fmaf(f, sm_l[i][row], ll);
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) acc[e] = fmaf(f, outs[(i * kRows + row) * DP + lane + 32 * e], acc[e]);
      }
      const uint64_t place = row0 + row;
      const uint64_t token = w.q.start + place / a.group;
      const uint32_t h = head * a.group + static_cast<uint32_t>(place % a.group);
      bool nan = false;
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) nan = nan || (lane + 32 * e < c.D && acc[e] != acc[e]);
      if (uneven && ll == ll && __any_sync(0xffffffffu, nan)) {
        // A value that other rows of the tile see, and this one does not, is not
        // finite (0 times it is NaN): the row's own keys one by one.
        float again[kMaxHead / 32];
        seen(a, w.q.length, position0 + static_cast<int64_t>(place / a.group), f, t);
        const T *q = static_cast<const T *>(a.q.p) + token * a.q.row_stride + h * a.q.head_stride;
        row_over_keys<T>(a, s, head, q, max(f, b_lo * KEYS), min(t, key_hi), lane, mm, ll, again);
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) acc[e] = again[e];
      }
      if (opens && ends) {
        TO *out = static_cast<TO *>(const_cast<void *>(a.out.p)) + token * a.out.row_stride + h * a.out.head_stride;
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
          if (lane + 32 * e < c.D) heads::set_element(out[lane + 32 * e], ll == 0.0f ? 0.0f : acc[e] / ll);
        if (lane == 0 && a.lse) a.lse[token * a.q_heads + h] = ll == 0.0f ? -INFINITY : mm * kLn2 + logf(ll);
      } else {
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) part[row * DP + lane + 32 * e] = acc[e];
        if (lane == 0) {
          part[kRows * DP + row] = mm;
          part[kRows * DP + kRows + row] = ll;
        }
      }
    }
    if (!opens && ends) join = Join{static_cast<uint32_t>((at - block0) / share.full), s, head, tile};
    __syncthreads();  // the ring is free again
    offset += take;
    at += take;
    left -= take;
  }
  if (!a.whole && threadIdx.x == 0) a.joins[blockIdx.x] = join;
}

// The jobs that were cut: a warp per row adds the partial results up in the
// order of the keys.
template <typename TO, int DP>
__global__ void __launch_bounds__(kThreads) join_kernel(const AttentionArgs a) {
  pdl_enter();
  const Join j = a.joins[blockIdx.x];
  if (j.first == 0xffffffffu) return;
  const uint32_t lane = threadIdx.x & 31, row = blockIdx.y * kWarps + threadIdx.x / 32, end = blockIdx.x;
  const Sequence q = sequence_of(a.cache, j.sequence, a.most);
  const uint64_t place = static_cast<uint64_t>(j.tile) * kRows + row;
  if (place >= static_cast<uint64_t>(q.count) * a.group) return;
  const auto part = [&](uint32_t cta) { return a.parts + (static_cast<size_t>(cta) * 2 + (cta == j.first ? 1 : 0)) * part_floats<DP>(); };
  float mm = -INFINITY;
  for (uint32_t i = j.first + lane; i <= end; i += 32) mm = fmaxf(mm, part(i)[kRows * DP + row]);
  mm = warp_max(mm);
  float ll = 0.0f, acc[DP / 32];
#pragma unroll
  for (int e = 0; e < DP / 32; ++e) acc[e] = 0.0f;
#pragma unroll 4
  for (uint32_t i = j.first; i <= end; ++i) {
    const float *p = part(i);
    const float wm = p[kRows * DP + row], f = wm == -INFINITY ? 0.0f : ex2_approx(wm - mm);
    ll = fmaf(f, p[kRows * DP + kRows + row], ll);
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) {
      const float x = p[row * DP + lane + 32 * e];
      if (f != 0.0f) acc[e] = fmaf(f, x, acc[e]);
    }
  }
  const uint64_t token = q.start + place / a.group;
  const uint32_t h = j.head * a.group + static_cast<uint32_t>(place % a.group);
  TO *out = static_cast<TO *>(const_cast<void *>(a.out.p)) + token * a.out.row_stride + h * a.out.head_stride;
#pragma unroll
  for (int e = 0; e < DP / 32; ++e)
    if (lane + 32 * e < a.cache.D) heads::set_element(out[lane + 32 * e], ll == 0.0f ? 0.0f : acc[e] / ll);
  if (lane == 0 && a.lse) a.lse[token * a.q_heads + h] = ll == 0.0f ? -INFINITY : mm * kLn2 + logf(ll);
}

template <typename T, typename TO, int DP> void launch(const AttentionArgs &a, const Plan &p, cudaStream_t s) {
  constexpr size_t smem = smem_bytes<T, DP>();
  (void)cudaFuncSetAttribute(step_kernel<T, TO, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_pdl(step_kernel<T, TO, DP>, p.ctas, kThreads, smem, s, a);
  if (!p.whole) launch_pdl(join_kernel<TO, DP>, dim3(p.ctas, kRows / kWarps), kThreads, 0, s, a);
}

}  // namespace

Plan step_plan(const AttentionArgs &a, uint32_t max_new) {
  const uint32_t keys = kWarps * (a.cache.type == TL_FLOAT32 ? Step<float>::kKeys : Step<__half>::kKeys);
  const uint32_t dp = a.cache.D > 64 ? 128 : 64;
  Plan p{};
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
