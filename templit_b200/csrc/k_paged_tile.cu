// Attention over a paged cache for many query rows a key head (chunks of a
// prompt) in 16-bit types (include/templit_cuda.h: tl_paged_attention).
//
// Bound by the softmax's exponentials and the tensor cores: 128 x 128 scores of
// 128 elements are 1024 cycles of the 16 exponentials a cycle of an SM and 512 of
// each product.  So a CTA, one an SM, holds two tiles of 128
// query rows (tokens, a token's heads of one key head side by side), and
// while one is in the softmax the other is multiplied:
//   warps 0-3, 4-7  softmax of tile 0 and 1, a row a thread, 64 keys at a time: scores
//                   out of TMEM, numerators rounded to the type back over them,
//                   where the second product takes them from;
//                   running maximum and sum in registers.  The output stays
//                   in TMEM and is rescaled only when a row's maximum grew
//                   by more than 2^8 (numerators then are at most 2^8, which
//                   fp32 sums and 16-bit types hold)
//   warps 8-11      keys and values, 128 at a time (32 a warp), into a ring, and
//                   the queries.  By TMA where a page holds whole runs of 8, 16 or
//                   32 keys and all 32 are there; else row by row with cp.async,
//                   16 bytes a lane, which writes zeros for the keys that are
//                   not there (3600 cycles of a warp for a block, more than its
//                   products take; TMA's boxes are a few instructions)
//   warp 12         one thread issues S = Q K^T and O += P V (tcgen05.mma
//                   kind::f16, fp32 in TMEM)
//   warp 13         one thread works out the CTA's pieces of jobs, ahead of the others
//   warps 14, 15    nothing (without them the compiler gives a thread 144 registers in
//                   place of 128, and the prompt below took 556 us in place of 546, both in the first calls)
// TMEM: 2 x 2 buffers of 64 columns of scores, 2 x 128 of outputs.  With two buffers a
// tile, the next scores are multiplied while the last ones are in the softmax; one of 128
// leaves each waiting for the other (710 us where this took 580), although scores of 64
// keys take 48 cycles of a product of 32 (of 128 keys 64).  Every wait is bounded
// (2 s); where one gives up, the CTA raises TL_FLAG_TIMEOUT, waits for what it issued
// and returns.  Shares of the keys and their joining: paged_attention.cuh.
//
// 8192 tokens of one prompt, 8 key heads of 128 bf16, 4 query heads each, causal: 538 us in
// the first calls, at 1965 MHz; 604 to 620 (897 to 920 TFLOP/s of the 1372 of a large library
// product that is as long under way) repeated, where the power limit leaves 1710 MHz.  980000
// cycles of the tile kernel are 225 blocks of 2 x 128 x 128 scores an SM and 7 jobs' ends
// of 8500 (256 rows out of TMEM): 4100 cycles a block, of which the exponentials take the
// unit for 2^x 2048 and the products the tensor cores 2200, half each.  Both tiles' softmax
// warps share the schedulers, two a scheduler, and hand-overs come between.  A polynomial
// for some of the exponentials gained nothing: the instructions that are issued then
// bound it.  24 chunks of up to 509 tokens, 3 query heads of 64 a key head, behind up to
// 4093 keys: 80 us; jobs are short there, their ends and ragged first and last tiles are
// half of it.
#include "paged_attention.cuh"
#include "tc_ptx.cuh"

namespace tl {
namespace paged {
namespace {

constexpr uint32_t kTile = 128, kRows = 2 * kTile, kKeys = 128;
constexpr int kThreads = 16 * 32, kLoaders = 128;
constexpr uint64_t kWaitLimitNs = 2000000000ull;
constexpr float kSlack = 8.0f;  // log2 of how far numerators may pass 1
constexpr int kLag = 2;         // ring places between a copy's issue and its hand-over
// Values of block j and keys of block j + 1 (places 2 j + 1 and 2 j + 2 of the ring's
// sequence) are given back together: one arrival in place of two, 200 cycles each.
constexpr int kPairs = 8;
constexpr int kJobs = 4;        // pieces worked out ahead
constexpr int kMasks = 8;       // blocks whose missing keys are remembered: more than the ring is ahead

template <int DP> constexpr uint32_t tile_bytes() { return kTile * DP * 2; }
template <int DP> constexpr int stages() { return DP == 128 ? 4 : 8; }
constexpr uint32_t kStaging = 8 * 4096;  // 32 rows of 128 bytes for each softmax warp

struct Barriers {
  uint64_t full[8], empty[kPairs];
  uint64_t job_full[kJobs], job_free[kJobs];
  uint64_t q_full, q_empty, s_full[2][2], p_full[2][2], o_tail[2], o_full[2], o_free[2], drained;
};
// A piece and the blocks that its two tiles take, from the piece's first on;
// more == false: there are no more.
struct Job {
  Piece p;
  uint32_t n[2], most;
  bool more;
};
struct Shared {
  Barriers b;
  Job jobs[kJobs];
  uint32_t tmem, gave_up;
  uint32_t not_finite;  // rows may ask for mend_rows()
  Share share;
  uint32_t mask[kMasks][4];  // a bit for every key of a block that is there
};
template <int DP> constexpr size_t smem_bytes() {
  return 1024 + 2 * tile_bytes<DP>() + stages<DP>() * static_cast<size_t>(tile_bytes<DP>()) + kStaging + sizeof(Shared);
}

// Waits for a phase; false where it gave up, here or elsewhere in the CTA.  The
// first look is inline, a few instructions; the rest is not.
__device__ __noinline__ bool wait_longer(Shared &sh, uint64_t *bar, uint32_t parity, uint32_t *status) {
  const uint64_t t0 = ptx::global_timer_ns();
  for (uint32_t i = 1;; ++i) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0) {
      if (*reinterpret_cast<volatile uint32_t *>(&sh.gave_up)) return false;
      if (ptx::global_timer_ns() - t0 > kWaitLimitNs) {
        *reinterpret_cast<volatile uint32_t *>(&sh.gave_up) = 1;
        raise_flag(status, TL_FLAG_TIMEOUT);
        return false;
      }
    }
  }
}
__device__ __forceinline__ bool wait(Shared &sh, uint64_t *bar, uint32_t parity, uint32_t *status) {
  return ptx::mbar_try_wait(bar, parity) || wait_longer(sh, bar, parity, status);
}

// The same for a whole warp, with one answer.
__device__ __forceinline__ bool wait_warp(Shared &sh, uint64_t *bar, uint32_t parity, uint32_t *status) {
  return __all_sync(0xffffffffu, wait(sh, bar, parity, status));
}

// How keys, values and queries lie, for TMA: boxes of `rows` keys (0: none), of
// a tile's queries where `queries` (a power of two of query heads a key head).
struct Maps {
  CUtensorMap k, v, q;  // (D, slot, head, page); (D, head, token)
  uint32_t rows, queries;
};
__device__ __forceinline__ void tma_box4(uint32_t to, const CUtensorMap *map, uint64_t *bar, uint32_t x, uint32_t slot,
                                         uint32_t head, uint32_t page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(ptx::smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tma_box3(uint32_t to, const CUtensorMap *map, uint64_t *bar, uint32_t x, uint32_t head,
                                         uint32_t token) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(token), "r"(ptx::smem_addr(bar))
      : "memory");
}

// Vector `ch` (16 bytes) of row `r` of a tile: 128-byte rows of 64 elements
// with the 128-byte swizzle, one block of 128 rows after another.
__device__ __forceinline__ uint32_t spot(uint32_t r, uint32_t ch) {
  return (ch >> 3) * (kTile * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
}
// Queries and keys, K-major, from element 0 on; 16 elements further are 2, 64
// are a block of 128 rows more.
__device__ __forceinline__ uint64_t row_desc(uint32_t base) { return ptx::smem_desc(base, 16, 1024, ptx::kSwizzle128B); }
__host__ __device__ constexpr uint32_t row_step(uint32_t k) { return (k >> 2) * (kTile * 128 / 16) + (k & 3) * 2; }
// Values, MN-major (a row is a key), 64 elements a block; 16 keys further are 128 more.
__device__ __forceinline__ uint64_t value_desc(uint32_t base) {
  return ptx::smem_desc(base, kTile * 128, 1024, ptx::kSwizzle128B);
}
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// kind::f16 with fp32 sums: type 0 = fp16, 1 = bf16.
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t type, uint32_t M, uint32_t N, bool b_mn) {
  return (1u << 4) | (type << 7) | (type << 10) | ((b_mn ? 1u : 0u) << 16) | ((N >> 3) << 17) | ((M >> 4) << 24);
}
__device__ __forceinline__ void mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
using heads::fma2;
using heads::halves;
using heads::Pair;
__device__ __forceinline__ Pair pair(uint32_t lo, uint32_t hi) { return heads::pair(__uint_as_float(lo), __uint_as_float(hi)); }
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// The larger of three; NaN where one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 16 and 32 columns of this warp's 32 lanes into TMEM
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T> __device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2 &>(r) = __floats2half2_rn(lo, hi);
  else reinterpret_cast<__nv_bfloat162 &>(r) = __floats2bfloat162_rn(lo, hi);
  return r;
}
// log2 of what the largest numerator is at least: with kSlack, fp16's stay
// below 2^15 and keep their bits down to 2^-21 of the largest
template <typename T> constexpr float shift() { return std::is_same<T, __half>::value ? 7.0f : 0.0f; }

// Blocks of a piece that tile t takes, from the piece's first on; both tiles
// start there.
__device__ __forceinline__ uint32_t tile_blocks(const AttentionArgs &a, const Piece &p, uint32_t t) {
  if (t * kTile > p.last) return 0;
  uint32_t from, to;
  seen(a, p.length, p.position(a, min((t + 1) * kTile - 1, p.last)), from, to);
  const uint32_t end = min(to / kKeys + (to % kKeys != 0), p.block_hi);
  return end > p.block_lo ? end - p.block_lo : 0;
}

// The next piece, when it has been worked out; its readers are done with it
// after release_job().
__device__ __forceinline__ const Job *next_job(Shared &sh, uint32_t i, uint32_t *status, bool *ok) {
  *ok = wait(sh, &sh.b.job_full[i % kJobs], (i / kJobs) & 1, status);
  return &sh.jobs[i % kJobs];
}
__device__ __forceinline__ void release_job(Shared &sh, uint32_t i) { ptx::mbar_arrive(&sh.b.job_free[i % kJobs]); }

__device__ __forceinline__ void plan_jobs(const AttentionArgs &a, const Share &share, Shared &sh) {
  Walk<kRows, kKeys> walk;
  Piece p;
  walk.start(a, share);
  bool more = true;
  for (uint32_t i = 0; more; ++i) {
    more = walk.next(a, share, p);
    if (!wait(sh, &sh.b.job_free[i % kJobs], ((i / kJobs) & 1) ^ 1, a.status)) return;
    Job &job = sh.jobs[i % kJobs];
    job.more = more;
    if (more) {
      job.p = p;
      job.n[0] = tile_blocks(a, p, 0);
      job.n[1] = tile_blocks(a, p, 1);
      job.most = max(job.n[0], job.n[1]);
      if (!p.opens && p.ends) a.joins[blockIdx.x] = Join{p.first_cta, p.sequence, p.head, p.tile};
    }
    ptx::mbar_arrive(&sh.b.job_full[i % kJobs]);
  }
}

template <typename T, int DP>
__device__ __forceinline__ void load(const AttentionArgs &a, const Maps &maps, Shared &sh, uint32_t queries, uint32_t ring) {
  constexpr int S = stages<DP>();
  constexpr uint32_t CH = DP / 8, kBytes = tile_bytes<DP>(), kBlocks = DP / 64;
  const uint32_t lane = threadIdx.x & 31, warp = (threadIdx.x - 256) / 32;
  const tl_paged_cache &c = a.cache;
  uint32_t item = 0, handed = 0, by_rows = 0, block_count = 0, q_phase = 0;
  // cp.async's copies up to `upto` (a bit of by_rows each) have arrived and are
  // the tensor cores' to read
  const auto hand_over = [&](uint32_t upto) {
    if (by_rows) {
      ptx::fence_proxy_async_smem();
      __syncwarp();
    }
    for (; handed < upto; ++handed) {
      const uint32_t bit = 1u << (handed & 31);
      if (by_rows & bit && lane == 0) ptx::mbar_arrive(&sh.b.full[handed % S]);
      by_rows &= ~bit;
    }
  };
  for (uint32_t i_job = 0;; ++i_job) {
    bool ok;
    const Job *const job = next_job(sh, i_job, a.status, &ok);
    if (!__all_sync(0xffffffffu, ok)) return;
    if (!job->more) break;
    const Piece &p = job->p;
    const uint32_t n = job->most, head = p.head;
    // this lane's key of a block: its page (no page: UINT32_MAX) and slot
    const uint32_t *const table = c.table + static_cast<uint64_t>(p.sequence) * c.table_stride;
    const auto look_up = [&](uint32_t block, uint32_t &page, uint32_t &slot) {
      const uint32_t j = (p.block_lo + block) * kKeys + warp * 32 + lane, i = j / c.page_size;
      slot = j - i * c.page_size;
      page = block < n && j >= p.from && j < p.to ? table[i] : 0xffffffffu;
    };
    uint32_t page, slot, next_page, next_slot;
    look_up(0, page, slot);
    for (uint32_t j = 0; j < n; ++j) {
      look_up(j + 1, next_page, next_slot);
      const uint32_t key = (p.block_lo + j) * kKeys + warp * 32 + lane;
      const bool there = page < c.pages;
      if (!there && key >= p.from && key < p.to) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
      const uint32_t good = __ballot_sync(0xffffffffu, there);
      const bool boxes = maps.rows && good == 0xffffffffu;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // a slot is free again when what was multiplied from it is done
        if (item >= static_cast<uint32_t>(S)) {
          const uint32_t pair = (item - S + 1) / 2;
          if (!wait_warp(sh, &sh.b.empty[pair % kPairs], (pair / kPairs) & 1, a.status)) return;
        }
        if (half == 0 && lane == 0) sh.mask[block_count % kMasks][warp] = good;
        const uint32_t to = ring + (item % S) * kBytes + warp * 32 * 128;
        uint64_t *const full = &sh.b.full[item % S];
        if (boxes) {
          const uint32_t from = lane * maps.rows & 31;
          const uint32_t b_page = __shfl_sync(0xffffffffu, page, from), b_slot = __shfl_sync(0xffffffffu, slot, from);
          if (lane == 0) ptx::mbar_arrive_expect_tx(full, 32 * 128 * kBlocks);
          __syncwarp();
          if (lane * maps.rows < 32)
#pragma unroll
            for (uint32_t b = 0; b < kBlocks; ++b)
              tma_box4(to + b * (kTile * 128) + from * 128, half ? &maps.v : &maps.k, full, b * 64, b_slot, head, b_page);
        } else {
          const T *base = static_cast<const T *>(half ? c.v : c.k) + head * c.head_stride;
          const int64_t at = there ? static_cast<int64_t>(page * c.page_stride + slot * c.slot_stride) : -1;
#pragma unroll 4
          for (uint32_t i = 0; i < CH; ++i) {
            const uint32_t row = (lane + 32 * i) / CH, ch = (lane + 32 * i) % CH;
            const int64_t from = __shfl_sync(0xffffffffu, at, row);
            const bool put = from >= 0 && ch * 8 < c.D;
            copy16(to + spot(row, ch), put ? base + from + ch * 8 : static_cast<const T *>(a.q.p), put);
          }
          by_rows |= 1u << (item & 31);
        }
        commit();
        ++item;
        if (j == 0 && half == 0) {
          // the queries: the rows of this warp, 32 of each tile
          await<0>();
          hand_over(item);
          if (!wait_warp(sh, &sh.b.q_empty, (q_phase & 1) ^ 1, a.status)) return;
          ++q_phase;
          if (maps.queries) {
            if (warp == 0 && lane == 0) {
              const bool both = p.last >= kTile;
              ptx::mbar_arrive_expect_tx(&sh.b.q_full, (both ? 2 : 1) * kBytes);
              const uint32_t token = p.start + p.row0 / a.group;
              for (uint32_t t = 0; t < (both ? 2u : 1u); ++t)
                for (uint32_t b = 0; b < kBlocks; ++b)
                  tma_box3(queries + t * kBytes + b * (kTile * 128), &maps.q, &sh.b.q_full, b * 64, head * a.group,
                           token + t * (kTile / a.group));
            } else if (lane == 0) {
              ptx::mbar_arrive(&sh.b.q_full);
            }
          } else {
            for (uint32_t t = 0; t < 2; ++t) {
              const uint32_t mine = t * kTile + warp * 32 + lane;
              const uint32_t place = p.row0 + mine;
              int64_t at = -1;
              if (mine <= p.last)
                at = static_cast<int64_t>((p.start + static_cast<uint64_t>(place / a.group)) * a.q.row_stride +
                                          (head * a.group + place % a.group) * a.q.head_stride);
#pragma unroll 4
              for (uint32_t i = 0; i < CH; ++i) {
                const uint32_t row = (lane + 32 * i) / CH, ch = (lane + 32 * i) % CH;
                const int64_t from = __shfl_sync(0xffffffffu, at, row);
                const bool put = from >= 0 && ch * 8 < c.D;
                copy16(queries + t * kBytes + warp * 32 * 128 + spot(row, ch), static_cast<const T *>(a.q.p) + (put ? from + ch * 8 : 0), put);
              }
            }
            commit();
            await<0>();
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&sh.b.q_full);
          }
        } else {
          await<kLag>();
          if (item > kLag) hand_over(max(handed, item - kLag));
        }
      }
      ++block_count;
      page = next_page;
      slot = next_slot;
    }
    if (n == 0) {
      // A piece without keys: the last copies before it go on here, as they do with a
      // piece's first keys.  Kept back over several such pieces, they would hold up the
      // piece that waits for them, and with it the next one's place in the jobs' ring.
      await<0>();
      hand_over(item);
    }
    __syncwarp();
    if (lane == 0) release_job(sh, i_job);
  }
  await<0>();
  hand_over(item);
  // the last reads of the ring are over
  if (item && !wait_warp(sh, &sh.b.empty[item / 2 % kPairs], (item / 2 / kPairs) & 1, a.status)) return;
}

// By one thread.  A product's instructions are unrolled with descriptors that
// differ by constants (worked out one by one they took 100 cycles each, as long
// as the product itself), the four steps of a block are one copy of the code,
// and a wait that is over costs a few instructions: what this thread does
// between products the tensor cores wait for.
template <typename T, int DP>
__device__ __forceinline__ void multiply(const AttentionArgs &a, Shared &sh, uint32_t queries, uint32_t ring) {
  constexpr uint32_t S = stages<DP>();
  constexpr uint32_t kBytes = tile_bytes<DP>();
  constexpr uint32_t type = std::is_same<T, __half>::value ? 0 : 1;
  const uint32_t ksteps = (a.cache.D + 15) / 16;
  const uint32_t score = idesc_f16(type, kTile, kKeys / 2, false), output = idesc_f16(type, kTile, ksteps * 16, true);
  const uint32_t tmem = sh.tmem;
  const uint64_t q_desc = row_desc(queries), k_desc = row_desc(ring), v_desc = value_desc(ring);
  uint32_t item = 0, piece = 0, p_phase = 0, o_phase = 3;  // a bit for each tile
  // scores of the 64 keys of half h
  const auto scores = [&](uint32_t t, uint32_t slot, uint32_t h) {
    const uint64_t q = q_desc + t * (kBytes / 16), k = k_desc + slot * (kBytes / 16) + h * (64 * 128 / 16);
#pragma unroll
    for (uint32_t i = 0; i < DP / 16; ++i)
      if (i < ksteps) mma_smem(tmem + t * 128 + h * 64, q + row_step(i), k + row_step(i), score, i > 0);
    ptx::mma_commit(&sh.b.s_full[t][h]);
  };
  for (uint32_t i_job = 0;; ++i_job) {
    bool ok;
    const Job *const job = next_job(sh, i_job, a.status, &ok);
    if (!ok) return;
    if (!job->more) break;
    const uint32_t n0 = job->n[0], n1 = job->n[1], most = job->most;
    release_job(sh, i_job);
    if (!most) continue;
    if (!wait(sh, &sh.b.q_full, piece & 1, a.status)) return;
    ++piece;
    const uint32_t first = item;  // block j: keys in place first + 2 j, values behind them
    if (!wait(sh, &sh.b.full[first % S], (first / S) & 1, a.status)) return;
    ptx::tc_fence_after();
#pragma unroll 1
    for (uint32_t e = 0; e < 4; ++e)
      if (e & 1 ? n1 : n0) scores(e & 1, first % S, e >> 1);
    ptx::mma_commit(&sh.b.empty[first / 2 % kPairs]);
#pragma unroll 1
    for (uint32_t j = 0; j < most; ++j) {
      const uint32_t v = first + 2 * j + 1, k = v + 1;
      if (!wait(sh, &sh.b.full[v % S], (v / S) & 1, a.status)) return;
      if (j + 1 < most && !wait(sh, &sh.b.full[k % S], (k / S) & 1, a.status)) return;
      const uint64_t values = v_desc + v % S * (kBytes / 16);
#pragma unroll 1
      for (uint32_t e = 0; e < 4; ++e) {
        const uint32_t t = e & 1, h = e >> 1, n = t ? n1 : n0;
        if (j >= n) continue;
        if (j + h == 0) {  // the tile's last output has been read
          if (!wait(sh, &sh.b.o_free[t], o_phase >> t & 1, a.status)) return;
          o_phase ^= 1u << t;
        }
        if (!wait(sh, &sh.b.p_full[t][h], p_phase >> t & 1, a.status)) return;
        p_phase ^= h << t;
        ptx::tc_fence_after();
        const uint32_t o_at = tmem + 256 + t * 128, p_at = tmem + t * 128 + h * 64;
        const uint64_t rows = values + h * 512;
#pragma unroll
        for (uint32_t i = 0; i < kKeys / 32; ++i) mma_tmem(o_at, p_at + i * 8, rows + i * 128, output, (j | h | i) > 0);
        if (j + 1 == n) ptx::mma_commit(h ? &sh.b.o_full[t] : &sh.b.o_tail[t]);
        // the buffer is free again behind that product: the tensor cores keep the order
        else scores(t, k % S, h);
      }
      // the last block's values go back with the next piece's first keys
      if (j + 1 < most) ptx::mma_commit(&sh.b.empty[k / 2 % kPairs]);
    }
    ptx::mma_commit(&sh.b.q_empty);
    item += 2 * most;
  }
  if (item) ptx::mma_commit(&sh.b.empty[item / 2 % kPairs]);
}

// A warp's 32 rows of the output, 128 bytes of each at a time through its 4 KB
// of shared memory: stored row by row, a lane 16 bytes of its own, each
// instruction touched 32 lines and a piece took 9000 cycles to end.  `row` is where the
// lane's row begins, null where it goes nowhere.
template <typename U>
__device__ __forceinline__ bool put_rows(uint32_t o_at, bool any, uint32_t D, float factor, U *row, uint4 *staging) {
  constexpr uint32_t E = 128 / sizeof(U);  // elements of a row at a time
  const uint32_t lane = threadIdx.x & 31;
  bool nan = false;
#pragma unroll 1
  for (uint32_t d0 = 0; d0 < D; d0 += E) {
#pragma unroll
    for (uint32_t b = 0; b < E / 32; ++b) {
      uint32_t x[32];
      if (any) ptx::tmem_load_32x32b_x32(o_at + d0 + 32 * b, x);
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (!any) x[i] = 0;
        const float y = __uint_as_float(x[i]);
        nan = nan || (y != y && d0 + 32 * b + i < D);
        x[i] = __float_as_uint(y * factor);
      }
#pragma unroll
      for (uint32_t v = 0; v < 32 * sizeof(U) / 16; ++v) {
        constexpr int N = 16 / sizeof(U);
        float y[N];
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = __uint_as_float(x[v * N + i]);
        heads::Raw<U, N> raw;
        raw.set(y);
        const uint32_t ch = b * (32 * sizeof(U) / 16) + v;
        staging[lane * 8 + (ch ^ (lane & 7))] = raw.r[0];
      }
    }
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t r = i * 4 + lane / 8, ch = lane & 7, d = d0 + ch * (16 / sizeof(U));
      U *const to = reinterpret_cast<U *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(row), r));
      if (to && d < D) *reinterpret_cast<uint4 *>(to + d) = staging[r * 8 + (ch ^ (r & 7))];
    }
    __syncwarp();
  }
  return nan;
}

template <typename T, typename TO, int DP>
__device__ __forceinline__ void soften(const AttentionArgs &a, Shared &sh, uint8_t *all_staging) {
  const uint32_t lane = threadIdx.x & 31, t = threadIdx.x / 128, row = threadIdx.x & 127;
  const uint32_t lanes = (threadIdx.x / 32 & 3) << 21;  // this warp's 32 lanes of TMEM
  const uint32_t s_at = sh.tmem + t * 128 + lanes, o_at = sh.tmem + 256 + t * 128 + lanes;
  uint4 *const staging = reinterpret_cast<uint4 *>(all_staging + threadIdx.x / 32 * 4096);
  const float c = a.scale * kLog2e;
  const Pair c2 = pair(__float_as_uint(c), __float_as_uint(c));
  const tl_paged_cache &cache = a.cache;
  uint32_t done = 0, outputs = 0, block_count = 0;  // of this tile: blocks whose scores were taken, pieces; all blocks
  for (uint32_t i_job = 0;; ++i_job) {
    bool ok;
    const Job *const job = next_job(sh, i_job, a.status, &ok);
    if (!__all_sync(0xffffffffu, ok) || !job->more) return;
    const Piece &p = job->p;
    const uint32_t n = job->n[t];
    const uint32_t in_job = t * kTile + row;
    const bool there = in_job <= p.last;
    // rows behind the last one see everything: their scores go nowhere
    uint32_t from = 0, to = 0xffffffffu;
    if (there) seen(a, p.length, p.position(a, in_job), from, to);
    // A warp without rows only passes its tile's turns on (what TMEM holds goes through
    // the products to outputs that nobody reads).
    const bool idle = t * kTile + (row & ~31u) > p.last;
    float m = -INFINITY, l = 0.0f;
    for (uint32_t j = 0; j < n; ++j) {
      // By halves of 64 keys, each with its scores' buffer; one copy of the code, which
      // the warps' instruction caches hold.
#pragma unroll 1
      for (uint32_t h = 0; h < 2; ++h) {
        if (!wait_warp(sh, &sh.b.s_full[t][h], done & 1, a.status)) return;
        if (idle) {
          if (lane == 0) ptx::mbar_arrive(&sh.b.p_full[t][h]);
          continue;
        }
        ptx::tc_fence_after();
        const uint32_t key = (p.block_lo + j) * kKeys + h * 64, at = s_at + h * 64;
        const uint32_t *good = &sh.mask[(block_count + j) % kMasks][2 * h];
        const bool whole = key >= from && to >= 64 && key <= to - 64 && (good[0] & good[1]) == 0xffffffffu;
        // Numerators by the maximum of the keys before, in one pass: the scores' own
        // maximum is looked at behind it, and seldom passes that one by 2^8.
        bool settled = __all_sync(0xffffffffu, whole && m != -INFINITY);
        if (settled) {
          const uint32_t base = __float_as_uint(-m);
          const Pair base2 = pair(base, base);
          float top[2] = {-INFINITY, -INFINITY};
          Pair sums[2] = {0, 0};
          uint32_t y[32];
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            uint32_t x[32];
            ptx::tmem_load_32x32b_x32(at + 32 * w, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              top[i & 1] = max3_nan(top[i & 1], __uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1]));
              const Pair z = fma2(pair(x[2 * i], x[2 * i + 1]), c2, base2);
              const float2 v = halves(z);
              const float e0 = ex2_approx(v.x), e1 = ex2_approx(v.y);
              sums[i & 1] = add2(sums[i & 1], pair(__float_as_uint(e0), __float_as_uint(e1)));
              // the numerators' rounding to the type, which the second product asks for;
              // their sum stays in fp32
              y[16 * w + i] = pack<T>(e0, e1);
            }
          }
          // (not so for NaN)
          settled = __all_sync(0xffffffffu, max3_nan(top[0], top[0], top[1]) * c - shift<T>() <= m + kSlack);
          if (settled) {
            tmem_store32(at, y);
            const float2 sum = halves(add2(sums[0], sums[1]));
            l += sum.x + sum.y;
          }
        }
        if (!settled) {
          // bit i: the row sees key 32 w + i
          const auto see = [&](uint32_t w) {
            const int64_t lo = static_cast<int64_t>(from) - key - 32 * w, hi = static_cast<int64_t>(to) - key - 32 * w;
            uint32_t bits = hi <= 0 || lo >= 32 ? 0u : 0xffffffffu;
            if (bits && hi < 32) bits &= (1u << hi) - 1;
            if (bits && lo > 0) bits &= ~((1u << lo) - 1);
            return there ? bits & good[w] : 0xffffffffu;
          };
          float top = -INFINITY;
#pragma unroll 1
          for (uint32_t w = 0; w < 2; ++w) {
            uint32_t x[32];
            ptx::tmem_load_32x32b_x32(at + 32 * w, x);
            const uint32_t bits = see(w);
#pragma unroll
            for (int i = 0; i < 32; ++i) top = fmaxf(top, bits >> i & 1 ? __uint_as_float(x[i]) : -INFINITY);
          }
          top = top * c - shift<T>();
          const bool grow = top > m + kSlack || (m == -INFINITY && top > m);
          if (__any_sync(0xffffffffu, grow)) {
            float f = 1.0f;
            if (grow) {
              f = ex2_approx(m - top);
              m = top;
              l *= f;
            }
            if (j + h > 0) {
              // The output so far: complete where the next half's scores are, which were
              // multiplied behind it, or by an arrival of its own before the last half.
              if (h == 0) {
                if (!wait_warp(sh, &sh.b.s_full[t][1], done & 1, a.status)) return;
              } else if (j + 1 < n) {
                if (!wait_warp(sh, &sh.b.s_full[t][0], (done + 1) & 1, a.status)) return;
              } else if (!wait_warp(sh, &sh.b.o_tail[t], outputs & 1, a.status)) {
                return;
              }
              ptx::tc_fence_after();
#pragma unroll 1
              for (uint32_t d = 0; d < cache.D; d += 32) {
                uint32_t x[32];
                ptx::tmem_load_32x32b_x32(o_at + d, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
                tmem_store32(o_at + d, x);
              }
            }
          }
          const float base = m == -INFINITY ? 0.0f : -m;
#pragma unroll 1
          for (uint32_t w = 0; w < 2; ++w) {
            uint32_t x[32], y[16];
            ptx::tmem_load_32x32b_x32(at + 32 * w, x);
            const uint32_t bits = see(w);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float e0 = bits >> 2 * i & 1 ? ex2_approx(fmaf(__uint_as_float(x[2 * i]), c, base)) : 0.0f;
              const float e1 = bits >> (2 * i + 1) & 1 ? ex2_approx(fmaf(__uint_as_float(x[2 * i + 1]), c, base)) : 0.0f;
              l += e0 + e1;
              y[i] = pack<T>(e0, e1);
            }
            tmem_store16(at + 16 * w, y);
          }
        }
        tmem_store_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&sh.b.p_full[t][h]);
      }
      ++done;
    }
    block_count += job->most;
    if (n) {
      if (!wait_warp(sh, &sh.b.o_full[t], outputs & 1, a.status)) return;
      ++outputs;
      ptx::tc_fence_after();
    }
    if (idle) {
      if (lane == 0) {
        if (n) ptx::mbar_arrive(&sh.b.o_free[t]);
        release_job(sh, i_job);
      }
      continue;
    }
    const uint32_t place = p.row0 + in_job, in_sequence = place / a.group;
    const uint64_t token = p.start + in_sequence;
    const uint32_t h = p.head * a.group + (place - in_sequence * a.group);
    const bool complete = p.opens && p.ends;
    float *const part = a.parts + (static_cast<size_t>(blockIdx.x) * 2 + (p.opens ? 1 : 0)) * part_floats<kRows, DP>();
    bool nan;
    if (complete) {
      TO *const out = static_cast<TO *>(const_cast<void *>(a.out.p)) + token * a.out.row_stride + h * a.out.head_stride;
      nan = put_rows<TO>(o_at, n > 0, cache.D, l == 0.0f ? 0.0f : 1.0f / l, there ? out : nullptr, staging);
    } else {
      nan = put_rows<float>(o_at, n > 0, cache.D, 1.0f, there ? part + in_job * DP : nullptr, staging);
    }
    if (n) {
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sh.b.o_free[t]);
    }
    if (there) {
      if (complete) put_lse(a, token, h, m, l);
      else {
        part[kRows * DP + in_job] = m;
        part[kRows * DP + kRows + in_job] = l;
      }
    }
    if (there && nan && l == l) *reinterpret_cast<volatile uint32_t *>(&sh.not_finite) = 1;
    __syncwarp();
    if (lane == 0) release_job(sh, i_job);
  }
}

// NaN from finite sums: where a value that other rows of the tile see, and this one does
// not, is not finite (0 times it is NaN), the row's own keys one by one.  By all warps of the
// CTA when its pieces are done: a row of 200003 keys takes 0.1 s, for which no wait of the
// pipeline is made (300 sequences of 40 such rows 872 ms, without infinite values 4.3).
template <typename T, typename TO, int DP> __device__ __forceinline__ void mend_rows(const AttentionArgs &a, const Share &share) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32, D = a.cache.D;
  Walk<kRows, kKeys> walk;
  Piece p;
  walk.start(a, share);
  while (walk.next(a, share, p)) {
    const bool complete = p.opens && p.ends;
    float *const part = a.parts + (static_cast<size_t>(blockIdx.x) * 2 + (p.opens ? 1 : 0)) * part_floats<kRows, DP>();
    for (uint32_t row = warp; row <= p.last; row += kThreads / 32) {
      const uint32_t lo = max(p.block_lo * kKeys, p.from);
      const uint32_t hi = min((p.block_lo + tile_blocks(a, p, row / kTile)) * kKeys, p.to);
      uint32_t from, to;
      seen(a, p.length, p.position(a, row), from, to);
      if (lo >= hi || (from <= lo && to >= hi)) continue;
      const uint32_t place = p.row0 + row, h = p.head * a.group + place % a.group;
      const uint64_t token = p.start + static_cast<uint64_t>(place / a.group);
      TO *const out = static_cast<TO *>(const_cast<void *>(a.out.p)) + token * a.out.row_stride + h * a.out.head_stride;
      bool nan = false;
      for (uint32_t d = lane; d < D; d += 32) {
        const float y = complete ? heads::element_of(out[d]) : part[row * DP + d];
        nan = nan || y != y;
      }
      if (!__any_sync(0xffffffffu, nan)) continue;
      if (!any_infinite<T>(a, p.sequence, p.head, lo, min(from, hi), lane) &&
          !any_infinite<T>(a, p.sequence, p.head, max(to, lo), hi, lane))
        continue;
      float acc[kMaxHead / 32], m, l;
      const T *q = static_cast<const T *>(a.q.p) + token * a.q.row_stride + h * a.q.head_stride;
      row_over_keys<T>(a, p.sequence, p.head, q, max(from, lo), min(to, hi), lane, m, l, acc);
      __syncwarp();
#pragma unroll
      for (int e = 0; e < static_cast<int>(kMaxHead) / 32; ++e) {
        if (lane + 32 * e >= D) continue;
        if (complete) heads::set_element(out[lane + 32 * e], l == 0.0f ? 0.0f : acc[e] / l);
        else part[row * DP + lane + 32 * e] = acc[e];
      }
      if (lane == 0) {
        if (complete) put_lse(a, token, h, m, l);
        else {
          part[kRows * DP + row] = m;
          part[kRows * DP + kRows + row] = l;
        }
      }
    }
  }
}

template <typename T, typename TO, int DP>
__global__ void __launch_bounds__(kThreads, 1) tile_kernel(const AttentionArgs a, const __grid_constant__ Maps maps) {
  constexpr int S = stages<DP>();
  extern __shared__ uint8_t raw[];
  uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t queries = ptx::smem_addr(smem), ring = queries + 2 * tile_bytes<DP>();
  uint8_t *const staging = smem + (2 + S) * tile_bytes<DP>();
  Shared &sh = *reinterpret_cast<Shared *>(staging + kStaging);
  const uint32_t warp = threadIdx.x / 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      ptx::mbar_init(&sh.b.full[i], kLoaders / 32);
    }
    for (int i = 0; i < kPairs; ++i) ptx::mbar_init(&sh.b.empty[i], 1);
    ptx::mbar_init(&sh.b.q_full, kLoaders / 32);
    ptx::mbar_init(&sh.b.q_empty, 1);
    for (int t = 0; t < 2; ++t) {
      for (int h = 0; h < 2; ++h) {
        ptx::mbar_init(&sh.b.s_full[t][h], 1);
        ptx::mbar_init(&sh.b.p_full[t][h], 4);
      }
      ptx::mbar_init(&sh.b.o_tail[t], 1);
      ptx::mbar_init(&sh.b.o_full[t], 1);
      ptx::mbar_init(&sh.b.o_free[t], 4);
    }
    for (int i = 0; i < kJobs; ++i) {
      ptx::mbar_init(&sh.b.job_full[i], 1);
      ptx::mbar_init(&sh.b.job_free[i], 8 + kLoaders / 32 + 1);  // softmax, loading, multiplying
    }
    ptx::mbar_init(&sh.b.drained, 1);
    sh.gave_up = 0;
    sh.not_finite = 0;
    ptx::fence_barrier_init();
  }
  if (warp == 12) {
    ptx::tmem_alloc(&sh.tmem, 512);
    ptx::tmem_relinquish();
  }
  pdl_enter();
  if (threadIdx.x == 13 * 32) a.joins[blockIdx.x] = Join{0xffffffffu, 0, 0, 0};
  ptx::tc_fence_before();
  const Share share = share_of<kRows, kKeys, kThreads>(a, blockIdx.x, gridDim.x, 2 * kKeys);
  if (threadIdx.x == 0) sh.share = share;  // for mend_rows, behind the last barrier
  ptx::tc_fence_after();
  if (warp < 8) {
    soften<T, TO, DP>(a, sh, staging);
  } else if (warp < 12) {
    load<T, DP>(a, maps, sh, queries, ring);
    await<0>();
    if (*reinterpret_cast<volatile uint32_t *>(&sh.gave_up)) {
      // TMA's copies may be on their way to this CTA's shared memory
      const uint64_t t0 = ptx::global_timer_ns();
      while (ptx::global_timer_ns() - t0 < 1000000) {
      }
    }
  } else if (warp == 12) {
    if (elect()) {
      multiply<T, DP>(a, sh, queries, ring);
      // everything issued is done before TMEM and the barriers go
      ptx::mma_commit(&sh.b.drained);
      if (!ptx::mbar_wait_bounded(&sh.b.drained, 0, kWaitLimitNs)) raise_flag(a.status, TL_FLAG_TIMEOUT);
    }
  } else if (threadIdx.x == 13 * 32) {
    plan_jobs(a, share, sh);
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 12) ptx::tmem_dealloc(sh.tmem, 512);
  if (sh.not_finite && !sh.gave_up) mend_rows<T, TO, DP>(a, sh.share);
}

bool encode(CUtensorMap *map, int32_t type, const void *base, uint32_t rank, const cuuint64_t *dims, const uint64_t *strides,
            const cuuint32_t *box) {
  EncodeTiledFn enc = tensor_map_encoder();
  if (!enc) return false;
  cuuint64_t bytes[3];
  for (uint32_t i = 0; i + 1 < rank; ++i) bytes[i] = strides[i] * 2;
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return enc(map, type == TL_FLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
             const_cast<void *>(base), dims, bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Boxes where the layout allows them; without, rows are copied one by one.
// x is 0 or 64 elements, so that every box starts on a 16-byte boundary.
Maps make_maps(const AttentionArgs &a) {
  const tl_paged_cache &c = a.cache;
  Maps m{};
  uint32_t rows = 32;
  while (rows >= 8 && c.page_size % rows) rows /= 2;
  if (rows >= 8 && c.pages) {
    const cuuint64_t dims[4] = {c.D, c.page_size, c.heads, c.pages};
    const uint64_t strides[3] = {c.slot_stride, c.heads > 1 ? c.head_stride : c.slot_stride, c.pages > 1 ? c.page_stride : c.slot_stride};
    const cuuint32_t box[4] = {64, rows, 1, 1};
    if (encode(&m.k, c.type, c.k, 4, dims, strides, box) && encode(&m.v, c.type, c.v, 4, dims, strides, box)) m.rows = rows;
  }
  // (heads or tokens that lie on one another, broadcast queries, are copied row by row)
  const bool apart = (a.q_heads == 1 || a.q.head_stride >= c.D) && (c.tokens == 1 || a.q.row_stride >= c.D);
  if (apart && a.group <= kTile && (a.group & (a.group - 1)) == 0) {
    const cuuint64_t dims[3] = {c.D, a.q_heads, c.tokens};
    const uint64_t strides[2] = {a.q_heads > 1 ? a.q.head_stride : c.D * 2u, c.tokens > 1 ? a.q.row_stride : c.D * 2u};
    const cuuint32_t box[3] = {64, a.group, kTile / a.group};
    m.queries = encode(&m.q, c.type, a.q.p, 3, dims, strides, box);
  }
  return m;
}

template <typename T, typename TO, int DP> void launch(const AttentionArgs &a, const Plan &p, cudaStream_t s) {
  constexpr size_t smem = smem_bytes<DP>();
  (void)cudaFuncSetAttribute(tile_kernel<T, TO, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  launch_pdl(tile_kernel<T, TO, DP>, p.ctas, kThreads, smem, s, a, make_maps(a));
  launch_pdl(join_kernel<TO, kRows, DP>, dim3(p.ctas, kRows / 16), 128, 0, s, a);
}

}  // namespace

Plan tile_plan(const AttentionArgs &a) {
  Plan p{};
  p.ctas = kNumSMs;
  p.part_floats = kRows * (a.cache.D > 64 ? 128 : 64) + 2 * kRows;
  return p;
}

void launch_tile(const AttentionArgs &a, const Plan &p, bool wide, cudaStream_t s) {
  const bool narrow = a.cache.D <= 64;
#define L(T, TO) narrow ? launch<T, TO, 64>(a, p, s) : launch<T, TO, 128>(a, p, s)
  if (a.cache.type == TL_FLOAT16) { if (wide) L(__half, float); else L(__half, __half); }
  else if (wide) L(__nv_bfloat16, float);
  else L(__nv_bfloat16, __nv_bfloat16);
#undef L
}

}  // namespace paged
}  // namespace tl
