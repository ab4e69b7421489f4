// Token scoring: log probability of given tokens, entropy and top
// alternatives of rows of logits, and their gradient
// (tl_token_logprob_rows, tl_token_logprob_backward_rows).
#include "token_rows.cuh"

namespace tl {
namespace token {

static int bad(const char *who, const char *what) {
  return fail(TL_ERR_INVALID, std::string(who) + ": " + what);
}

int check_rows(const char *who, const void *logits, int32_t type, uint32_t rows, uint32_t vocab,
               float temperature, uint64_t &row_stride) {
  if (type != TL_FLOAT32 && type != TL_FLOAT16 && type != TL_BFLOAT16)
    return bad(who, "unknown logit type");
  if (vocab == 0) return bad(who, "logits need a non-empty final dimension");
  if (!(temperature > 0.0f) || std::isinf(temperature))
    return bad(who, "temperature must be positive and finite");
  if (rows == 0) return TL_OK;
  if (row_stride == 0) row_stride = vocab;
  if (row_stride < vocab && rows > 1) return bad(who, "row stride below the row's length");
  if (row_stride > static_cast<uint64_t>(LLONG_MAX) / 4 / rows)
    return fail(TL_ERR_RANGE, std::string(who) + ": rows reach beyond the address space");
  if (!logits) return bad(who, "null logits");
  if (reinterpret_cast<uintptr_t>(logits) % type_size(type))
    return bad(who, "logits not aligned to their type");
  return TL_OK;
}

int check_gradient(const char *who, const void *logits, uint64_t row_stride, void *dlogits,
                   int32_t type, uint32_t rows, uint32_t vocab, uint64_t &d_row_stride) {
  if (d_row_stride == 0) d_row_stride = vocab;
  if (d_row_stride < vocab && rows > 1) return bad(who, "gradient row stride below the row's length");
  if (d_row_stride > static_cast<uint64_t>(LLONG_MAX) / 4 / rows)
    return fail(TL_ERR_RANGE, std::string(who) + ": gradient rows reach beyond the address space");
  if (!dlogits) return bad(who, "null dlogits");
  if (reinterpret_cast<uintptr_t>(dlogits) % type_size(type))
    return bad(who, "dlogits not aligned to their type");
  if (dlogits == logits && rows > 1 && d_row_stride != row_stride)
    return bad(who, "a gradient in place of the logits needs their row stride");
  return TL_OK;
}

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

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
  uint32_t *status;
};

// log q of a logit from its row's sums; -inf in a row of -inf.
__device__ __forceinline__ float log_q(float z, const Sums &r, float log_s, float inv_t) {
  if (r.m == -INFINITY) return r.s != r.s ? r.s : -INFINITY;
  return (z - r.m) * inv_t - log_s;
}

// One CTA per row.
template <typename T>
__global__ void __launch_bounds__(kThreads) score_kernel(const ScoreArgs a) {
  __shared__ Sums scratch[kWarps];
  __shared__ uint64_t best[kWarps];
  pdl_enter();
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    Sums v = empty_sums();
    for (uint32_t j = threadIdx.x; j < a.vocab; j += kThreads) add_logit(v, to_float(z[j]), a.c);
    v = block_merge<kWarps>(v, a.c, scratch);
    const float log_s = logf(v.s);
    if (threadIdx.x == 0) {
      if (a.targets) {
        const uint32_t t = a.targets[row];
        float out = 0.0f;
        if (t < a.vocab) out = log_q(to_float(z[t]), v, log_s, a.inv_t);
        else if (t != TL_NO_TOKEN) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
        a.logprob[row] = out;
      }
      if (a.entropy) a.entropy[row] = v.s == 0.0f ? 0.0f : log_s - v.h * a.inv_t / v.s;
      if (a.stats) {
        a.stats[2 * row] = v.m;
        a.stats[2 * row + 1] = v.s;
      }
    }
    // the i-th alternative: the largest (logit, lowest id) below the last
    uint64_t last = ~0ull;
    for (uint32_t i = 0; i < a.top; ++i) {
      uint64_t mine = 0;
      for (uint32_t j = threadIdx.x; j < a.vocab; j += kThreads) {
        const uint64_t key = (static_cast<uint64_t>(order_of(to_float(z[j]))) << 32) | ~j;
        if (key < last && key > mine) mine = key;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, mine, o);
        if (other > mine) mine = other;
      }
      __syncthreads();
      if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = mine;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w)
        if (best[w] > mine) mine = best[w];
      last = mine;
      if (threadIdx.x == 0) {
        const uint32_t id = ~static_cast<uint32_t>(mine);
        a.top_ids[row * a.top + i] = id;
        a.top_logprob[row * a.top + i] = log_q(to_float(z[id]), v, log_s, a.inv_t);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) score_backward_kernel(const ScoreArgs a) {
  pdl_enter();
  for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *z = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *dz = static_cast<T *>(a.dlogits) + row * a.d_row_stride;
    const float m = a.stats[2 * row], s = a.stats[2 * row + 1];
    uint32_t t = TL_NO_TOKEN;
    float gl = 0.0f, ge = 0.0f, entropy = 0.0f;
    if (a.d_logprob) {
      t = a.targets[row];
      if (t < a.vocab) gl = a.d_logprob[row] * a.inv_t;
      else if (t != TL_NO_TOKEN && threadIdx.x == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
    }
    if (a.d_entropy) {
      ge = a.d_entropy[row] * a.inv_t;
      if (ge != 0.0f) entropy = a.entropy[row];
    }
    const bool none = s == 0.0f || (gl == 0.0f && ge == 0.0f);
    // dz = q (-gl - ge (log q + H)) + gl [j = t]
    const float inv_s = 1.0f / s, log_s = logf(s), base = entropy - log_s;
    for (uint32_t j = threadIdx.x; j < a.vocab; j += kThreads) {
      float g = 0.0f;
      if (!none) {
        const float d = to_float(z[j]) - m;
        const float q = ex2_approx(d * a.c) * inv_s;
        g = q == 0.0f ? 0.0f : -q * fmaf(ge, fmaf(d, a.inv_t, base), gl);
        if (j == t) g += gl;
      }
      dz[j] = from_float<T>(g);
    }
  }
}

unsigned grid_of(uint32_t rows) {
  const uint32_t most = kNumSMs * 64u;
  return rows < most ? rows : most;
}

int score_args(const char *who, const tl_token_logprob_desc *d, ScoreArgs &a) {
  if (!d) return bad(who, "null descriptor");
  a.row_stride = d->row_stride;
  if (int rc = check_rows(who, d->logits, d->type, d->rows, d->vocab, d->temperature, a.row_stride))
    return rc;
  a.logits = d->logits;
  a.rows = d->rows;
  a.vocab = d->vocab;
  a.top = d->top;
  a.c = static_cast<float>(1.4426950408889634 / d->temperature);
  a.inv_t = static_cast<float>(1.0 / d->temperature);
  a.targets = d->targets;
  a.logprob = d->logprob;
  a.entropy = d->entropy;
  a.stats = d->stats;
  a.top_logprob = d->top_logprob;
  a.top_ids = d->top_ids;
  a.d_logprob = d->d_logprob;
  a.d_entropy = d->d_entropy;
  a.dlogits = d->dlogits;
  a.d_row_stride = d->d_row_stride;
  return TL_OK;
}

}  // namespace
}  // namespace token
}  // namespace tl

using namespace tl;
using namespace tl::token;

#define TL_BY_TYPE(TYPE, LAUNCH)                   \
  switch (TYPE) {                                  \
    case TL_FLOAT32: LAUNCH(float); break;         \
    case TL_FLOAT16: LAUNCH(__half); break;        \
    default: LAUNCH(__nv_bfloat16); break;         \
  }

extern "C" {

int tl_token_logprob_rows(const tl_token_logprob_desc *desc, void *stream) {
  const char *who = "tl_token_logprob_rows";
  ScoreArgs a{};
  if (int rc = score_args(who, desc, a)) return rc;
  if (a.top > TL_TOKEN_MAX_TOP) return fail(TL_ERR_RANGE, std::string(who) + ": more than 128 alternatives");
  if (a.top > a.vocab) return bad(who, "more alternatives than tokens");
  if (a.rows == 0) return TL_OK;
  if (!a.targets != !a.logprob) return bad(who, "targets and logprob go together");
  if (a.top && (!a.top_logprob || !a.top_ids)) return bad(who, "null top_logprob or top_ids");
  if (!a.logprob && !a.entropy && !a.stats && !a.top) return bad(who, "no output");
  a.status = device_status_ptr();
  if (!a.status) return fail(TL_ERR_CUDA, std::string(who) + ": no status word");
#define L(T) launch_pdl(score_kernel<T>, grid_of(a.rows), kThreads, 0, as_stream(stream), a)
  TL_BY_TYPE(desc->type, L)
#undef L
  return launch_status(who);
}

int tl_token_logprob_backward_rows(const tl_token_logprob_desc *desc, void *stream) {
  const char *who = "tl_token_logprob_backward_rows";
  ScoreArgs a{};
  if (int rc = score_args(who, desc, a)) return rc;
  if (a.rows == 0) return TL_OK;
  if (int rc = check_gradient(who, a.logits, a.row_stride, a.dlogits, desc->type, a.rows, a.vocab,
                              a.d_row_stride))
    return rc;
  if (!a.stats) return bad(who, "null stats");
  if (!a.d_logprob && !a.d_entropy) return bad(who, "no incoming gradient");
  if (a.d_logprob && !a.targets) return bad(who, "d_logprob without targets");
  if (a.d_entropy && !a.entropy) return bad(who, "d_entropy without entropy");
  a.status = device_status_ptr();
  if (!a.status) return fail(TL_ERR_CUDA, std::string(who) + ": no status word");
#define L(T) launch_pdl(score_backward_kernel<T>, grid_of(a.rows), kThreads, 0, as_stream(stream), a)
  TL_BY_TYPE(desc->type, L)
#undef L
  return launch_status(who);
}

}  // extern "C"
