// Attention of new tokens over a paged cache (include/templit_cuda.h:
// tl_paged_attention): softmax(scale q k^T) v over the keys that each token
// sees.
#include "paged_attention.cuh"

#include <cmath>

namespace tl {
namespace paged {
namespace {

constexpr int kRowWarps = 4;

template <typename T, typename TO>
__global__ void __launch_bounds__(kRowWarps * 32) rows_kernel(const AttentionArgs a) {
  pdl_enter();
  const tl_paged_cache &c = a.cache;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t items = static_cast<uint64_t>(c.tokens) * a.q_heads, warps = static_cast<uint64_t>(gridDim.x) * kRowWarps;
  for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * kRowWarps + threadIdx.x / 32; item < items; item += warps) {
    const uint32_t token = static_cast<uint32_t>(item / a.q_heads), h = static_cast<uint32_t>(item % a.q_heads);
    const uint32_t s = sequence_at(c, token, lane);
    if (s == 0xffffffffu) continue;
    const Sequence q = sequence_of(c, s, a.most);
    if (q.bad && lane == 0) raise_flag(a.status, TL_FLAG_INDEX_RANGE);
    if (token < q.start || token - q.start >= q.count) continue;
    const int64_t position = static_cast<int64_t>(q.length) - q.count + (token - q.start);
    uint32_t from, to;
    seen(a, q.length, position, from, to);
    float m, l, acc[kMaxHead / 32];
    const T *row = static_cast<const T *>(a.q.p) + token * a.q.row_stride + h * a.q.head_stride;
    row_over_keys<T>(a, s, h / a.group, row, from, to, lane, m, l, acc);
    TO *out = static_cast<TO *>(const_cast<void *>(a.out.p)) + token * a.out.row_stride + h * a.out.head_stride;
#pragma unroll
    for (int i = 0; i < static_cast<int>(kMaxHead) / 32; ++i)
      if (lane + 32 * i < c.D) heads::set_element(out[lane + 32 * i], l == 0.0f ? 0.0f : acc[i] / l);
    if (lane == 0 && a.lse) a.lse[static_cast<uint64_t>(token) * a.q_heads + h] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
  }
}

}  // namespace
}  // namespace paged
}  // namespace tl

using namespace tl;
using namespace tl::paged;

extern "C" {

size_t tl_paged_attention_workspace_size(const tl_paged_attention_desc *d) {
  (void)d;
  return 0;
}

int tl_paged_attention(const tl_paged_attention_desc *d, void *stream) {
  const char *who = "tl_paged_attention";
  const std::string w = std::string(who) + ": ";
  if (!d) return fail(TL_ERR_INVALID, w + "null descriptor");
  AttentionArgs a{};
  a.cache = d->cache;
  bool aligned = false;
  if (int rc = check_cache(who, a.cache, &aligned)) return rc;
  const tl_paged_cache &c = a.cache;
  if (c.D > kMaxHead || c.D % 8) return fail(TL_ERR_UNSUPPORTED, w + "heads are a multiple of 8 elements, at most 128");
  if (!d->q_heads || d->q_heads % c.heads) return fail(TL_ERR_INVALID, w + "q_heads is a multiple of the key heads");
  if (d->out_type != c.type && d->out_type != TL_FLOAT32) return fail(TL_ERR_INVALID, w + "out_type is the cache's or fp32");
  if (d->causal != 0 && d->causal != 1) return fail(TL_ERR_INVALID, w + "causal is 0 or 1");
  if (d->window && !d->causal) return fail(TL_ERR_INVALID, w + "a window needs causal");
  if (!std::isfinite(d->scale)) return fail(TL_ERR_INVALID, w + "scale is finite");
  if (!c.tokens || !c.sequences) return TL_OK;
  if (int rc = heads::check_view(who, "q", d->q, c.type, 1, c.tokens, d->q_heads, c.D, false)) return rc;
  if (int rc = heads::check_view(who, "out", d->out, d->out_type, 1, c.tokens, d->q_heads, c.D, true)) return rc;
  if (heads::half_in_place(d->out, d->out_type, d->q, c.type, false))
    return fail(TL_ERR_INVALID, w + "out is q with another layout or type");
  if (!aligned || !heads::aligned_view(d->q, c.type, false) || !heads::aligned_view(d->out, d->out_type, false))
    return fail(TL_ERR_UNSUPPORTED, w + "rows are not 16-byte aligned");
  a.q = d->q;
  a.out = d->out;
  a.q_heads = d->q_heads;
  a.group = d->q_heads / c.heads;
  a.window = d->window;
  a.causal = static_cast<uint32_t>(d->causal);
  a.most = table_keys(c);
  if (d->max_length && d->max_length < a.most) a.most = d->max_length;
  a.scale = d->scale;
  a.lse = d->lse;
  a.status = device_status_ptr();
  if (!a.status) return fail(TL_ERR_CUDA, w + "no status word");
  const uint64_t ctas = (static_cast<uint64_t>(c.tokens) * a.q_heads + kRowWarps - 1) / kRowWarps;
  const unsigned grid = static_cast<unsigned>(ctas < kNumSMs * 64ull ? ctas : kNumSMs * 64ull);
  cudaStream_t s = as_stream(stream);
  const bool wide = d->out_type == TL_FLOAT32;
  if (c.type == TL_FLOAT32) launch_pdl(rows_kernel<float, float>, grid, kRowWarps * 32, 0, s, a);
  else if (c.type == TL_FLOAT16) {
    if (wide) launch_pdl(rows_kernel<__half, float>, grid, kRowWarps * 32, 0, s, a);
    else launch_pdl(rows_kernel<__half, __half>, grid, kRowWarps * 32, 0, s, a);
  } else {
    if (wide) launch_pdl(rows_kernel<__nv_bfloat16, float>, grid, kRowWarps * 32, 0, s, a);
    else launch_pdl(rows_kernel<__nv_bfloat16, __nv_bfloat16>, grid, kRowWarps * 32, 0, s, a);
  }
  return launch_status(who);
}

}  // extern "C"
