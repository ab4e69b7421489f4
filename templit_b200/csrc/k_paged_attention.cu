// Attention of new tokens over a paged cache (include/templit_cuda.h:
// tl_paged_attention): softmax(scale q k^T) v over the keys that each token
// sees.  Checks, and the choice between the kernels.
#include "paged_attention.cuh"

#include <cmath>

namespace tl {
namespace paged {
namespace {

// Checks a descriptor; *nothing where there is no work.
int attention_args(const char *who, const tl_paged_attention_desc *d, AttentionArgs &a, bool *nothing) {
  const std::string w = std::string(who) + ": ";
  if (!d) return fail(TL_ERR_INVALID, w + "null descriptor");
  a.cache = d->cache;
  bool aligned = false;
  if (int rc = check_cache(who, a.cache, &aligned)) return rc;
  const tl_paged_cache &c = a.cache;
  if (c.D > kMaxHead || c.D % 8) return fail(TL_ERR_UNSUPPORTED, w + "heads are a multiple of 8 elements, at most 128");
  if (!d->q_heads || d->q_heads % c.heads) return fail(TL_ERR_INVALID, w + "q_heads is a multiple of the key heads");
  if (d->out_type != c.type && d->out_type != TL_FLOAT32) return fail(TL_ERR_INVALID, w + "out_type is the cache's or fp32");
  if (d->causal != 0 && d->causal != 1) return fail(TL_ERR_INVALID, w + "causal is 0 or 1");
  if (d->window && !d->causal) return fail(TL_ERR_INVALID, w + "a window needs causal");
  if (!std::isfinite(d->scale * kLog2e)) return fail(TL_ERR_INVALID, w + "scale / ln 2 is finite");
  if (static_cast<uint64_t>(c.tokens) * d->q_heads >> 32) return fail(TL_ERR_RANGE, w + "more than 2^32 - 1 query rows");
  *nothing = !c.tokens || !c.sequences;
  if (*nothing) return TL_OK;
  if (int rc = heads::check_view(who, "q", d->q, c.type, 1, c.tokens, d->q_heads, c.D, false)) return rc;
  if (int rc = heads::check_view(who, "out", d->out, d->out_type, 1, c.tokens, d->q_heads, c.D, true)) return rc;
  // rows with values that are not finite may be read again when others are written
  if (d->out.p == d->q.p) return fail(TL_ERR_INVALID, w + "out is q");
  if (!aligned || !heads::aligned_view(d->q, c.type, false, 8) || !heads::aligned_view(d->out, d->out_type, false, 8))
    return fail(TL_ERR_UNSUPPORTED, w + "rows are not 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(d->lse) % 4) return fail(TL_ERR_INVALID, w + "lse not aligned");
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
  return TL_OK;
}

// Many rows a key head go to the tensor cores' tiles (16-bit types; a scale
// that is not positive would turn the order of the scores round there): more than the
// 16 that read a sequence's keys once in the other kernel.  64 sequences of 8191 keys,
// 8 key heads of 128 bf16: 16 rows take 429 us there and 382 in the other, 20 rows 424
// and 708, 256 rows 586 and 4933.  (One sequence of them: 20 rows 44 us and 36.)
// One choice for the whole call: of 64 sequences of 16 to 8191 keys with one token and 4
// query heads a key head each, 91 us in the other kernel, 122 here where max_new is not given.
// The tiles' waits end after 2 s, and a job is waited for as a whole: 2^26 keys take 1.1 s
// there (2.1 us for 128), so that sequences which may be longer stay with the other kernel,
// whose warps wait for nothing but their own copies.
bool tiled(const tl_paged_attention_desc *d, const AttentionArgs &a, uint32_t max_new) {
  return a.cache.type != TL_FLOAT32 && d->scale > 0.0f && static_cast<uint64_t>(max_new) * a.group > 16 && a.most <= 1u << 26;
}

uint32_t most_new(const tl_paged_attention_desc *d) {
  return d->max_new && d->max_new < d->cache.tokens ? d->max_new : d->cache.tokens;
}

}  // namespace
}  // namespace paged
}  // namespace tl

using namespace tl;
using namespace tl::paged;

extern "C" {

size_t tl_paged_attention_workspace_size(const tl_paged_attention_desc *d) {
  AttentionArgs a{};
  bool nothing = false;
  if (attention_args("tl_paged_attention_workspace_size", d, a, &nothing) || nothing) return 0;
  const uint32_t n = most_new(d);
  return plan_bytes(tiled(d, a, n) ? tile_plan(a) : step_plan(a, n));
}

int tl_paged_attention(const tl_paged_attention_desc *d, void *stream) {
  const char *who = "tl_paged_attention";
  const std::string w = std::string(who) + ": ";
  AttentionArgs a{};
  bool nothing = false;
  if (int rc = attention_args(who, d, a, &nothing)) return rc;
  if (nothing) return TL_OK;
  const uint32_t n = most_new(d);
  const bool tiles = tiled(d, a, n);
  const Plan p = tiles ? tile_plan(a) : step_plan(a, n);
  const uint64_t bytes = plan_bytes(p);
  if (bytes) {
    if (!d->workspace || d->workspace_bytes < bytes) return fail(TL_ERR_INVALID, w + "workspace too small");
    if (!aligned16(d->workspace)) return fail(TL_ERR_INVALID, w + "workspace is not 16-byte aligned");
  }
  a.whole = p.whole;
  a.joins = static_cast<Join *>(d->workspace);
  a.parts = reinterpret_cast<float *>(a.joins + p.ctas);
  a.status = device_status_ptr();
  if (!a.status) return fail(TL_ERR_CUDA, w + "no status word");
  (tiles ? launch_tile : launch_step)(a, p, d->out_type != a.cache.type, as_stream(stream));
  return launch_status(who);
}

}  // extern "C"
