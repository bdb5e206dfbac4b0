// Causal attention over the quantised K/V cache: checks, plan and dispatch.
#include <cmath>

#include "kv_attention.cuh"
#include "tmap.cuh"

namespace icx {

AttendPlan plan_attend(const KvView& c, const KvTokens& w, int q_heads, int type) {
  AttendPlan p{};
  if (prompt_preferred(c, w, q_heads, type)) {
    p.bytes = plan_prompt(c, w, q_heads, type).bytes;
    return p;
  }
  const int share = q_heads / c.heads;
  const int64_t rows = (w.tokens + w.batch - 1) / w.batch * share;
  const int64_t reach = (int64_t)w.width << c.page_shift;
  p.nt = 1;
  if (type == ICX_F32 && att_most_nt<float>(c.dim) == 2 && rows > 8) {
    // steps per warp with one tile of 8 rows: from 64 on, two
    const int64_t steps = (w.tokens * share / 8 + w.batch) * c.heads * (reach / att_step(c.dim, c.bits, 8) + 1);
    if (steps >= 64ll * sm_count() * kAttWarps * att_resident(c.dim, 1, 4)) p.nt = 2;
  }
  const int R = 8 * p.nt, step = att_step(c.dim, c.bits, R);
  const int64_t runs = (w.tokens * share / R + w.batch) * c.heads;   // row tiles
  const int64_t resident = (int64_t)sm_count() * att_resident(c.dim, p.nt, (int)float_bytes(type));
  // Up to four steps per warp of a CTA, or in one warp, are over before a second
  // launch would be; many row tiles are shared out evenly instead.
  if (reach <= step || (reach <= 4 * step && runs > resident)) {
    p.split = kSplitNone;
    p.unit = 4 * step;
  } else if (reach <= 4 * kAttWarps * step && runs <= 2 * resident) {
    p.split = kSplitCta;
    p.unit = 1 << 30;
    p.ctas = (int)runs;
    return p;
  } else {
    p.split = kSplitAny;
    p.unit = step;
  }
  const int64_t blocks = reach > p.unit ? (reach + p.unit - 1) / p.unit : 1;
  const int64_t want = (runs * blocks + kAttWarps - 1) / kAttWarps;
  p.ctas = (int)(want < resident ? want : resident);
  if (p.split == kSplitAny) {
    p.prefix_bytes = ((size_t)(w.batch + 1) * 8 + 255) & ~size_t(255);
    p.bytes = p.prefix_bytes + (size_t)p.ctas * kAttWarps * 2 * R * (c.dim + 2) * 4;
  }
  return p;
}

}  // namespace icx

using namespace icx;

extern "C" size_t icx_kv_cache_attention_workspace_bytes(const icx_kv_cache* cache, const icx_kv_tokens* where,
                                                         int q_heads, int type) {
  KvView c;
  KvTokens w;
  if (kv_views("KvCacheAttention", cache, where, &c, &w) || w.tokens == 0 || w.batch == 0 || q_heads < 1 ||
      q_heads % c.heads)
    return 0;
  if (!is_float_type(type)) return 0;
  return plan_attend(c, w, q_heads, type).bytes;
}

extern "C" int icx_kv_cache_attention(void* stream, const icx_kv_cache* cache, const icx_kv_tokens* where,
                                      const void* d_q, int type, int q_heads, int64_t q_token_stride,
                                      int64_t q_head_stride, float scale, void* d_out, void* d_workspace,
                                      size_t workspace_bytes) {
  KvView c;
  KvTokens w;
  const int rc = kv_views("KvCacheAttention", cache, where, &c, &w);
  if (rc) return rc;
  ICX_REQUIRE(is_float_type(type), "KvCacheAttention: q must be Float32, Float16 or BFloat16");
  ICX_REQUIRE(q_heads >= 1 && q_heads % c.heads == 0, "KvCacheAttention: q_heads %d is no multiple of kv_heads %d",
              q_heads, c.heads);
  ICX_REQUIRE(q_token_stride >= 0 && q_head_stride >= 0, "KvCacheAttention: negative stride");
  scale *= 1.4426950408889634f;
  ICX_REQUIRE(std::isfinite(scale), "KvCacheAttention: scale must be finite");
  ICX_REQUIRE(w.tokens * q_heads < (1ll << 31), "KvCacheAttention: tokens x q_heads beyond 2^31");
  if (w.tokens == 0 || w.batch == 0) return ICX_OK;
  ICX_REQUIRE(d_q && d_out, "KvCacheAttention: null operand");
  ICX_REQUIRE((reinterpret_cast<uintptr_t>(d_out) & 15) == 0, "KvCacheAttention: out must be 16-byte aligned");
  const bool prompt = prompt_preferred(c, w, q_heads, type);
  const AttendPlan p = plan_attend(c, w, q_heads, type);
  if (p.bytes > 0 && (!d_workspace || workspace_bytes < p.bytes)) {
    set_error("KvCacheAttention: workspace %zu bytes < %zu required", d_workspace ? workspace_bytes : 0, p.bytes);
    return ICX_ERR_WORKSPACE;
  }
  ICX_REQUIRE((reinterpret_cast<uintptr_t>(d_workspace) & 15) == 0, "KvCacheAttention: workspace must be 16-byte aligned");
  const size_t e = float_bytes(type);
  AttendArgs a{};
  a.q = d_q;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.q_heads = q_heads;
  a.q_vec = (reinterpret_cast<uintptr_t>(d_q) | (size_t)q_token_stride * e | (size_t)q_head_stride * e) % (4 * e) == 0;
  a.scale = scale;
  a.out = d_out;
  a.split = p.split;
  a.unit = p.unit;
  a.prefix = static_cast<int64_t*>(d_workspace);
  a.partial = reinterpret_cast<float*>(static_cast<char*>(d_workspace) + p.prefix_bytes);
  cudaStream_t s = as_stream(stream);
  if (prompt) return launch_prompt(s, c, w, a, type);
  int r = ICX_OK;
  ICX_FLOAT_DISPATCH(type, r = launch_attend<T>(s, c, w, a, p));
  return r;
}
