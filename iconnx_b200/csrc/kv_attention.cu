// Causal attention over the quantised K/V cache.
#include <cmath>

#include "capi.cuh"
#include "common.cuh"
#include "kv_cache.cuh"

namespace icx {

template <typename T>
struct QueryArgs {
  const T* q;
  int64_t token_stride, head_stride;
  int q_heads;
  float scale;   // of the scores, times log2(e)
  T* out;
};

__device__ __forceinline__ uint32_t k_code(const uint8_t* row, int dim, int bits, int d) {
  const int j = d >> 4, t = (d >> 2) & 3, i = d & 3;
  const uint8_t* chunk = row + t * (dim * bits / 32);
  if (bits == 8) return chunk[4 * j + (((i & 1) << 1) | (i >> 1))];
  const int nib = (((i & 1) << 2) | (i & 2)) + (j & 1);
  return (chunk[4 * (j >> 1) + (nib >> 1)] >> (4 * (nib & 1))) & 15u;
}

__device__ __forceinline__ uint32_t v_code(const uint8_t* row, int dim, int bits, int d) {
  const int m = d >> 4, g = (d >> 1) & 7, k = 2 * m + (d & 1);
  const uint8_t* chunk = row + g * (dim * bits / 64);
  return bits == 8 ? chunk[k] : (chunk[k >> 1] >> (4 * (k & 1))) & 15u;
}

// One warp per (token, query head), one position at a time.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_attend_kernel(const KvView c, const KvTokens w, const QueryArgs<T> a) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= w.tokens * a.q_heads) return;
  const int64_t token = item / a.q_heads;
  const int hq = (int)(item % a.q_heads), head = hq / (a.q_heads / c.heads);
  const int b = kv_sequence(w, token);
  if (b < 0) return;
  const int64_t end = w.cu ? (int64_t)w.cu[b + 1] : token + 1;
  const int64_t last = (int64_t)w.lens[b] - end + token;
  float q[E], o[E] = {};
#pragma unroll
  for (int e = 0; e < E; ++e)
    q[e] = to_f32(a.q[token * a.token_stride + hq * a.head_stride + lane + 32 * e]) * a.scale;
  float m = -INFINITY, l = 0.0f;
  for (int p = 0; p <= last; ++p) {
    const int64_t page = kv_page(c, w, b, p);
    if (page < 0) {
      record_status(ICX_DEVICE_BAD_PAGE);
      continue;
    }
    const int64_t row = kv_row(c, page, head, p);
    const uint8_t* kr = c.codes[0] + row * (D * c.bits / 8);
    const uint8_t* vr = c.codes[1] + row * (D * c.bits / 8);
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + 32 * e;
      const uint32_t pr = c.params[0][row * (D / c.group) + d / c.group];
      s = fmaf(q[e], fmaf((float)k_code(kr, D, c.bits, d), param_scale(pr), param_low(pr)), s);
    }
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.0f : exp2f(m - mn), pw = exp2f(s - mn);
    m = mn;
    l = fmaf(l, f, pw);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + 32 * e;
      const uint32_t pr = c.params[1][row * (D / c.group) + d / c.group];
      o[e] = fmaf(o[e], f, pw * fmaf((float)v_code(vr, D, c.bits, d), param_scale(pr), param_low(pr)));
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.out[(token * a.q_heads + hq) * D + lane + 32 * e] = from_f32<T>(l != 0.0f ? o[e] / l : 0.0f);
}

}  // namespace icx

using namespace icx;

extern "C" size_t icx_kv_cache_attention_workspace_bytes(const icx_kv_cache* cache, const icx_kv_tokens* where,
                                                         int q_heads) {
  return 0;
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
  ICX_REQUIRE(std::isfinite(scale), "KvCacheAttention: scale must be finite");
  if (w.tokens == 0 || w.batch == 0) return ICX_OK;
  ICX_REQUIRE(d_q && d_out, "KvCacheAttention: null operand");
  cudaStream_t s = as_stream(stream);
  const dim3 grid((unsigned)((w.tokens * q_heads + 7) / 8));
  ICX_FLOAT_DISPATCH(type, {
    QueryArgs<T> a{static_cast<const T*>(d_q), q_token_stride, q_head_stride, q_heads, scale * 1.4426950408889634f,
                   static_cast<T*>(d_out)};
    auto kern = c.dim == 64 ? kv_attend_kernel<T, 64> : c.dim == 128 ? kv_attend_kernel<T, 128> : kv_attend_kernel<T, 256>;
    ICX_CUDA(launch_pdl(kern, grid, dim3(256), 0, s, c, w, a));
  });
  return ICX_OK;
}
