// Quantised K/V cache: append (quantise) and read (dequantise).
//
// Half a warp takes 64 dimensions of one (token, head) of K or V, four
// consecutive ones per lane, so a quantisation group is 8 or 16 lanes and
// every code word of the layout is put together from lanes of one half warp.
#include "kv_cache.cuh"

#include "capi.cuh"
#include "common.cuh"

namespace icx {

int kv_views(const char* what, const icx_kv_cache* c, const icx_kv_tokens* w, KvView* view,
             KvTokens* tokens) {
  ICX_REQUIRE(c && w, "%s: null argument", what);
  ICX_REQUIRE(c->bits == 4 || c->bits == 8, "%s: bits must be 4 or 8, got %d", what, c->bits);
  ICX_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256,
              "%s: head_dim must be 64, 128 or 256, got %d", what, c->head_dim);
  ICX_REQUIRE(c->group == 32 || c->group == 64, "%s: group must be 32 or 64, got %d", what, c->group);
  int shift = 4;
  while (shift < 10 && (1 << shift) < c->page_size) ++shift;
  ICX_REQUIRE((1 << shift) == c->page_size, "%s: page_size must be a power of two in 16..1024, got %d", what,
              c->page_size);
  ICX_REQUIRE(c->kv_heads >= 1 && c->kv_heads <= 1024, "%s: kv_heads must be in 1..1024, got %d", what,
              c->kv_heads);
  ICX_REQUIRE(c->pages >= 0 && c->pages < (1ll << 31), "%s: pages out of range", what);
  ICX_REQUIRE(w->batch >= 0 && w->batch < (1 << 20) && w->table_width >= 0 && w->tokens >= 0 &&
                  w->tokens < (1ll << 31),
              "%s: batch, table width or tokens out of range", what);
  ICX_REQUIRE((int64_t)w->table_width << shift < (1ll << 31), "%s: page table row beyond 2^31 positions", what);
  ICX_REQUIRE(w->d_cu_tokens || w->tokens == w->batch,
              "%s: without cu_tokens there is one token per sequence (%lld tokens, batch %d)", what,
              (long long)w->tokens, w->batch);
  if (w->tokens > 0 && w->batch > 0) {
    ICX_REQUIRE(w->d_seq_lens && (w->d_page_table || w->table_width == 0), "%s: null index array", what);
    ICX_REQUIRE(c->pages == 0 || (c->k_codes && c->v_codes && c->k_params && c->v_params),
                "%s: null cache buffer", what);
    const uintptr_t all = reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes) |
                          reinterpret_cast<uintptr_t>(c->k_params) | reinterpret_cast<uintptr_t>(c->v_params);
    ICX_REQUIRE((all & 15) == 0, "%s: cache buffers must be 16-byte aligned", what);
  }
  *view = KvView{{static_cast<uint8_t*>(c->k_codes), static_cast<uint8_t*>(c->v_codes)},
                 {static_cast<uint32_t*>(c->k_params), static_cast<uint32_t*>(c->v_params)},
                 c->pages, shift, c->kv_heads, c->head_dim, c->bits, c->group};
  *tokens = KvTokens{w->d_page_table, w->d_seq_lens, w->d_cu_tokens, w->tokens, w->batch, w->table_width};
  return ICX_OK;
}

// Position of packed row i, or -1; *seq receives its sequence.
__device__ __forceinline__ int token_position(const KvTokens& w, int64_t i, int* seq) {
  const int b = kv_sequence(w, i);
  *seq = b;
  if (b < 0) return -1;
  const int64_t end = w.cu ? (int64_t)w.cu[b + 1] : i + 1;
  const int64_t p = (int64_t)w.lens[b] - end + i;
  return p < 0 ? -1 : (int)p;   // lens is s32 and end > i, so p fits
}

// ------------------------------------------------------------- quantising
__device__ __forceinline__ uint32_t bf16_down(float x) {   // finite x
  const uint32_t u = __float_as_uint(x);
  uint32_t h = u >> 16;
  if ((u & 0xffffu) && (u >> 31)) ++h;   // truncation moved a negative value up
  return h == 0xff80u ? 0xff7fu : h;     // not below the lowest finite bf16
}
__device__ __forceinline__ uint32_t bf16_up(float x) {     // finite x >= 0
  const uint32_t u = __float_as_uint(x);
  return (u >> 16) + ((u & 0xffffu) ? 1u : 0u);
}

// Low end and scale of a group's range [mn, mx] (finite).  The quotient
// (mx - lo) / L is bounded from above in 64 bits, rounded up to bf16, and the
// bf16 below is taken instead if it is already enough: no division, and the
// result is the exact quotient rounded up.
template <int BITS>
__device__ __forceinline__ uint32_t group_params(float mn, float mx) {
  constexpr int L = (1 << BITS) - 1;
  const uint32_t lo = bf16_down(mn);
  // (not negative: a maximum below the lowest finite bf16 gives s = 0)
  const double range = fmax((double)mx - (double)__uint_as_float(lo << 16), 0.0);
  uint32_t s = bf16_up(__double2float_ru(range * ((1.0 + 1e-15) / L)));
  if (s > 0) {
    const double below = (double)__uint_as_float((s - 1) << 16);
    if (range <= below * L) --s;
  }
  return s | (lo << 16);
}

// rte((x - lo) / s) clamped to [0, L]: rounded from an f32 quotient (off by
// less than 1e-4 of a step), and where that is within 2e-4 of a half, decided
// by comparing x with the midpoint in 64 bits ((k + 1/2) * s is exact).
// Scales whose reciprocal or range may not be finite take the 64-bit quotient.
template <int BITS>
__device__ __forceinline__ uint32_t group_code(float x, float lo, float s, float inv) {
  constexpr float L = (float)((1 << BITS) - 1);
  if (s < 1e-36f || s > 1e36f)
    return (uint32_t)fmin(fmax(rint(((double)x - (double)lo) / (double)s), 0.0), (double)L);
  const float u = fminf(fmaxf((x - lo) * inv, 0.0f), L);
  float c = rintf(u);
  if (fabsf(u - c) > 0.4998f) {
    const float k = floorf(u);
    const double d = ((double)x - (double)lo) - (double)k * (double)s - 0.5 * (double)s;
    c = d > 0.0 ? k + 1.0f : d < 0.0 ? k : 2.0f * rintf(0.5f * k + 0.25f);
    c = fminf(c, L);
  }
  return (uint32_t)c;
}

// One 64-dimension block: four dimensions per lane of the half warp.  The
// shuffles stay inside the half warp; all 32 lanes take part.
template <int BITS, int D>
__device__ __forceinline__ void store_block(uint8_t* row, int token, int which, int block, int l,
                                            const uint32_t (&c)[4], bool valid) {
  constexpr int ROW = D * BITS / 8;
  const int j = l >> 2, t = l & 3;   // 16-dimension step within the block, quarter of it
  auto put = [&](int at, uint32_t w) { *reinterpret_cast<uint32_t*>(row + at) = w; };
  if (which == 0) {
    if (BITS == 4) {
      uint32_t w = (c[0] | (c[1] << 16) | (c[2] << 8) | (c[3] << 24)) << (4 * (j & 1));
      w |= __shfl_xor_sync(0xffffffffu, w, 4);
      if (valid && !(j & 1)) put(k_word_at<ROW>(token, t, block * 2 + (j >> 1)), w);
    } else {
      const uint32_t w = c[0] | (c[1] << 16) | (c[2] << 8) | (c[3] << 24);
      if (valid) put(k_word_at<ROW>(token, t, block * 4 + j), w);
    }
  } else {
    // this lane: chunks 2t and 2t+1, codes 2j and 2j+1 of the block
    if (BITS == 4) {
      uint32_t a = (c[0] | (c[1] << 4)) << (8 * j), b = (c[2] | (c[3] << 4)) << (8 * j);
      a |= __shfl_xor_sync(0xffffffffu, a, 4);
      b |= __shfl_xor_sync(0xffffffffu, b, 4);
      a |= __shfl_xor_sync(0xffffffffu, a, 8);
      b |= __shfl_xor_sync(0xffffffffu, b, 8);
      if (valid && j < 2) put(v_word_at<ROW>(token, 2 * t + j, block), j ? b : a);
    } else {
      uint32_t a = (c[0] | (c[1] << 8)) << (16 * (j & 1)), b = (c[2] | (c[3] << 8)) << (16 * (j & 1));
      a |= __shfl_xor_sync(0xffffffffu, a, 4);
      b |= __shfl_xor_sync(0xffffffffu, b, 4);
      if (valid) put(v_word_at<ROW>(token, 2 * t + (j & 1), block * 2 + (j >> 1)), (j & 1) ? b : a);
    }
  }
}

template <int BITS, int D>
__device__ __forceinline__ void load_block(const uint8_t* row, int token, int which, int block, int l,
                                           uint32_t (&c)[4]) {
  constexpr int ROW = D * BITS / 8;
  const int j = l >> 2, t = l & 3;
  constexpr uint32_t mask = (1u << BITS) - 1;
  auto get = [&](int at) { return *reinterpret_cast<const uint32_t*>(row + at); };
  if (which == 0) {
    const uint32_t w = BITS == 4 ? get(k_word_at<ROW>(token, t, block * 2 + (j >> 1))) >> (4 * (j & 1))
                                 : get(k_word_at<ROW>(token, t, block * 4 + j));
    c[0] = w & mask;
    c[1] = (w >> 16) & mask;
    c[2] = (w >> 8) & mask;
    c[3] = (w >> 24) & mask;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w = BITS == 4 ? get(v_word_at<ROW>(token, 2 * t + h, block)) >> (8 * j)
                                   : get(v_word_at<ROW>(token, 2 * t + h, block * 2 + (j >> 1))) >> (16 * (j & 1));
      c[2 * h] = w & mask;
      c[2 * h + 1] = (w >> BITS) & mask;
    }
  }
}

struct KvSource {
  const void* x[2];
  int64_t token_stride[2], head_stride[2];
  void* values[2];   // nullable
  int vec[2];        // four elements can be read in one access
};

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvView c, const KvTokens w, const KvSource src) {
  pdl_wait();
  pdl_trigger();
  constexpr int blocks = D / 64;
  const int64_t items = w.tokens * c.heads * blocks * 2;
  const int l = threadIdx.x & 15;
  const int64_t step = (int64_t)gridDim.x * 16;
  // both halves of a warp run the same number of rounds: shuffles use all lanes
  for (int64_t base = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 5) * 2; base < items; base += step) {
    const int64_t it = base + ((threadIdx.x >> 4) & 1);
    bool valid = it < items;
    const int64_t i = valid ? it : 0;
    const int block = (int)(i % blocks);
    const int which = (int)((i / blocks) & 1);
    const int head = (int)((i / (2 * blocks)) % c.heads);
    const int64_t token = i / ((int64_t)2 * blocks * c.heads);
    int b;
    const int pos = token_position(w, token, &b);
    valid = valid && pos >= 0;
    int64_t page = -1;
    if (valid) {
      page = kv_page(c, w, b, pos);
      if (page < 0) {
        valid = false;
        record_status(ICX_DEVICE_BAD_PAGE);
      }
    }
    const int d = block * 64 + 4 * l;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (valid)
      load_f32<T, 4>(static_cast<const T*>(src.x[which]) + token * src.token_stride[which] +
                         head * src.head_stride[which] + d,
                     x, src.vec[which]);
    float mn = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
    float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    uint32_t peak = 0;   // |x| by its bits: NaN and infinity are at the top
#pragma unroll
    for (int k = 0; k < 4; ++k) peak = max(peak, __float_as_uint(fabsf(x[k])));
    for (int o = 1; o < c.group / 4; o <<= 1) {
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    }
    const bool finite = peak < 0x7f800000u;
    const uint32_t p = finite ? group_params<BITS>(mn, mx) : 0x7fc07fc0u;
    const float s = param_scale(p), lo = param_low(p);
    uint32_t code[4] = {0, 0, 0, 0};
    if (finite && s > 0.0f) {
      const float inv = __frcp_rn(s);
#pragma unroll
      for (int k = 0; k < 4; ++k) code[k] = group_code<BITS>(x[k], lo, s, inv);
    }
    const int64_t row = valid ? kv_row(c, page, head, pos) : 0;
    store_block<BITS, D>(c.codes[which] + row * (D * BITS / 8), pos, which, block, l, code, valid);
    if (valid && 4 * l % c.group == 0)
      c.params[which][row * (D / c.group) + d / c.group] = p;
    if (valid && src.values[which]) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = fmaf((float)code[k], s, lo);
      store_f32<T, 4>(static_cast<T*>(src.values[which]) + (token * c.heads + head) * D + d, v);
    }
  }
}

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvView c, const KvTokens w, T* k_out, T* v_out) {
  pdl_wait();
  pdl_trigger();
  constexpr int blocks = D / 64;
  const int64_t items = w.tokens * c.heads * blocks * 2;
  const int l = threadIdx.x & 15;
  for (int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); i < items; i += (int64_t)gridDim.x * 16) {
    const int block = (int)(i % blocks);
    const int which = (int)((i / blocks) & 1);
    T* out = which ? v_out : k_out;
    if (!out) continue;
    const int head = (int)((i / (2 * blocks)) % c.heads);
    const int64_t token = i / ((int64_t)2 * blocks * c.heads);
    int b;
    const int pos = token_position(w, token, &b);
    if (pos < 0) continue;
    const int64_t page = kv_page(c, w, b, pos);
    if (page < 0) {
      record_status(ICX_DEVICE_BAD_PAGE);
      continue;
    }
    const int64_t row = kv_row(c, page, head, pos);
    const int d = block * 64 + 4 * l;
    const uint32_t p = c.params[which][row * (D / c.group) + d / c.group];
    uint32_t code[4];
    load_block<BITS, D>(c.codes[which] + row * (D * BITS / 8), pos, which, block, l, code);
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = fmaf((float)code[k], param_scale(p), param_low(p));
    store_f32<T, 4>(out + (token * c.heads + head) * D + d, v);
  }
}

#define ICX_KV_DISPATCH(kernel)                                                                        \
  (c.bits == 4 ? (c.dim == 64 ? kernel<T, 4, 64> : c.dim == 128 ? kernel<T, 4, 128> : kernel<T, 4, 256>) \
               : (c.dim == 64 ? kernel<T, 8, 64> : c.dim == 128 ? kernel<T, 8, 128> : kernel<T, 8, 256>))

static unsigned item_grid(int64_t items) {
  const int64_t blocks = (items + 15) / 16;
  return (unsigned)(blocks < 148 * 32 ? blocks : 148 * 32);
}

}  // namespace icx

using namespace icx;

extern "C" int icx_kv_cache_append(void* stream, const icx_kv_cache* cache, const icx_kv_tokens* where,
                                   const void* d_k, const void* d_v, int type, int64_t k_token_stride,
                                   int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                   void* d_k_values, void* d_v_values) {
  KvView c;
  KvTokens w;
  const int rc = kv_views("KvCacheAppend", cache, where, &c, &w);
  if (rc) return rc;
  ICX_REQUIRE(is_float_type(type), "KvCacheAppend: k and v must be Float32, Float16 or BFloat16");
  ICX_REQUIRE(k_token_stride >= 0 && k_head_stride >= 0 && v_token_stride >= 0 && v_head_stride >= 0,
              "KvCacheAppend: negative stride");
  if (w.tokens == 0 || w.batch == 0) return ICX_OK;
  ICX_REQUIRE(d_k && d_v, "KvCacheAppend: null operand");
  const size_t e = float_bytes(type);
  auto vec = [&](const void* p, int64_t ts, int64_t hs) {
    return (int)((reinterpret_cast<uintptr_t>(p) | (size_t)ts * e | (size_t)hs * e) % (4 * e) == 0);
  };
  ICX_REQUIRE(((reinterpret_cast<uintptr_t>(d_k_values) | reinterpret_cast<uintptr_t>(d_v_values)) & 15) == 0,
              "KvCacheAppend: value buffers must be 16-byte aligned");
  KvSource src{{d_k, d_v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride},
               {d_k_values, d_v_values},
               {vec(d_k, k_token_stride, k_head_stride), vec(d_v, v_token_stride, v_head_stride)}};
  const dim3 grid(item_grid(w.tokens * c.heads * (c.dim / 64) * 2));
  cudaStream_t s = as_stream(stream);
  ICX_FLOAT_DISPATCH(type,
                     ICX_CUDA(launch_pdl(ICX_KV_DISPATCH(kv_append_kernel), grid, dim3(256), 0, s, c, w, src)));
  return ICX_OK;
}

extern "C" int icx_kv_cache_read(void* stream, const icx_kv_cache* cache, const icx_kv_tokens* where, int type,
                                 void* d_k, void* d_v) {
  KvView c;
  KvTokens w;
  const int rc = kv_views("KvCacheRead", cache, where, &c, &w);
  if (rc) return rc;
  ICX_REQUIRE(is_float_type(type), "KvCacheRead: output must be Float32, Float16 or BFloat16");
  ICX_REQUIRE(((reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v)) & 15) == 0,
              "KvCacheRead: output buffers must be 16-byte aligned");
  if (w.tokens == 0 || w.batch == 0) return ICX_OK;
  const dim3 grid(item_grid(w.tokens * c.heads * (c.dim / 64) * 2));
  cudaStream_t s = as_stream(stream);
  ICX_FLOAT_DISPATCH(type, ICX_CUDA(launch_pdl(ICX_KV_DISPATCH(kv_read_kernel), grid, dim3(256), 0, s, c, w,
                                               static_cast<T*>(d_k), static_cast<T*>(d_v))));
  return ICX_OK;
}
