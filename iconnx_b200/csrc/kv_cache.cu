// Quantised K/V cache: append (quantise) and read (dequantise).
//
// HBM sets the floor: 7 f16 prompts of up to 3,000 tokens into 8 bits, 8 heads of
// 128, 57 us (2.4 TB/s; floor 21; f32 58, floor 38); 6 sequences of up to 8,100 read
// from 4 bits to bf16 or f16, 40 us (4.0 TB/s; floor 25), to f32 60 (floor 44); a
// decode step's append or read 2.6 to 2.8.  What lies between: about 350 (append)
// and 107 (read) instructions per 256 values, of which one issues in 63% and 64% of
// the cycles (integer pipe 53% and 62%), while three warps wait for memory per
// instruction: lookups, then one token's values (append) or four tokens' codes
// (read) in flight.  Nothing is full.
// Eight lanes take 64 dimensions of one (token, head) of K or V,
// eight consecutive ones (one or two 16-byte accesses) per lane, so a
// quantisation group is 4 or 8 lanes and every code word of the layout is put
// together from lanes of one such eighth.
#include "kv_cache.cuh"

#include <type_traits>

#include "capi.cuh"
#include "common.cuh"
#include "tmap.cuh"

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
  // kernels look up to 1024 positions ahead of the last in 32 bits
  ICX_REQUIRE((int64_t)w->table_width << shift <= (1ll << 31) - 4096,
              "%s: page table row beyond 2^31 - 4096 positions", what);
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
                 c->pages, shift, c->kv_heads, c->head_dim, c->bits, c->group, c->group == 32 ? 5 : 6};
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

// Low end and scale of a group's range [mn, mx] (finite).  t bounds the
// quotient (mx - lo) / L from above and is rounded up to bf16; the bf16 below
// is taken instead if it is already enough: below * L is exact, and with the
// difference rounded up, "difference <= below * L" decides exactly (an f32 is
// not below the exact difference if and only if it is not below that
// difference rounded up).  Ranges that may pass f32 are taken at a sixteenth.
template <int BITS>
__device__ __forceinline__ uint32_t group_params(float mn, float mx) {
  constexpr int L = (1 << BITS) - 1;
  const bool wide = fmaxf(fabsf(mn), fabsf(mx)) > 1e38f;
  const float z = wide ? 0.0625f : 1.0f;
  const uint32_t lo = bf16_down(mn);
  // (not negative: a maximum below the lowest finite bf16 gives s = 0)
  const float range = fmaxf(__fsub_ru(mx * z, __uint_as_float(lo << 16) * z), 0.0f);
  uint32_t s = bf16_up(__fmul_ru(range, (float)((1.0 + 1e-6) / L)));
  if (s > 0 && range <= __uint_as_float((s - 1) << 16) * (float)L) --s;
  if (wide && s > 0) s += 4 << 7;   // times 16
  return s | (lo << 16);
}

// rte((x - lo) / s) clamped to [0, L].  An f32 quotient is off by less than 7e-5
// (roundings of 2^-24, 2^-23 and 2^-24 at most at 255); where it is within 2e-4
// of a half, x is compared with the midpoint lo + m, m = (k + 1/2) s, in f32
// alone: m is exact (9 + 8 bits), t + e = lo + m exactly, and x - t is exact
// where x and t are within a factor of two, while otherwise t is all but
// cancelled, so that e = 0 and the sign of x - t is what counts.
__device__ __forceinline__ float code_near_half(float x, float lo, float s, float u) {
  const float k = floorf(u), m = (k + 0.5f) * s;
  const float t = __fadd_rn(lo, m), b = __fsub_rn(t, lo);
  const float e = __fadd_rn(__fsub_rn(lo, __fsub_rn(t, b)), __fsub_rn(m, b));
  const float d = __fsub_rn(x, t);
  return d > e ? k + 1.0f : d < e ? k : 2.0f * rintf(0.5f * k + 0.25f);
}

// The codes, each on the bits of kRound (the code in the low byte).  x is used
// up.  Where the reciprocal of the scale or the range might not be finite (or
// normal), all are scaled by a power of two first: |lo| is below 2^33 s, so
// that nothing overflows.
constexpr float kRound = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer (half to even)

template <int BITS>
__device__ __forceinline__ void group_codes(float (&x)[8], float lo, float s, bool finite, uint32_t (&code)[8]) {
  if (!(finite && s > 0.0f)) {
#pragma unroll
    for (int k = 0; k < 8; ++k) code[k] = __float_as_uint(kRound);
    return;
  }
  if (s < 1e-36f || s > 1e36f) {
    const float z = s < 1.0f ? 1.2676506e30f : 0.0625f;   // 2^100, 2^-4
    s *= z;
    lo *= z;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] *= z;
  }
  // lo <= x <= lo + L s, so that the quotient needs no clamp, unless lo itself
  // was clamped to the lowest finite bf16
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = fmaxf(x[k], lo);
  float inv, worst = 0.0f;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float u = (x[k] - lo) * inv, r = __fadd_rn(u, kRound);
    worst = fmaxf(worst, fabsf(u - __fsub_rn(r, kRound)));
    code[k] = __float_as_uint(r);
  }
  // One at a time, by its index: in 16-bit types such values are exact ties
  // more often than not, one in a few hundred.
  uint32_t near = 0;
  if (worst > 0.4998f) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      near |= fabsf((x[k] - lo) * inv - (__uint_as_float(code[k]) - kRound)) > 0.4998f ? 1u << k : 0u;
  }
  while (near) {
    const int at = __ffs(near) - 1;
    near &= near - 1;
    float xv = x[0];
#pragma unroll
    for (int k = 1; k < 8; ++k) xv = at == k ? x[k] : xv;
    const uint32_t n =
        __float_as_uint(fminf(code_near_half(xv, lo, s, (xv - lo) * inv), (float)((1 << BITS) - 1)) + kRound);
#pragma unroll
    for (int k = 0; k < 8; ++k) code[k] = at == k ? n : code[k];
  }
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// One block of 64 dimensions: eight lanes (l = 0..7) of eight consecutive
// dimensions.  Lane l holds step / row tile j = l / 2 of the block, quarters
// 2 (l & 1) and 2 (l & 1) + 1 of it (K), or g = 4 (l & 1) .. + 3 (V).  The shuffles stay inside the eight lanes; all 32 lanes take part.
template <int BITS, int D>
__device__ __forceinline__ void store_block(uint8_t* row, int token, int which, int block, int l,
                                            const uint32_t (&c)[8], bool valid) {
  constexpr int ROW = D * BITS / 8;
  const int j = l >> 1, odd = l & 1;
  auto put = [&](int at, uint32_t w) {
    if (valid) *reinterpret_cast<uint32_t*>(row + at) = w;
  };
  if (which == 0) {
    uint32_t a = low_bytes(c[0], c[2], c[1], c[3]), b = low_bytes(c[4], c[6], c[5], c[7]);
    if (BITS == 4) {
      // words of both quarters need steps 2n and 2n+1, which are lanes l and l ^ 2
      a <<= 4 * (j & 1);
      b <<= 4 * (j & 1);
      const uint32_t other = __shfl_xor_sync(0xffffffffu, (j & 1) ? a : b, 2);
      put(k_word_at<ROW>(token, 2 * odd + (j & 1), block * 2 + (j >> 1)), ((j & 1) ? b : a) | other);
    } else {
      put(k_word_at<ROW>(token, 2 * odd, block * 4 + j), a);
      put(k_word_at<ROW>(token, 2 * odd + 1, block * 4 + j), b);
    }
  } else if (BITS == 4) {
    // byte i: g = 4 odd + i, tile j; lanes j and j ^ 1 hold the two tiles of a
    // piece and exchange so that each stores the half words of two g
    const uint32_t u = low_bytes(c[0], c[2], c[4], c[6]) | (low_bytes(c[1], c[3], c[5], c[7]) << 4);
    const uint32_t v = __shfl_xor_sync(0xffffffffu, u, 2);
    put(((block * 2 + (j >> 1)) ^ v_swizzle<ROW>(token)) * 16 + 8 * odd + 4 * (j & 1),
        (j & 1) ? __byte_perm(v, u, 0x7362) : __byte_perm(u, v, 0x5140));
  } else if (valid) {
    *reinterpret_cast<uint2*>(row + ((block * 4 + j) ^ v_swizzle<ROW>(token)) * 16 + 8 * odd) =
        make_uint2(low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7]));
  }
}

// The inverse: the codes of this lane's eight dimensions.  Split in two, so
// that several blocks' loads can be in flight.
template <int BITS, int D>
__device__ __forceinline__ void load_block_words(const uint8_t* row, int token, int which, int block, int l,
                                                 uint32_t (&w)[2]) {
  constexpr int ROW = D * BITS / 8;
  const int j = l >> 1, odd = l & 1;
  auto get = [&](int at) { return *reinterpret_cast<const uint32_t*>(row + at); };
  if (which == 0) {
    const int n = BITS == 4 ? block * 2 + (j >> 1) : block * 4 + j;
    w[0] = get(k_word_at<ROW>(token, 2 * odd, n));
    w[1] = get(k_word_at<ROW>(token, 2 * odd + 1, n));
  } else if (BITS == 4) {
    w[0] = get(((block * 2 + (j >> 1)) ^ v_swizzle<ROW>(token)) * 16 + 8 * odd + 4 * (j & 1));
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(row + ((block * 4 + j) ^ v_swizzle<ROW>(token)) * 16 + 8 * odd);
    w[0] = u.x;
    w[1] = u.y;
  }
}
// Eight codes, each on the bits of 2^23 (2^23 + code as an f32).
constexpr uint32_t kCodeOne = 0x4b000000u;

__device__ __forceinline__ uint32_t code_at(uint32_t bytes, int i) {   // byte i of a word
  return __byte_perm(bytes, kCodeOne, 0x7440 + i);
}

template <int BITS>
__device__ __forceinline__ void block_codes(int which, int l, const uint32_t (&w)[2], uint32_t (&c)[8]) {
  const int j = l >> 1;
  if (which == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t u = BITS == 4 ? (w[h] >> (4 * (j & 1))) & 0x0f0f0f0fu : w[h];
      c[4 * h] = code_at(u, 0);
      c[4 * h + 1] = code_at(u, 2);
      c[4 * h + 2] = code_at(u, 1);
      c[4 * h + 3] = code_at(u, 3);
    }
  } else if (BITS == 4) {
    const uint32_t v = __shfl_xor_sync(0xffffffffu, w[0], 2);
    const uint32_t u = (j & 1) ? __byte_perm(v, w[0], 0x7531) : __byte_perm(w[0], v, 0x6420);
    const uint32_t even = u & 0x0f0f0f0fu, odd = (u >> 4) & 0x0f0f0f0fu;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[2 * i] = code_at(even, i);
      c[2 * i + 1] = code_at(odd, i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = code_at(w[0], i);
      c[4 + i] = code_at(w[1], i);
    }
  }
}

// Minimum and maximum that a NaN passes through.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct KvSource {
  const void* x[2];
  int64_t token_stride[2], head_stride[2];
  void* values[2];   // nullable
  int vec[2];        // eight elements can be read in 16-byte accesses
};

// A warp takes K or V of `run` consecutive tokens (at most 32): `per` blocks of
// 64 dimensions of their heads, four at a time, several fours in flight.  Lane
// i looks up the sequence and page of token i, all at once, since each lookup
// is a chain of dependent loads.
struct WarpPart {
  int64_t token0, row0;   // row0: this lane's token's cache row of head 0
  int tokens, which, from, to;
  int pos;                // this lane's token's position, or -1: nothing to do
};

struct Parts {
  int run, parts, per;
  unsigned items;
};

__device__ __forceinline__ WarpPart warp_part(const KvView& c, const KvTokens& w, const Parts& n, unsigned item,
                                              int blocks) {
  WarpPart p;
  const int lane = threadIdx.x & 31;
  const unsigned side = item / (unsigned)n.parts;
  const int part = (int)(item - side * (unsigned)n.parts);
  p.which = (int)(side & 1);
  p.token0 = (int64_t)(side >> 1) * n.run;
  p.tokens = (int)min((int64_t)n.run, w.tokens - p.token0);
  p.from = part * n.per;
  p.to = min(p.from + n.per, blocks);
  p.pos = -1;
  p.row0 = 0;
  if (lane < p.tokens) {
    int b;
    p.pos = token_position(w, p.token0 + lane, &b);
    if (p.pos >= 0) {
      const int64_t page = kv_page(c, w, b, p.pos);
      if (page < 0) {
        p.pos = -1;
        record_bad_page();
      } else {
        p.row0 = kv_row(c, page, 0, p.pos);
      }
    }
  }
  return p;
}

// Eight values, and the smallest and largest of them (NaN if one is).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8], bool vec, float& mn, float& mx) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    Vec<T, 8> v;
    if (vec) {
      v = *reinterpret_cast<const Vec<T, 8>*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v.v[i] = p[i];
    }
    const T2* w = reinterpret_cast<const T2*>(&v);
    const T2 lo = __hmin2_nan(__hmin2_nan(w[0], w[1]), __hmin2_nan(w[2], w[3]));
    const T2 hi = __hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3]));
    mn = min_nan(to_f32(lo.x), to_f32(lo.y));
    mx = max_nan(to_f32(hi.x), to_f32(hi.y));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(v.v[i]);
  } else {
    load_f32<T, 4>(p, *reinterpret_cast<float(*)[4]>(&x[0]), vec);
    load_f32<T, 4>(p + 4, *reinterpret_cast<float(*)[4]>(&x[4]), vec);
    mn = mx = x[0];
#pragma unroll
    for (int k = 1; k < 8; ++k) {
      mn = min_nan(mn, x[k]);
      mx = max_nan(mx, x[k]);
    }
  }
}

// Over the four or eight lanes of a group.  16-bit types: both ends in one
// word, the larger negated, so that one minimum serves both.
template <typename T>
__device__ __forceinline__ void group_range(float& mn, float& mx, bool eight) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 v;
    v.x = from_f32<T>(mn);   // exact: values of the type
    v.y = from_f32<T>(-mx);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      if (o == 4 && !eight) break;
      uint32_t u = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<uint32_t*>(&v), o);
      v = __hmin2_nan(v, *reinterpret_cast<T2*>(&u));
    }
    mn = to_f32(v.x);
    mx = -to_f32(v.y);
  } else {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      if (o == 4 && !eight) break;
      mn = min_nan(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if (sizeof(T) == 2) {
    store_f32<T, 8>(p, x);
  } else {
    store_f32<T, 4>(p, *reinterpret_cast<const float(*)[4]>(&x[0]));
    store_f32<T, 4>(p + 4, *reinterpret_cast<const float(*)[4]>(&x[4]));
  }
}

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(128, 8)
    kv_append_kernel(const __grid_constant__ KvView c, const __grid_constant__ KvTokens w,
                     const __grid_constant__ KvSource src, const Parts n) {
  pdl_wait();
  pdl_trigger();
  constexpr int kPerHead = D / 64, ROW = D * BITS / 8;
  const unsigned item = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= n.items) return;
  const WarpPart p = warp_part(c, w, n, item, c.heads * kPerHead);
  const int l = threadIdx.x & 7, sub = (threadIdx.x >> 3) & 3;
  const bool vec = src.vec[p.which] != 0, store_group = (8 * l & (c.group - 1)) == 0;
  const int64_t x_step = src.token_stride[p.which], v_step = (int64_t)c.heads * D;
  for (int b0 = p.from; b0 < p.to; b0 += 4) {
    // this lane's place in every token
    const int b = min(b0 + sub, p.to - 1), head = b / kPerHead, block = b % kPerHead, d = block * 64 + 8 * l;
    const bool valid = b0 + sub < p.to;
    const T* x_at = static_cast<const T*>(src.x[p.which]) + p.token0 * x_step + head * src.head_stride[p.which] + d;
    T* v_at = static_cast<T*>(src.values[p.which]);
    const bool values = valid && v_at != nullptr;
    v_at += (p.token0 * c.heads + head) * D + d;
    const int64_t head_row = (int64_t)head << c.page_shift;
    uint8_t* codes = c.codes[p.which] + head_row * ROW;
    uint32_t* params = c.params[p.which] + (head_row * D + d >> c.group_shift);
    for (int i = 0; i < p.tokens; ++i, x_at += x_step, v_at += v_step) {
      const int pos = __shfl_sync(0xffffffffu, p.pos, i);
      const int64_t row0 = __shfl_sync(0xffffffffu, p.row0, i);
      if (pos < 0) continue;
      float x[8], mn, mx;
      load8<T>(x_at, x, vec, mn, mx);
      group_range<T>(mn, mx, c.group == 64);
      const bool finite = fabsf(mn) < INFINITY && fabsf(mx) < INFINITY;
      const uint32_t prm = finite ? group_params<BITS>(mn, mx) : 0x7fc07fc0u;
      const float s = param_scale(prm), lo = param_low(prm);
      uint32_t code[8];
      group_codes<BITS>(x, lo, s, finite, code);
      store_block<BITS, D>(codes + row0 * ROW, pos, p.which, block, l, code, valid);
      if (valid && store_group) params[row0 * D >> c.group_shift] = prm;
      if (values) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = fmaf(__uint_as_float(code[k]) - kRound, s, lo);
        store8<T>(v_at, x);
      }
    }
  }
}

template <typename T, int BITS, int D>
__global__ void __launch_bounds__(128, 8)
    kv_read_kernel(const __grid_constant__ KvView c, const __grid_constant__ KvTokens w, T* k_out, T* v_out,
                   const Parts n) {
  pdl_wait();
  pdl_trigger();
  constexpr int kPerHead = D / 64, ROW = D * BITS / 8, U = 4;   // tokens in flight
  const unsigned item = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= n.items) return;
  const WarpPart p = warp_part(c, w, n, item, c.heads * kPerHead);
  T* out = p.which ? v_out : k_out;
  if (!out) return;
  const int l = threadIdx.x & 7, sub = (threadIdx.x >> 3) & 3;
  const int64_t step = (int64_t)c.heads * D;
  for (int b0 = p.from; b0 < p.to; b0 += 4) {
    const int b = min(b0 + sub, p.to - 1), head = b / kPerHead, block = b % kPerHead, d = block * 64 + 8 * l;
    const bool valid = b0 + sub < p.to;
    const int64_t head_row = (int64_t)head << c.page_shift;
    const uint8_t* codes = c.codes[p.which] + head_row * ROW;
    const uint32_t* params = c.params[p.which] + (head_row * D + d >> c.group_shift);
    T* out_at = out + (p.token0 * c.heads + head) * D + d;
    for (int i0 = 0; i0 < p.tokens; i0 += U, out_at += U * step) {
      uint32_t words[U][2], prm[U];
      int pos[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        pos[i] = i0 + i < p.tokens ? __shfl_sync(0xffffffffu, p.pos, i0 + i) : -1;
        const int64_t row0 = __shfl_sync(0xffffffffu, p.row0, (i0 + i) & 31);
        if (pos[i] < 0) continue;
        load_block_words<BITS, D>(codes + row0 * ROW, pos[i], p.which, block, l, words[i]);
        prm[i] = params[row0 * D >> c.group_shift];
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (pos[i] < 0) continue;
        uint32_t code[8];
        block_codes<BITS>(p.which, l, words[i], code);
        const float s = param_scale(prm[i]), lo = param_low(prm[i]);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = fmaf(__uint_as_float(code[k]) - 8388608.0f, s, lo);
        if (valid) store8<T>(out_at + i * step, v);
      }
    }
  }
}

// Enough warps to fill the GPU: with few tokens their heads are divided (down
// to four blocks per warp), with many a warp takes up to eight tokens.
static Parts make_parts(const KvView& c, const KvTokens& w) {
  const int blocks = c.heads * (c.dim / 64), fours = (blocks + 3) / 4;
  const int64_t warps = (int64_t)sm_count() * 32;
  Parts n{1, 1, 0, 0};
  while (n.parts < fours && w.tokens * 2 * n.parts < warps) ++n.parts;
  n.per = (fours + n.parts - 1) / n.parts * 4;
  n.parts = (blocks + n.per - 1) / n.per;
  if (n.parts == 1)
    while (n.run < 8 && w.tokens * 2 / (n.run * 2) >= warps) n.run *= 2;
  n.items = (unsigned)((w.tokens + n.run - 1) / n.run * 2 * n.parts);   // tokens < 2^31, and parts > 1 for few
  return n;
}

#define ICX_KV_DISPATCH(kernel)                                                                        \
  (c.bits == 4 ? (c.dim == 64 ? kernel<T, 4, 64> : c.dim == 128 ? kernel<T, 4, 128> : kernel<T, 4, 256>) \
               : (c.dim == 64 ? kernel<T, 8, 64> : c.dim == 128 ? kernel<T, 8, 128> : kernel<T, 8, 256>))

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
    return (int)((reinterpret_cast<uintptr_t>(p) | (size_t)ts * e | (size_t)hs * e) % 16 == 0);
  };
  ICX_REQUIRE(((reinterpret_cast<uintptr_t>(d_k_values) | reinterpret_cast<uintptr_t>(d_v_values)) & 15) == 0,
              "KvCacheAppend: value buffers must be 16-byte aligned");
  KvSource src{{d_k, d_v}, {k_token_stride, v_token_stride}, {k_head_stride, v_head_stride},
               {d_k_values, d_v_values},
               {vec(d_k, k_token_stride, k_head_stride), vec(d_v, v_token_stride, v_head_stride)}};
  const Parts n = make_parts(c, w);
  const dim3 grid((unsigned)((n.items + 3) / 4));
  cudaStream_t s = as_stream(stream);
  ICX_FLOAT_DISPATCH(type,
                     ICX_CUDA(launch_pdl(ICX_KV_DISPATCH(kv_append_kernel), grid, dim3(128), 0, s, c, w, src, n)));
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
  const Parts n = make_parts(c, w);
  const dim3 grid((unsigned)((n.items + 3) / 4));
  cudaStream_t s = as_stream(stream);
  ICX_FLOAT_DISPATCH(type, ICX_CUDA(launch_pdl(ICX_KV_DISPATCH(kv_read_kernel), grid, dim3(128), 0, s, c, w,
                                               static_cast<T*>(d_k), static_cast<T*>(d_v), n)));
  return ICX_OK;
}
