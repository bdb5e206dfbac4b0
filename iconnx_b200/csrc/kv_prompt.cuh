// Pieces shared by the two kernels for prompt chunks over the quantised K/V
// cache: the spread of codes over 16-byte pieces, matrix instructions of
// kind::f16, and the row tiles.
#pragma once

#include "capi.cuh"
#include "common.cuh"
#include "kv_attention.cuh"

namespace icx {

constexpr int kPrRows = 128, kPrKeys = 64, kPrGroup = 64, kPrThreads = 256;

// kind::f16, f32 accumulator, M = 128: [4,6) D format 1, A and B f16 (0), [16]
// B MN-major, [17,23) N >> 3, [24,29) M >> 4.
constexpr uint32_t prompt_idesc(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kPrRows >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// The eight f16 of a 16-byte piece come from one 4-bit word or two 8-bit ones.
// K: piece 2 t + n of a group's 64 dimensions, r-th value: dimension
// 16 step + 4 t + i of the group.
template <int BITS>
__host__ __device__ constexpr int k_step(int n, int r) {
  return BITS == 4 ? 2 * n + ((r >> 1) & 1) : 2 * n + (r >> 2);
}
template <int BITS>
__host__ __device__ constexpr int k_dim(int r) {
  return BITS == 4 ? (r & 1) + 2 * (r >> 2) : ((r >> 1) & 1) * 2 + (r & 1);
}
// V: a group's pieces 4 n .. 4 n + 3 are its dimensions 32 n .. 32 n + 31; the
// r-th value of the j-th of them is dimension 32 n + v_dim(j, r).
template <int BITS>
__host__ __device__ constexpr int v_dim(int j, int r) {
  const int pair = ((r & 1) << 1) | ((r >> 1) & 1);   // {0, 2, 1, 3}
  return BITS == 4 ? 16 * (r >> 2) + 4 * j + pair : 16 * (j >> 1) + 8 * (j & 1) + 4 * (r >> 2) + pair;
}
// 4 bits: these values are sixteen times their code
template <int BITS>
__host__ __device__ constexpr bool times16(int r) {
  return BITS == 4 && ((r >> 1) & 1);
}

template <int BITS>
__device__ __forceinline__ uint4 spread(uint32_t w0, uint32_t w1) {
  if (BITS == 4) return make_uint4(w0 & 0x000f000fu, w0 & 0x00f000f0u, (w0 >> 8) & 0x000f000fu, (w0 >> 8) & 0x00f000f0u);
  return make_uint4(w0 & 0x00ff00ffu, (w0 >> 8) & 0x00ff00ffu, w1 & 0x00ff00ffu, (w1 >> 8) & 0x00ff00ffu);
}

// All lanes poll: the roles hand over several times per tile, and a lane that
// sleeps between polls wakes too late for that.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
}

// The want-th row tile of the batch, the last tiles of a sequence (the longest)
// first; *seq = -1 if there is none.  One warp.
__device__ __forceinline__ void find_row_tile(const KvView& c, const KvTokens& w, int share, int rows, int want,
                                              int* seq_out, int* tile_out) {
  const int lane = threadIdx.x & 31;
  int before = 0, seq = -1, tile = 0;
  for (int b0 = 0; b0 < w.batch && seq < 0; b0 += 32) {
    const int b = b0 + lane;
    const int n = b < w.batch ? seq_units(c, w, share, rows, b).tiles : 0;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + inc > want);
    if (hit) {
      const int l = __ffs(hit) - 1;
      seq = b0 + l;
      tile = __shfl_sync(0xffffffffu, n, l) - 1 - (want - before - __shfl_sync(0xffffffffu, inc - n, l));
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) {
    *seq_out = seq;
    *tile_out = tile;
  }
}

// Half the codes of one position: words of K chunks 2 half, 2 half + 1, and the
// V words of each group's dimensions 32 half .. 32 half + 31.
template <int D, int BITS>
struct RawCodes {
  static constexpr int ROW = D * BITS / 8, KW = D * BITS / 128, VW = BITS, G = D / 64;
  uint32_t k[2][KW], v[G][VW];
  __device__ __forceinline__ void load(const KvView& c, int64_t row, int token, int half) {
    load_k(c, row, token, half);
    load_v(c, row, token, half);
  }
  __device__ __forceinline__ void load_v(const KvView& c, int64_t row, int token, int half) {
    const uint8_t* vr = c.codes[1] + row * ROW;
#pragma unroll
    for (int x = 0; x < G; ++x)
#pragma unroll
      for (int n = 0; n < VW / 4; ++n) {
        const int piece = BITS == 4 ? 2 * x + half : 4 * x + 2 * half + n;
        const uint4 u = *reinterpret_cast<const uint4*>(vr + ((piece ^ v_swizzle<ROW>(token)) << 4));
        v[x][4 * n] = u.x;
        v[x][4 * n + 1] = u.y;
        v[x][4 * n + 2] = u.z;
        v[x][4 * n + 3] = u.w;
      }
  }
  __device__ __forceinline__ void load_k(const KvView& c, int64_t row, int token, int half) {
    const uint8_t* kr = c.codes[0] + row * ROW;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if constexpr (KW < 4) {
        load_words(reinterpret_cast<const uint32_t*>(kr + k_word_at<ROW>(token, 2 * half + x, 0)), k[x]);
      } else {
#pragma unroll
        for (int n = 0; n < KW; n += 4) {
          const uint4 u = *reinterpret_cast<const uint4*>(kr + k_word_at<ROW>(token, 2 * half + x, n));
          k[x][n] = u.x;
          k[x][n + 1] = u.y;
          k[x][n + 2] = u.z;
          k[x][n + 3] = u.w;
        }
      }
    }
  }
};

// A query row as the left operand: scaled by 2^e into f16's range (and by the
// sign of the scale, so that the score's factor is positive), in the order of
// the K pieces.  *f is the factor from products with codes that count 2^-24
// (exact) or with values (24 bits less) to scores in powers of two; sum[k] the
// sum of the scaled row over group k.
template <typename T, int G, int BITS, bool CODES>
__device__ __forceinline__ void put_query(const AttendArgs& a, const T* q, bool mine, int row, uint8_t* s_q, float* f,
                                          float (&sum)[G]) {
  // A group is fetched with eight 16-byte loads at once: with nearly all of the
  // SM's memory shared there is no L1 that would keep a row, and a warp's load
  // touches 32 of them (all of it in 8-byte loads: 265 us instead of 250 where
  // kv_prompt_bf16.cu states 253 now).
  Vec<T, 8> u[kPrGroup / 8];
  const bool wide = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
  auto fetch = [&](int k) {
    if (wide) {
#pragma unroll
      for (int i = 0; i < kPrGroup / 8; ++i) u[i] = *reinterpret_cast<const Vec<T, 8>*>(q + k * kPrGroup + 8 * i);
    } else {
#pragma unroll
      for (int i = 0; i < kPrGroup / 8; ++i)
#pragma unroll
        for (int x = 0; x < 8; ++x) u[i].v[x] = q[k * kPrGroup + 8 * i + x];
    }
  };
  float peak = 0.0f;
#pragma unroll 1
  for (int k = 0; k < G; ++k) {
    fetch(k);
#pragma unroll
    for (int i = 0; i < kPrGroup / 8; ++i)
#pragma unroll
      for (int x = 0; x < 8; ++x) peak = fmaxf(peak, fabsf(to_f32(u[i].v[x])));
  }
  const int e = mine && peak > 0.0f ? max(-60, min(120, 14 - (int)((__float_as_uint(peak) >> 23) & 255) + 127)) : 0;
  const float up = mine && a.scale != 0.0f ? copysignf(__uint_as_float((uint32_t)(e + 127) << 23), a.scale) : 0.0f;
  *f = score_factor(a.scale, CODES ? 16777216.0f : 1.0f, e);
#pragma unroll 1
  for (int k = G - 1; k >= 0; --k) {   // the last group is there
    if (k < G - 1) fetch(k);
    float total = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      // step j's dimensions 16 j + 4 t .. + 3 of the group
      float v[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 16 * j + 4 * t + i;
          v[j][i] = up != 0.0f ? to_f32(u[d >> 3].v[d & 7]) * up : 0.0f;
          total += v[j][i];
        }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = v[k_step<BITS>(n, i)][k_dim<BITS>(i)] * (CODES && times16<BITS>(i) ? 0.0625f : 1.0f);
        const int piece = 2 * t + n;
        *reinterpret_cast<uint4*>(s_q + k * kPrRows * 128 + row * 128 + ((piece ^ (row & 7)) << 4)) =
            make_uint4(pack_f16(x[0], x[1]), pack_f16(x[2], x[3]), pack_f16(x[4], x[5]), pack_f16(x[6], x[7]));
      }
    }
#pragma unroll
    for (int kk = 0; kk < G; ++kk)
      if (kk == k) sum[kk] = total;
  }
}

// A CTA's share of the positions below `see`: whole tiles of `keys`.
struct PromptShare {
  int first, end, tiles;
  __device__ __forceinline__ PromptShare(int see, int keys, int splits) {
    const int all = (see + keys - 1) / keys, t0 = (int)((int64_t)all * blockIdx.z / splits);
    tiles = (int)((int64_t)all * (blockIdx.z + 1) / splits) - t0;
    first = t0 * keys;
    end = min(see, first + tiles * keys);
  }
};

// A row's output, or with several shares its part in the workspace: the values
// over the share's own weights, the reference of its scores and the sum of its
// weights, at [share][token][query head].
template <typename T, int D>
struct PromptOut {
  T* out;
  float* part;
  __device__ __forceinline__ PromptOut(const AttendArgs& a, const KvTokens& w, int splits, int64_t row) {
    out = static_cast<T*>(a.out) + row * D;
    part = splits > 1 ? a.partial + ((int64_t)blockIdx.z * w.tokens * a.q_heads + row) * (D + 2) : nullptr;
  }
  __device__ __forceinline__ void put(int d, const float (&y)[4][8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!part) {
        store_f32<T, 8>(out + d + 8 * j, y[j]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2*>(part + d + 8 * j + e) = make_float2(y[j][e], y[j][e + 1]);
      }
    }
  }
  __device__ __forceinline__ void put_weight(float m, float l) const {
    if (part) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
  }
};

// Joins the shares of a (token, query head), in their order.  One warp each.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    kv_prompt_join_kernel(const __grid_constant__ KvTokens w, const __grid_constant__ AttendArgs a, int splits) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t rows = w.tokens * a.q_heads, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows || kv_sequence(w, row / a.q_heads) < 0) return;
  auto part = [&](int z) { return a.partial + (z * rows + row) * (D + 2); };
  float top = kNoScore, l = 0.0f, o[E] = {};
  for (int z = 0; z < splits; ++z) top = fmaxf(top, part(z)[D]);
  auto weight = [&](int z) {
    const float2 ml = *reinterpret_cast<const float2*>(part(z) + D);
    return ml.y * ex2(ml.x - top);
  };
  for (int z = 0; z < splits; ++z) l += weight(z);
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  for (int z = 0; z < splits; ++z) {
    const float f = weight(z) * inv;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(part(z) + lane * E + e);
      o[e] = fmaf(v.x, f, o[e]);
      o[e + 1] = fmaf(v.y, f, o[e + 1]);
    }
  }
  store_f32<T, E>(static_cast<T*>(a.out) + row * D + lane * E, o);
}

inline dim3 prompt_grid(const KvView& c, const KvTokens& w, const AttendArgs& a, const PromptPlan& p) {
  // at most so many row tiles
  return dim3((unsigned)(w.tokens * (a.q_heads / c.heads) / p.rows + w.batch), (unsigned)c.heads, (unsigned)p.splits);
}
template <typename T, int D>
static int launch_prompt_join(cudaStream_t s, const KvTokens& w, const AttendArgs& a, const PromptPlan& p) {
  if (p.splits == 1) return ICX_OK;
  ICX_CUDA(launch_pdl(kv_prompt_join_kernel<T, D>, dim3((unsigned)((w.tokens * a.q_heads + 7) / 8)), dim3(256), 0, s, w, a,
                      p.splits));
  return ICX_OK;
}

int launch_prompt_bf16(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, const PromptPlan& p);

}  // namespace icx
