// Attention of many bf16 query rows over the quantised K/V cache (prompt
// chunks), on the 5th-generation tensor cores.
//
// A bf16 output has 8 significant bits, so here K and V are dequantised to f16
// (11 bits: half a step is 2^-12, an eighth of the output's) on their way into
// shared memory, scaled by powers of two into f16's range (K by tile, V by the
// largest value met so far), and the weights are rounded to one f16.  Scores,
// their maximum and all sums stay f32.  That leaves the softmax warps with
// about five instructions per score, against ten in kv_prompt.cu, whose
// operands are exact and which f16 outputs take.
//
// A CTA takes 128 query rows of one (sequence, K/V head), 48 positions at a
// time, two CTAs per SM:
//   warps 0..3  softmax, thread = row.  Two score accumulators, so the next
//               tile's scores are computed meanwhile; the weights go back over
//               the accumulator they came from, as the left operand of the
//               output product.
//   warps 4..6  bring codes and scales from the pages, dequantise and store
//               (K and V apart, two stages each).
//   warp 7      issues the products: the output's of tile i and the scores' of
//               tile i + 2 when tile i's weights are there.
// (48 positions rather than 64: three warps fill them, the fourth of that
// group is free to issue, and a row's scores stay in 128 registers.)
// Rows that do not see a position must not meet its NaN: a V group that holds
// one is stored as zeros and noted, and the rows that see it end as NaN.
#include "kv_prompt.cuh"

namespace icx {

constexpr int kB16Keys = 48;   // positions per tile: what three warps dequantise, two threads to each
constexpr int kB16Threads = 256;
constexpr int kB16Cols = 64;   // tensor memory columns of an accumulator

template <int D>
struct PromptB16Config {
  static constexpr int G = D / kPrGroup;
  static constexpr int kQ = G * kPrRows * 128;
  static constexpr int kTile = G * kB16Keys * 128;    // K or V of a stage
  static constexpr int kSmem = 1024 + kQ + 4 * kTile;
  static constexpr int kTmemCols = 256;               // two score accumulators, D columns of output
};


// What a tile's scores and output need beside the operands; a ring of four:
// a K stage is free when the scores of two tiles ago are there, which were
// issued after the weights of four tiles ago were.
struct TileNote {
  float k_unit;           // scores: accumulator x f x k_unit
  float v_fix;            // factor of the output so far
  float v_unit;           // output: accumulator x v_unit
  uint32_t special;       // any of the following: bit (tile / 4) % 32, left set once it is
  uint32_t holes[4];      // positions without a page: two equal bits each, 16 positions per word
  uint32_t v_nan[4][2];   // positions whose V group holds a NaN, likewise, per group
};

__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// 2^-E that brings top into [2^(n-1), 2^n), and 2^E.
__device__ __forceinline__ void unit_for(float top, int n, float& down, float& up) {
  const int E = min(max((int)(__float_as_uint(top) >> 23) - 126 - n, -100), 120);
  down = __uint_as_float((uint32_t)(127 - E) << 23);
  up = __uint_as_float((uint32_t)(127 + E) << 23);
}

// Eight dequantised values of a 16-byte piece: code x s + lo, one rounding.
// s16 is s / 16 for the values that come out sixteen times too large.
template <int BITS>
__device__ __forceinline__ uint4 dequantize(uint32_t w0, uint32_t w1, __half2 s, __half2 s16, __half2 lo) {
  const uint32_t one = 0x64006400u;   // 1024 in both halves: a code in its low bits is 1024 + code
  const __half2 base = __float2half2_rn(1024.0f);
  uint4 u;
  if (BITS == 4)
    u = make_uint4((w0 & 0x000f000fu) | one, (w0 & 0x00f000f0u) | one, ((w0 >> 8) & 0x000f000fu) | one,
                   ((w0 >> 8) & 0x00f000f0u) | one);
  else
    u = make_uint4((w0 & 0x00ff00ffu) | one, ((w0 >> 8) & 0x00ff00ffu) | one, (w1 & 0x00ff00ffu) | one,
                   ((w1 >> 8) & 0x00ff00ffu) | one);
  uint32_t* v = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 c = __hsub2(*reinterpret_cast<const __half2*>(&v[i]), base);
    const __half2 y = __hfma2(c, times16<BITS>(2 * i) ? s16 : s, lo);
    v[i] = *reinterpret_cast<const uint32_t*>(&y);
  }
  return u;
}

template <int D, int BITS>
__global__ void __launch_bounds__(kB16Threads, 2)
    kv_prompt_bf16_kernel(const __grid_constant__ KvView c, const __grid_constant__ KvTokens w,
                          const __grid_constant__ AttendArgs a) {
  using T = __nv_bfloat16;
  using C = PromptB16Config<D>;
  constexpr int G = C::G;
  constexpr float L = (float)((1 << BITS) - 1);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  auto s_k = [&](int n) { return smem + C::kQ + n * C::kTile; };
  auto s_v = [&](int n) { return smem + C::kQ + (2 + n) * C::kTile; };
  __shared__ __align__(8) uint64_t bars[18];
  uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6, *s_full = bars + 8,
           *p_full = bars + 10, *q_full = bars + 12, *o_full = bars + 13, *note_full = bars + 14;
  __shared__ __align__(16) TileNote note[4];
  __shared__ uint32_t s_top[2][3][2];
  __shared__ uint32_t tmem_slot;
  __shared__ int s_seq, s_tile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = a.q_heads / c.heads;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      note[i].special = 0u;
      mbar_init(&note_full[i], 3);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 3);    // one arrival per warp
      mbar_init(&v_full[i], 3);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    mbar_init(q_full, 4);
    mbar_init(o_full, 1);
    fence_barrier_init();
  }
  if (warp == 7) {
    tmem_alloc(&tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 0) find_row_tile(c, w, share, blockIdx.x, &s_seq, &s_tile);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int seq = s_seq, head = blockIdx.y;
  if (seq >= 0) {
    const SeqUnits su = seq_units(c, w, share, kPrRows, seq);
    const int r0 = s_tile * kPrRows, nrows = min(kPrRows, su.rows - r0);
    const int64_t first_pos = (int64_t)su.len - su.n;
    const int reach = (int)min((int64_t)su.len, (int64_t)w.width << c.page_shift);
    const int see_any = (int)max((int64_t)0, min(first_pos + (r0 + nrows - 1) / share + 1, (int64_t)reach));
    const int see_all = (int)max((int64_t)0, min(first_pos + r0 / share + 1, (int64_t)reach));
    const int tiles = (see_any + kB16Keys - 1) / kB16Keys;
    if (threadIdx.x == 0 && su.len > reach) record_status(ICX_DEVICE_BAD_PAGE);

    if (warp == 7) {
      // ---------------------------------------------------------- products
      if (elect_one()) {
        constexpr uint32_t id_s = prompt_idesc(kB16Keys, false), id_o = prompt_idesc(kPrGroup, true);
        const uint32_t t_o = tmem + 2 * kB16Cols;
        // scores of tile i into accumulator i & 1 (its weights of two tiles ago
        // have been issued to the output product before)
        auto issue_scores = [&](int i) {
          const int st = i & 1;
          if (!mbar_wait(&k_full[st], (i >> 1) & 1, ICX_DEVICE_TIMEOUT_MMA)) return false;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < G; ++k) {
            const uint64_t qa = smem_desc_k128(smem_addr(s_q + k * kPrRows * 128));
            const uint64_t kb = smem_desc_k128(smem_addr(s_k(st) + k * kB16Keys * 128));
#pragma unroll
            for (int n = 0; n < kPrGroup / 16; ++n)
              mma_f16_ss(tmem + (uint32_t)(st * kB16Cols), qa + (uint64_t)(n * 2), kb + (uint64_t)(n * 2), id_s,
                         k > 0 || n > 0);
          }
          mma_commit(&s_full[st]);
          mma_commit(&k_empty[st]);
          return true;
        };
        bool ok = tiles > 0 && mbar_wait(q_full, 0, ICX_DEVICE_TIMEOUT_MMA);
        if (ok) ok = issue_scores(0);
        if (ok && tiles > 1) ok = issue_scores(1);
        for (int i = 0; i < tiles && ok; ++i) {
          const int st = i & 1;
          ok = mbar_wait(&v_full[st], (i >> 1) & 1, ICX_DEVICE_TIMEOUT_MMA) &&
               mbar_wait(&p_full[st], (i >> 1) & 1, ICX_DEVICE_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < G; ++k) {
            const uint64_t b = smem_desc_k128(smem_addr(s_v(st) + k * kB16Keys * 128));
#pragma unroll
            for (int n = 0; n < kB16Keys / 16; ++n)
              mma_f16_ts(t_o + (uint32_t)(k * kPrGroup), tmem + (uint32_t)(st * kB16Cols + n * 8), b + (uint64_t)(n * 128),
                         id_o, i > 0 || n > 0);
          }
          mma_commit(&v_empty[st]);
          if (i + 2 < tiles) ok = issue_scores(i + 2);
          if (i + 1 == tiles) mma_commit(o_full);
        }
      }
      __syncwarp();
    } else if (warp >= 4) {
      // ------------------------------------------------------ dequantising
      const int p = threadIdx.x - 128, key = p >> 1, half = p & 1;
      // the next tile's K codes and scales are fetched when this one's are
      // stored, its V codes likewise
      RawCodes<D, BITS> raw;
      uint32_t kp[G], vp[G];
      int64_t row = -1, row_next = -1;   // cache row of this thread's position, or -1
      bool hole = false, hole_next = false;
      auto find = [&](int i) {
        const int pos = i * kB16Keys + key;
        const int64_t page = pos < see_any ? kv_page(c, w, seq, pos) : -1;
        hole_next = pos < see_any && page < 0;
        if (hole_next && half == 0) record_status(ICX_DEVICE_BAD_PAGE);
        row_next = page >= 0 ? kv_row(c, page, head, pos) : -1;
      };
      auto fetch_k = [&](int i) {
        if (row_next < 0) return;
        raw.load_k(c, row_next, i * kB16Keys + key, half);
        load_words(c.params[0] + row_next * G, kp);
        load_words(c.params[1] + row_next * G, vp);
      };
      auto fetch_v = [&](int i) {
        if (row >= 0) raw.load_v(c, row, i * kB16Keys + key, half);
      };
      float v_max = 0.0f, v_down = 0.0f, v_up = 0.0f;
      bool ok = true;
      if (tiles > 0) {
        find(0);
        fetch_k(0);
        row = row_next;
        hole = hole_next;
        fetch_v(0);
        if (tiles > 1) find(1);
      }
      for (int i = 0; i < tiles; ++i) {
        const int st = i & 1;
        TileNote& nt = note[i & 3];
        // the largest |value| a group can stand for, over the tile
        float k_top = 0.0f, v_top = 0.0f;
        bool nan[G];
#pragma unroll
        for (int k = 0; k < G; ++k) {
          if (row < 0) kp[k] = vp[k] = 0u;
          nan[k] = isnan(param_scale(vp[k]));
          k_top = fmaxf(k_top, fmaxf(fabsf(param_low(kp[k])), fabsf(fmaf(L, param_scale(kp[k]), param_low(kp[k])))));
          v_top = fmaxf(v_top, fmaxf(fabsf(param_low(vp[k])), fabsf(fmaf(L, param_scale(vp[k]), param_low(vp[k])))));
        }
        const uint32_t kt = __reduce_max_sync(0xffffffffu, __float_as_uint(k_top));
        const uint32_t vt = __reduce_max_sync(0xffffffffu, __float_as_uint(v_top));
        if (lane == 0) {
          s_top[st][warp - 4][0] = kt;
          s_top[st][warp - 4][1] = vt;
        }
        asm volatile("bar.sync 1, 96;" ::: "memory");   // warps 4..6
        k_top = v_top = 0.0f;
#pragma unroll
        for (int x = 0; x < 3; ++x) {
          k_top = fmaxf(k_top, __uint_as_float(s_top[st][x][0]));
          v_top = fmaxf(v_top, __uint_as_float(s_top[st][x][1]));
        }
        float k_down, k_up, v_fix = 1.0f;
        unit_for(k_top, 8, k_down, k_up);
        if (v_top > v_max) {   // room for four times as much before the next change
          float down, up;
          unit_for(v_top, 6, down, up);
          v_fix = v_max > 0.0f ? down * v_up : 1.0f;
          v_down = down;
          v_up = up;
          v_max = up * 256.0f;
        }
        __half2 vs2[G], vs16[G], vlo2[G];
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const float s = nan[k] ? 0.0f : param_scale(vp[k]) * v_down, lo = nan[k] ? 0.0f : param_low(vp[k]) * v_down;
          vs2[k] = __float2half2_rn(s);
          vs16[k] = __float2half2_rn(s * 0.0625f);
          vlo2[k] = __float2half2_rn(lo);
        }
        // -- K, and the tile's note
        if (ok) ok = wait_warp(&k_empty[st], ((i >> 1) & 1) ^ 1, ICX_DEVICE_TIMEOUT_PRODUCER);
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const float s = param_scale(kp[k]) * k_down, lo = param_low(kp[k]) * k_down;
          const __half2 s2 = __float2half2_rn(s), s16 = __float2half2_rn(s * 0.0625f), lo2 = __float2half2_rn(lo);
          uint8_t* kr = s_k(st) + k * kB16Keys * 128 + key * 128;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const int piece = 2 * (2 * half + x) + n, at = BITS == 4 ? 2 * k + n : 4 * k + 2 * n;
              *reinterpret_cast<uint4*>(kr + ((piece ^ (key & 7)) << 4)) =
                  dequantize<BITS>(raw.k[x][at], raw.k[x][BITS == 4 ? at : at + 1], s2, s16, lo2);
            }
        }
        {
          const uint32_t holes = __ballot_sync(0xffffffffu, hole);
          uint32_t special = holes;
          if (lane == 0) nt.holes[warp - 4] = holes;
#pragma unroll
          for (int k = 0; k < G; ++k) {
            const uint32_t n = __ballot_sync(0xffffffffu, nan[k]);
            special |= n;
            if (lane == 0) nt.v_nan[warp - 4][k] = n;
          }
          if (lane == 0 && special) atomicOr(&nt.special, 1u << (i >> 2 & 31));
          if (p == 0) {
            nt.k_unit = k_up;
            nt.v_fix = v_fix;
            nt.v_unit = v_up;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&note_full[i & 3]);
          mbar_arrive(&k_full[st]);
        }
        if (i + 1 < tiles) fetch_k(i + 1);
        // -- V
        if (ok) ok = wait_warp(&v_empty[st], ((i >> 1) & 1) ^ 1, ICX_DEVICE_TIMEOUT_PRODUCER);
#pragma unroll
        for (int k = 0; k < G; ++k) {
          uint8_t* vr = s_v(st) + k * kB16Keys * 128 + key * 128;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int piece = 4 * half + x, at = BITS == 4 ? k : 2 * k;
            *reinterpret_cast<uint4*>(vr + ((piece ^ (key & 7)) << 4)) =
                dequantize<BITS>(raw.v[x][at], raw.v[x][BITS == 4 ? at : at + 1], vs2[k], vs16[k], vlo2[k]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
        row = row_next;
        hole = hole_next;
        if (i + 1 < tiles) fetch_v(i + 1);
        if (i + 2 < tiles) find(i + 2);
      }
    } else {
      // ---------------------------------------------------------- softmax
      const int row = threadIdx.x, r = r0 + row;   // this thread's row = TMEM lane
      const bool mine = r < su.rows;
      const int see = mine ? (int)max((int64_t)0, min(first_pos + r / share + 1, (int64_t)reach)) : 0;
      const uint32_t t_lane = (uint32_t)(warp * 32) << 16, t_o = tmem + 2 * kB16Cols;
      bool ok = true;
      const T* q = static_cast<const T*>(a.q) + (int64_t)(su.from + (mine ? r / share : 0)) * a.q_token_stride +
                   (int64_t)(head * share + (mine ? r % share : 0)) * a.q_head_stride;
      float f, qsum[G];
      put_query<T, G, BITS, false>(a, q, mine, row, s_q, &f, qsum);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      float m = kNoScore, l = 0.0f;   // m: in powers of two
      bool vnan[G];
#pragma unroll
      for (int k = 0; k < G; ++k) vnan[k] = false;
      for (int i = 0; i < tiles && ok; ++i) {
        const int st = i & 1;
        ok = wait_warp(&note_full[i & 3], (i >> 2) & 1, ICX_DEVICE_TIMEOUT_EPILOGUE);
        if (ok) ok = wait_warp(&s_full[st], (i >> 1) & 1, ICX_DEVICE_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = tmem + t_lane + (uint32_t)(st * kB16Cols);
        uint32_t x0[32], x1[16];
        tmem_ld_32x32b_x32(t_s, x0);
        tmem_ld_32x32b_x16(t_s + 32, x1);
        const float4 nt = *reinterpret_cast<const float4*>(&note[i & 3]);
        const bool special = (__float_as_uint(nt.w) >> (i >> 2 & 31) & 1u) != 0;
        tmem_ld_wait_regs(x0);
        tmem_ld_wait_regs16(x1);
        float s[kB16Keys];
#pragma unroll
        for (int j = 0; j < kB16Keys; ++j) s[j] = __uint_as_float(j < 32 ? x0[j & 31] : x1[j & 15]);
        if ((i + 1) * kB16Keys > see_all || special) {
          const uint32_t hw[3] = {note[i & 3].holes[0], note[i & 3].holes[1], note[i & 3].holes[2]};
#pragma unroll
          for (int j = 0; j < kB16Keys; ++j) {
            if (i * kB16Keys + j >= see || (hw[j >> 4] >> (2 * (j & 15)) & 1u)) {
              s[j] = -INFINITY;
            } else if (special) {
#pragma unroll
              for (int k = 0; k < G; ++k) vnan[k] |= (note[i & 3].v_nan[j >> 4][k] >> (2 * (j & 15)) & 1u) != 0;
            }
          }
        }
        const float ft = fminf(fmaxf(f * nt.x, 1e-37f), 1e37f);   // neither 0 nor infinity beside a masked -infinity
        float tops[4] = {s[0], s[1], s[2], s[3]};   // four chains
#pragma unroll
        for (int j = 4; j < kB16Keys; j += 4)
#pragma unroll
          for (int x = 0; x < 4; ++x) tops[x] = fmaxf(tops[x], s[j + x]);
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * ft;
        const bool move = top > m + 8.0f;
        if (__any_sync(0xffffffffu, move) || nt.y != 1.0f) {
          const float nm = move ? top : m;
          const float alpha = ex2(m - nm);
          m = nm;
          l *= alpha;
          if (i > 0) {
            // the output so far: its last product has to be there
            ok = wait_warp(&v_empty[(i - 1) & 1], ((i - 1) >> 1) & 1, ICX_DEVICE_TIMEOUT_EPILOGUE);
            if (!ok) break;
            tc_fence_after();
            const float g = alpha * nt.y;
#pragma unroll 1
            for (int n = 0; n < D; n += 16) {
              uint32_t x[16];
              tmem_ld_32x32b_x16(t_o + t_lane + (uint32_t)n, x);
              tmem_ld_wait_regs16(x);
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * g);
              tmem_st_32x32b_x16(t_o + t_lane + (uint32_t)n, x);
            }
          }
        }
        const float m_use = fmaxf(m, -3e38f);
        const F2 f_2 = f2(ft, ft), m_2 = f2(-m_use, -m_use);
        F2 l_a = f2(0.0f, 0.0f), l_b = f2(0.0f, 0.0f);
#pragma unroll
        for (int n = 0; n < kB16Keys; n += 16) {
          uint32_t pk[8];
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            float e0, e1, e2, e3;
            f2_split(f2_fma(f2(s[n + j], s[n + j + 1]), f_2, m_2), e0, e1);
            f2_split(f2_fma(f2(s[n + j + 2], s[n + j + 3]), f_2, m_2), e2, e3);
            e0 = ex2(e0);
            e1 = ex2(e1);
            e2 = ex2(e2);
            e3 = ex2(e3);
            l_a = f2_add(l_a, f2(e0, e1));
            l_b = f2_add(l_b, f2(e2, e3));
            pk[j / 2] = pack_f16(e0, e1);
            pk[j / 2 + 1] = pack_f16(e2, e3);
          }
          tmem_st_32x32b_x8(t_s + (uint32_t)(n / 2), pk);
        }
        float l0, l1;
        f2_split(f2_add(l_a, l_b), l0, l1);
        l += l0 + l1;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[st]);
      }
      // ----------------------------------------------------------- output
      if (tiles > 0 && ok) ok = wait_warp(o_full, 0, ICX_DEVICE_TIMEOUT_EPILOGUE);
      tc_fence_after();
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      const float up = tiles > 0 ? note[(tiles - 1) & 3].v_unit : 0.0f;
      T* out = static_cast<T*>(a.out) +
               ((int64_t)(su.from + (mine ? r / share : 0)) * a.q_heads + head * share + (mine ? r % share : 0)) * D;
      if (ok) {
#pragma unroll 1
        for (int k = 0; k < G; ++k) {
          bool bad = vnan[0];
#pragma unroll
          for (int kk = 1; kk < G; ++kk) bad = k == kk ? vnan[kk] : bad;
#pragma unroll 1
          for (int n = 0; n < 2; ++n) {   // pieces g = 4 n .. 4 n + 3
            uint32_t x[32];
            if (tiles > 0) {
              tmem_ld_32x32b_x32(t_o + t_lane + (uint32_t)(k * kPrGroup + 32 * n), x);
              tmem_ld_wait_regs(x);
            }
            float y[4][8];   // dimensions 16 m + 8 n .. + 7: 2 g + h of the four pieces
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float o = tiles > 0 ? __uint_as_float(x[8 * g + j]) : 0.0f;
                y[v_tile<BITS>(j)][2 * g + v_half(j)] = bad ? NAN : l != 0.0f ? o * inv * up : 0.0f;
              }
            if (mine)
#pragma unroll
              for (int mt = 0; mt < 4; ++mt) store_f32<T, 8>(out + k * kPrGroup + 16 * mt + 8 * n, y[mt]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 7) tmem_dealloc(tmem, C::kTmemCols);
}

template <int D, int BITS>
static int launch_kernel(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a) {
  using C = PromptB16Config<D>;
  auto kern = kv_prompt_bf16_kernel<D, BITS>;
  ICX_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
  const int64_t share = a.q_heads / c.heads;
  const dim3 grid((unsigned)(w.tokens * share / kPrRows + w.batch), (unsigned)c.heads);   // at most so many row tiles
  ICX_CUDA(launch_pdl(kern, grid, dim3(kB16Threads), C::kSmem, s, c, w, a));
  return ICX_OK;
}

int launch_prompt_bf16(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a) {
  if (c.dim == 64) return c.bits == 4 ? launch_kernel<64, 4>(s, c, w, a) : launch_kernel<64, 8>(s, c, w, a);
  return c.bits == 4 ? launch_kernel<128, 4>(s, c, w, a) : launch_kernel<128, 8>(s, c, w, a);
}

}  // namespace icx
