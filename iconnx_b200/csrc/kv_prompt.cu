// Attention of many query rows over the quantised K/V cache (prompt chunks),
// on the 5th-generation tensor cores.
//
// Same mathematics as kv_attention.cuh: the codes themselves are the f16
// operands (a code in the low bits of a half word is code * 2^-24, in bits
// 4..7 sixteen times that), so that with K = c s + lo per group of 64
// dimensions
//     S = sum_groups s (q . c) + lo sum(q),   O = sum (w s) c + sum w lo
// and the scores keep f32 exactness: one accumulator per group in tensor
// memory, scaled and joined in registers.  w s is rounded to two f16 (an f16
// output has as many bits as one; bf16 outputs take kv_prompt_bf16.cu).
//
// Matrix units cut off what falls below an f32 sum's last bit instead of rounding
// it, and sums of codes only grow: in one sum over 16,000 positions they drifted by
// 2.2e-3 of the output's norm (8 bits: 3.6e-3), where f16's rounding is 2.1e-4.  So
// tensor memory sums pieces of 8 tiles, which the softmax warps add in rounded f32
// (3.0e-4; 3.1e-4; pieces of 16: 4.0e-4 and 5.8e-4).  128 rows' earlier pieces are
// 64 KB, which neither tensor nor shared memory has left: they stand in local
// memory, and cost 821 -> 916 us where 916 is stated below (pieces of 16: 899).
//
// A CTA takes 128 query rows of one (sequence, K/V head), 64 positions at a
// time; two CTAs share an SM, so that one's softmax runs beside the other's
// matrix instructions:
//   warps 0..3  softmax: thread = row.  They put q into shared memory, turn
//               each tile's accumulators into weights, put w s back over them
//               in tensor memory (as the left operand of the output product),
//               rescale the output when the reference moves, and write it.
//   warps 4..7  bring the codes from the pages, spread them to f16 and store
//               them in the 128-byte swizzled layout (two stages); warp 4 also
//               decodes the scales, and warp 7 issues the products:
//               S = Q C_k^T (both K-major) and O += (W s) C_v (C_v as it
//               stands, position by position: MN-major).
// Bound by the softmax warps' chain of dependent steps (about ten instructions per
// score, pairs of f32 in one; an instruction issues in 42% of the cycles, most waits
// are for tensor and local memory; tensor cores 13% busy).  1024 tokens of each of 2 sequences of up to 6,000,
// 8 K/V heads of 4 query heads of 128, 4 bits: 916 us (floor 73 at 1.72 PFLOP/s,
// with one f16 for each operand).
#include "kv_prompt.cuh"
#include "tmap.cuh"

namespace icx {

constexpr int kPrPiece = 8;   // tiles whose products are summed in tensor memory

template <int D>
struct PromptConfig {
  static constexpr int G = D / kPrGroup;
  static constexpr int kQ = G * kPrRows * 128;       // per group: rows of 64 f16
  static constexpr int kTile = G * kPrKeys * 128;    // K or V of a stage
  static constexpr int kParam = 4 * G * kPrKeys * 4; // s_k, lo_k, s_v, lo_v per group and position
  static constexpr int kStage = 2 * kTile + kParam;
  static constexpr int kSmem = 1024 + kQ + 2 * kStage + 256;
  static constexpr int kSCols = G * kPrKeys;         // S; the left operand of the output over it
  static constexpr int kTmemCols = D == 64 ? 128 : 256;
};

template <typename T, int D, int BITS>
__global__ void __launch_bounds__(kPrThreads, 2)
    kv_prompt_kernel(const __grid_constant__ KvView c, const __grid_constant__ KvTokens w,
                     const __grid_constant__ AttendArgs a, int splits) {
  using C = PromptConfig<D>;
  constexpr int G = C::G;
  constexpr bool PLO = true;   // w s as two f16: an f16 output has as many bits as one
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  // stage n: K [G][64][128 bytes], V likewise, then the parameters
  auto s_k = [&](int n) { return smem + C::kQ + n * 2 * C::kTile; };
  auto s_v = [&](int n) { return smem + C::kQ + n * 2 * C::kTile + C::kTile; };
  auto s_p = [&](int n) { return reinterpret_cast<float*>(smem + C::kQ + 4 * C::kTile + n * C::kParam); };
  float* s_fix = reinterpret_cast<float*>(smem + C::kQ + 2 * C::kStage);   // [2][2] factors of the output, [2][4] holes, [2][2] 1 / unit of w s
  __shared__ __align__(8) uint64_t bars[8];
  uint64_t *full = bars, *empty = bars + 2, *q_full = bars + 4, *s_full = bars + 5, *p_full = bars + 6, *o_full = bars + 7;
  __shared__ uint32_t tmem_slot;
  __shared__ int s_seq, s_tile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = a.q_heads / c.heads;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full[i], 4);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 4);   // one per warp
    mbar_init(s_full, 1);
    mbar_init(p_full, 4);
    mbar_init(o_full, 1);
    fence_barrier_init();
  }
  if (warp == 7) {
    tmem_alloc(&tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 0) find_row_tile(c, w, share, kPrRows, blockIdx.x, &s_seq, &s_tile);
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
    const PromptShare part(see_any, kPrKeys, splits);
    const int tiles = part.tiles, p0 = part.first, p_end = part.end;
    if (threadIdx.x == 0 && su.len > reach) record_bad_page();

    if (warp >= 4) {
      // ------------------------------------------------------------ codes
      const int p = threadIdx.x - 128, key = p >> 1, half = p & 1;
      RawCodes<D, BITS> raw;
      int hole = 0;            // this position has no page (or does not exist)
      uint32_t kp[2][G], vp[2][G];   // warp 4: parameters of positions lane, lane + 32
      bool pvalid[2] = {false, false};
      auto fetch = [&](int i) {
        const int pos = p0 + i * kPrKeys + key;
        const int64_t page = pos < p_end ? kv_page(c, w, seq, pos) : -1;
        hole = pos < p_end && page < 0;
        if (hole && half == 0) record_bad_page();
        if (page >= 0) raw.load(c, kv_row(c, page, head, pos), pos, half);
        if (warp == 4) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int pp = p0 + i * kPrKeys + lane + 32 * x;
            const int64_t pg = pp < p_end ? kv_page(c, w, seq, pp) : -1;
            pvalid[x] = pg >= 0;
            if (pvalid[x]) {
              const int64_t row = kv_row(c, pg, head, pp) * G;
              load_words(c.params[0] + row, kp[x]);
              load_words(c.params[1] + row, vp[x]);
            }
          }
        }
      };
      float vmax[G], vdown[G];
#pragma unroll
      for (int k = 0; k < G; ++k) vmax[k] = vdown[k] = 0.0f;
      constexpr uint32_t id_s = prompt_idesc(kPrKeys, false), id_o = prompt_idesc(kPrGroup, true);
      const uint32_t t_s = tmem, t_o = tmem + C::kSCols;
      auto output = [&](int i) {   // O += (W s) C_v of tile i
        const int st = i & 1;
#pragma unroll
        for (int k = 0; k < G; ++k) {
          // MN-major: 64 dimensions are one 128-byte row, 8 positions 1024 bytes
          const uint64_t b = smem_desc_k128(smem_addr(s_v(st) + k * kPrKeys * 128));
#pragma unroll
          for (int lo = 0; lo < (PLO ? 2 : 1); ++lo)
#pragma unroll
            for (int n = 0; n < kPrKeys / 16; ++n)
              mma_f16_ts(t_o + k * kPrGroup, t_s + (lo * G + k) * (kPrKeys / 2) + n * 8, b + (uint64_t)(n * 128), id_o,
                         i % kPrPiece > 0 || lo > 0 || n > 0);
        }
      };
      bool ok = true;
      if (tiles > 0) fetch(0);
      for (int i = 0; i < tiles; ++i) {
        const int st = i & 1;
        if (ok) ok = wait_warp(&empty[st], ((i >> 1) & 1) ^ 1, ICX_DEVICE_TIMEOUT_PRODUCER);
        // spread to f16: row = position, piece n at place n ^ (row & 7)
#pragma unroll
        for (int k = 0; k < G; ++k) {
          uint8_t* kr = s_k(st) + k * kPrKeys * 128 + key * 128;
          uint8_t* vr = s_v(st) + k * kPrKeys * 128 + key * 128;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const int piece = 2 * (2 * half + x) + n, at = BITS == 4 ? 2 * k + n : 4 * k + 2 * n;
              *reinterpret_cast<uint4*>(kr + ((piece ^ (key & 7)) << 4)) = spread<BITS>(raw.k[x][at], raw.k[x][BITS == 4 ? at : at + 1]);
            }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int piece = 4 * half + x;
            *reinterpret_cast<uint4*>(vr + ((piece ^ (key & 7)) << 4)) = spread<BITS>(raw.v[k][BITS / 4 * x], raw.v[k][BITS == 4 ? x : 2 * x + 1]);
          }
        }
        const uint32_t holes = __ballot_sync(0xffffffffu, hole);   // bit: two lanes per position
        if (lane == 0) reinterpret_cast<uint32_t*>(s_fix)[4 + 4 * st + warp - 4] = holes;   // among the warp's 16 positions
        if (warp == 4) {
          float* prm = s_p(st);   // [4][G][64]: s_k, lo_k, s_v, lo_v
#pragma unroll
          for (int k = 0; k < G; ++k) {
            float s[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t kk = pvalid[x] ? kp[x][k] : 0u, vv = pvalid[x] ? vp[x][k] : 0u;
              prm[(0 * G + k) * kPrKeys + lane + 32 * x] = param_scale(kk);
              prm[(1 * G + k) * kPrKeys + lane + 32 * x] = param_low(kk);
              prm[(3 * G + k) * kPrKeys + lane + 32 * x] = param_low(vv);
              s[x] = param_scale(vv);
            }
            // w s is held times 2^-E, E following the largest s (w <= 2^8 keeps it below 2^15)
            float f = 1.0f;
            const float top = __uint_as_float(__reduce_max_sync(
                0xffffffffu, __float_as_uint(fmaxf(vmax[k], fmaxf(s[0], s[1])))));
            if (top > vmax[k]) {
              const int E = min(max((int)(__float_as_uint(top) >> 23) - 126, -90), 128);
              const float down = __uint_as_float((uint32_t)(5 - E + 127) << 23);
              f = vmax[k] > 0.0f ? down / vdown[k] : 1.0f;
              vmax[k] = __uint_as_float((uint32_t)(min(E + 2, 127) + 127) << 23);
              vdown[k] = down;
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) prm[(2 * G + k) * kPrKeys + lane + 32 * x] = s[x] * vdown[k];
            if (lane == 0) {
              s_fix[st * 2 + k] = f;
              s_fix[12 + st * 2 + k] = vdown[k];
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);
        if (i + 1 < tiles) fetch(i + 1);
        if (warp == 7) {
          // the products of this tile's scores and of the last tile's output
          if (ok && elect_one()) {
            if (i == 0) ok = mbar_wait(q_full, 0, ICX_DEVICE_TIMEOUT_MMA);
            if (ok && i > 0) {
              ok = mbar_wait(p_full, (i - 1) & 1, ICX_DEVICE_TIMEOUT_MMA);
              tc_fence_after();
              if (ok) {
                output(i - 1);
                mma_commit(&empty[(i - 1) & 1]);
              }
            }
            if (ok) ok = mbar_wait(&full[st], (i >> 1) & 1, ICX_DEVICE_TIMEOUT_MMA);
            if (ok) {
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < G; ++k) {
                const uint64_t qa = smem_desc_k128(smem_addr(s_q + k * kPrRows * 128));
                const uint64_t kb = smem_desc_k128(smem_addr(s_k(st) + k * kPrKeys * 128));
#pragma unroll
                for (int n = 0; n < kPrGroup / 16; ++n)
                  mma_f16_ss(t_s + k * kPrKeys, qa + (uint64_t)(n * 2), kb + (uint64_t)(n * 2), id_s, n > 0);
              }
              mma_commit(s_full);
            }
          }
          ok = __all_sync(0xffffffffu, ok);
        }
      }
      if (warp == 7 && ok && tiles > 0 && elect_one() && mbar_wait(p_full, (tiles - 1) & 1, ICX_DEVICE_TIMEOUT_MMA)) {
        tc_fence_after();
        output(tiles - 1);
        mma_commit(o_full);
      }
    } else {
      // ---------------------------------------------------------- softmax
      const int row = threadIdx.x, r = r0 + row;   // this thread's row = TMEM lane
      const bool mine = r < su.rows;
      const int see = mine ? (int)max((int64_t)0, min(first_pos + r / share + 1, (int64_t)reach)) : 0;
      const uint32_t t_s = tmem + ((uint32_t)(warp * 32) << 16), t_o = t_s + C::kSCols;
      float qsum[G], f;
      {
        const T* q = static_cast<const T*>(a.q) + (int64_t)(su.from + (mine ? r / share : 0)) * a.q_token_stride +
                     (int64_t)(head * share + (mine ? r % share : 0)) * a.q_head_stride;
        put_query<T, G, BITS, true>(a, q, mine, row, s_q, &f, qsum);
#pragma unroll
        for (int k = 0; k < G; ++k) qsum[k] *= 5.9604644775390625e-8f;   // in units where a code counts 2^-24
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      const float step = 8.0f / f;       // the reference moves by at least this
      float m = kNoScore, l = 0.0f, vlo[G];
#pragma unroll
      for (int k = 0; k < G; ++k) vlo[k] = 0.0f;
      // the output's sums of the pieces before this one, times kept_by
      alignas(16) float kept[D];   // (local memory: 128 rows take 64 KB)
      float kept_by[G];
#pragma unroll
      for (int k = 0; k < G; ++k) kept_by[k] = 1.0f;
      bool ok = true;
      for (int i = 0; i < tiles; ++i) {
        const int st = i & 1;
        if (ok) ok = wait_warp(&full[st], (i >> 1) & 1, ICX_DEVICE_TIMEOUT_EPILOGUE);
        if (ok) ok = wait_warp(s_full, i & 1, ICX_DEVICE_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
        const float* prm = s_p(st);
        const uint4 holes = *reinterpret_cast<const uint4*>(s_fix + 4 + 4 * st);
        const bool edge = p0 + (i + 1) * kPrKeys > see_all || (holes.x | holes.y | holes.z | holes.w) != 0;
        // -- scores (in units of 1 / f)
        float s[kPrKeys];
#pragma unroll
        for (int n = 0; n < kPrKeys; n += 16) {
          uint32_t x[G][16];
#pragma unroll
          for (int k = 0; k < G; ++k) tmem_ld_32x32b_x16(t_s + (uint32_t)(k * kPrKeys + n), x[k]);
#pragma unroll
          for (int k = 0; k < G; ++k) tmem_ld_wait_regs16(x[k]);
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            F2 u[2];
#pragma unroll
            for (int k = 0; k < G; ++k) {
              const float4 sc = *reinterpret_cast<const float4*>(prm + (0 * G + k) * kPrKeys + n + j);
              const float4 lo = *reinterpret_cast<const float4*>(prm + (1 * G + k) * kPrKeys + n + j);
              const F2 qs = f2(qsum[k], qsum[k]);
              const F2 x0 = f2(__uint_as_float(x[k][j]), __uint_as_float(x[k][j + 1]));
              const F2 x1 = f2(__uint_as_float(x[k][j + 2]), __uint_as_float(x[k][j + 3]));
              u[0] = k == 0 ? f2_mul(f2(lo.x, lo.y), qs) : f2_fma(f2(lo.x, lo.y), qs, u[0]);
              u[1] = k == 0 ? f2_mul(f2(lo.z, lo.w), qs) : f2_fma(f2(lo.z, lo.w), qs, u[1]);
              u[0] = f2_fma(f2(sc.x, sc.y), x0, u[0]);
              u[1] = f2_fma(f2(sc.z, sc.w), x1, u[1]);
            }
            f2_split(u[0], s[n + j], s[n + j + 1]);
            f2_split(u[1], s[n + j + 2], s[n + j + 3]);
          }
        }
        if (edge) {
          const uint32_t hw[4] = {holes.x, holes.y, holes.z, holes.w};
#pragma unroll
          for (int j = 0; j < kPrKeys; ++j)
            if (p0 + i * kPrKeys + j >= see || (hw[j >> 4] >> (2 * (j & 15)) & 1u)) s[j] = -INFINITY;
        }
        // -- the reference, and the output's factors when it or the scale of w s moves
        float top = s[0];
#pragma unroll
        for (int j = 1; j < kPrKeys; ++j) top = fmaxf(top, s[j]);
        bool move = top > m + step;
        bool fixed = false;
#pragma unroll
        for (int k = 0; k < G; ++k) fixed |= s_fix[st * 2 + k] != 1.0f;
        if (__any_sync(0xffffffffu, move) || fixed) {
          const float nm = move ? top : m;
          const float alpha = ex2((m - nm) * f);
          m = nm;
          l *= alpha;
#pragma unroll
          for (int k = 0; k < G; ++k) {
            vlo[k] *= alpha;
            kept_by[k] *= alpha * s_fix[st * 2 + k];
          }
          if (i > 0) {   // before the first tile's product there is no output
#pragma unroll 1
            for (int n = 0; n < D; n += 32) {
              uint32_t x[32];
              const float g = alpha * s_fix[st * 2 + n / kPrGroup];
              tmem_ld_32x32b_x32(t_o + (uint32_t)n, x);
              tmem_ld_wait_regs(x);
#pragma unroll
              for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * g);
              tmem_st_32x32b_x32(t_o + (uint32_t)n, x);
            }
          }
        }
        // -- the end of a piece: the next product starts its sum anew
        if (i > 0 && i % kPrPiece == 0) {
#pragma unroll
          for (int k = 0; k < G; ++k) {
#pragma unroll 1
            for (int n = k * kPrGroup; n < (k + 1) * kPrGroup; n += 16) {
              uint32_t x[16];
              tmem_ld_32x32b_x16(t_o + (uint32_t)n, x);
              tmem_ld_wait_regs16(x);
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                float4* sum = reinterpret_cast<float4*>(kept + n + j);
                const float4 old = i > kPrPiece ? *sum : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                *sum = make_float4(fmaf(old.x, kept_by[k], __uint_as_float(x[j])), fmaf(old.y, kept_by[k], __uint_as_float(x[j + 1])),
                                   fmaf(old.z, kept_by[k], __uint_as_float(x[j + 2])), fmaf(old.w, kept_by[k], __uint_as_float(x[j + 3])));
              }
            }
            kept_by[k] = 1.0f;
          }
        }
        // -- weights, and w s as the left operand over the accumulators
        const float mf = fmaxf(m * f, -3e38f);   // finite before the first score
        const F2 f_2 = f2(f, f), m_2 = f2(-mf, -mf);
        F2 lsum = f2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < kPrKeys; j += 2) {
          float e0, e1;
          f2_split(f2_fma(f2(s[j], s[j + 1]), f_2, m_2), e0, e1);
          s[j] = ex2(e0);
          s[j + 1] = ex2(e1);
          lsum = f2_add(lsum, f2(s[j], s[j + 1]));
        }
        {
          float l0, l1;
          f2_split(lsum, l0, l1);
          l += l0 + l1;
        }
#pragma unroll
        for (int k = 0; k < G; ++k) {
          F2 z = f2(0.0f, 0.0f);
#pragma unroll
          for (int n = 0; n < kPrKeys; n += 32) {
            uint32_t hi[16], lo[PLO ? 16 : 1];
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 sv = *reinterpret_cast<const float4*>(prm + (2 * G + k) * kPrKeys + n + j);
              const float4 lv = *reinterpret_cast<const float4*>(prm + (3 * G + k) * kPrKeys + n + j);
              const F2 w0 = f2(s[n + j], s[n + j + 1]), w1 = f2(s[n + j + 2], s[n + j + 3]);
              F2 a0 = f2_mul(w0, f2(sv.x, sv.y)), a1 = f2_mul(w1, f2(sv.z, sv.w));
              F2 b0 = f2(lv.x, lv.y), b1 = f2(lv.z, lv.w);
              float v0, v1, v2, v3;
              f2_split(a0, v0, v1);
              f2_split(a1, v2, v3);
              if (edge) {   // a position that a row does not see gives it nothing, NaN or not
                if (s[n + j] == 0.0f) v0 = 0.0f;
                if (s[n + j + 1] == 0.0f) v1 = 0.0f;
                if (s[n + j + 2] == 0.0f) v2 = 0.0f;
                if (s[n + j + 3] == 0.0f) v3 = 0.0f;
                b0 = f2(s[n + j] == 0.0f ? 0.0f : lv.x, s[n + j + 1] == 0.0f ? 0.0f : lv.y);
                b1 = f2(s[n + j + 2] == 0.0f ? 0.0f : lv.z, s[n + j + 3] == 0.0f ? 0.0f : lv.w);
              }
              z = f2_fma(w0, b0, z);
              z = f2_fma(w1, b1, z);
              hi[j / 2] = pack_f16(v0, v1);
              hi[j / 2 + 1] = pack_f16(v2, v3);
              if constexpr (PLO) {
                const float2 h0 = unpack_f16(hi[j / 2]), h1 = unpack_f16(hi[j / 2 + 1]);
                lo[j / 2] = pack_f16(v0 - h0.x, v1 - h0.y);
                lo[j / 2 + 1] = pack_f16(v2 - h1.x, v3 - h1.y);
              }
            }
            tmem_st_32x32b_x16(t_s + (uint32_t)(k * (kPrKeys / 2) + n / 2), hi);
            if constexpr (PLO) tmem_st_32x32b_x16(t_s + (uint32_t)((G + k) * (kPrKeys / 2) + n / 2), lo);
          }
          float z0, z1;
          f2_split(z, z0, z1);
          vlo[k] += z0 + z1;
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full);
      }
      // ----------------------------------------------------------- output
      if (tiles > 0 && ok) ok = wait_warp(o_full, 0, ICX_DEVICE_TIMEOUT_EPILOGUE);
      tc_fence_after();
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      const int64_t out_row = (int64_t)(su.from + (mine ? r / share : 0)) * a.q_heads + head * share + (mine ? r % share : 0);
      const PromptOut<T, D> out(a, w, splits, out_row);
      if (ok) {
#pragma unroll 1
        for (int k = 0; k < G; ++k) {
          const float vd = tiles > 0 ? s_fix[12 + ((tiles - 1) & 1) * 2 + k] : 0.0f;
          const float up = vd > 0.0f ? 1.0f / vd : 0.0f;
          float low = vlo[0], by = kept_by[0];
#pragma unroll
          for (int kk = 1; kk < G; ++kk) {
            low = k == kk ? vlo[kk] : low;
            by = k == kk ? kept_by[kk] : by;
          }
#pragma unroll 1
          for (int n = 0; n < 2; ++n) {   // dimensions 32 n .. 32 n + 31 of the group
            uint32_t x[32];
            if (tiles > 0) {
              tmem_ld_32x32b_x32(t_o + (uint32_t)(k * kPrGroup + 32 * n), x);
              tmem_ld_wait_regs(x);
            }
            if (tiles > kPrPiece) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                x[j] = __float_as_uint(fmaf(kept[k * kPrGroup + 32 * n + j], by, __uint_as_float(x[j])));
            }
            float y[4][8];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float o = tiles > 0 ? __uint_as_float(x[8 * j + i]) : 0.0f;
                const int d = v_dim<BITS>(j, i);
                y[d >> 3][d & 7] = l != 0.0f ? fmaf(o * (times16<BITS>(i) ? 1048576.0f : 16777216.0f), up, low) * inv : 0.0f;
              }
            if (mine) out.put(k * kPrGroup + 32 * n, y);
          }
        }
        if (mine) out.put_weight(fmaxf(m * f, -3e38f), l);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 7) tmem_dealloc(tmem, C::kTmemCols);
}

template <typename T, int D, int BITS>
static int launch_prompt_kernel(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, const PromptPlan& p) {
  using C = PromptConfig<D>;
  auto kern = kv_prompt_kernel<T, D, BITS>;
  static SharedMemoryOnce once;
  ICX_CUDA(once.allow(kern, C::kSmem));
  ICX_CUDA(launch_pdl(kern, prompt_grid(c, w, a, p), dim3(kPrThreads), C::kSmem, s, c, w, a, p.splits));
  return launch_prompt_join<T, D>(s, w, a, p);
}

static int launch_prompt_f16(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, const PromptPlan& p) {
  using T = __half;
  if (c.dim == 64) return c.bits == 4 ? launch_prompt_kernel<T, 64, 4>(s, c, w, a, p) : launch_prompt_kernel<T, 64, 8>(s, c, w, a, p);
  return c.bits == 4 ? launch_prompt_kernel<T, 128, 4>(s, c, w, a, p) : launch_prompt_kernel<T, 128, 8>(s, c, w, a, p);
}

bool prompt_preferred(const KvView& c, const KvTokens& w, int q_heads, int type) {
  if (type == ICX_F32 || c.group != kPrGroup || c.dim > 128) return false;
  const int64_t rows = w.tokens / w.batch * (q_heads / c.heads);
  return rows >= 64;
}

PromptPlan plan_prompt(const KvView& c, const KvTokens& w, int q_heads, int type) {
  PromptPlan p{kPrRows, 1, 0};
  const int64_t share = q_heads / c.heads;
  // about so many row tiles; bf16 takes twice the rows per CTA if they still
  // fill the GPU
  const auto tiles = [&](int rows) { return (w.tokens * share + rows - 1) / rows * c.heads; };
  if (type == ICX_BF16 && tiles(2 * kPrRows) >= sm_count()) p.rows = 2 * kPrRows;
  // Positions in shares where that fills the GPU (128 tokens of one sequence of
  // 32,000, 8 K/V heads of 4 query heads of 128, 4 bits: f16 2040 -> 328 us in 9
  // shares).  A CTA's start and end cost about what `own` positions cost, and its
  // number of positions is at most the page table's (the host does not know more).
  // Two sequences with 1024 rows each keep whole rows: four shares, which would
  // even out the last wave of CTAs, took 367 us instead of 258.
  const double own = type == ICX_BF16 ? 900 : 300, reach = (double)((int64_t)w.width << c.page_shift);
  const int64_t n = tiles(p.rows), at_once = (int64_t)sm_count() * (type == ICX_BF16 ? 1 : 2);
  double best = 0;
  for (int x = 1; x <= 32 && (x == 1 || n * x <= 2 * at_once); ++x) {
    const double time = (double)((n * x + at_once - 1) / at_once) * (reach / x + own);
    if (x == 1 || time < 0.9 * best) {
      best = time;
      p.splits = x;
    }
  }
  if (p.splits > 1) p.bytes = (size_t)p.splits * w.tokens * q_heads * (c.dim + 2) * 4;
  return p;
}

int launch_prompt(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, int type) {
  const PromptPlan p = plan_prompt(c, w, a.q_heads, type);
  return type == ICX_F16 ? launch_prompt_f16(s, c, w, a, p) : launch_prompt_bf16(s, c, w, a, p);
}

}  // namespace icx
