// Attention of many bf16 query rows over the quantised K/V cache (prompt
// chunks), on the 5th-generation tensor cores.
//
// A bf16 output has 8 significant bits, so here K and V are dequantised to f16
// (11 bits: half a step is 2^-11, an eighth of the output's 2^-8) on their way into
// shared memory, scaled by powers of two into f16's range, and the weights are
// rounded to one f16.  Scores, their maximum and all sums stay f32.  That leaves
// the softmax warps with about five instructions per score, against ten in
// kv_prompt.cu, whose operands are exact and which f16 outputs take.
// What it costs: a score is off by up to 2^-11 of scale * sum |q k|, its weight by
// that part of itself, and a value by 2^-11 of itself (chunks of 400 tokens on up to
// 9,000 positions: error 1.68e-3 of the output's norm, 1.66e-3 of which is bf16's
// own rounding).  Sums need no pieces here: they are of values, not of codes
// that only grow, and what matrix units cut off (up to 2^-23 of the sum per product,
// 16,000 positions are 1,000 products) stays far below 2^-8 of the output.
//
// Dequantising is three instructions per pair: a code put into the low bits of
// 1024 (f16) less 1024 is the code as a number, and code * (s 2^-E) + lo 2^-E is
// the value times 2^-E.  The CTA looks over the scales of all its positions
// first (a sixteenth of the cache) to choose E for K and for V; scales 2^20 times
// smaller than the largest of the CTA's positions keep their 11 bits.  (Those are
// the positions that the last of its rows sees: beyond that factor a row's bits
// depend on positions that it may not see itself.)
// (A code in the low bits of a half word is also the f16 number code * 2^-24,
// which saves the subtraction, but then s 2^24 2^-E has to fit f16: a scale
// 2^15 below the largest was off by half its step.)
//
// A CTA (one per SM) takes 256 query rows of one (sequence, K/V head) as two
// tiles of 128, 48 positions at a time, so that what is dequantised serves both;
// 128 rows where there are too few rows to fill the GPU otherwise:
//   warps 0..7   softmax, thread = row.  Two score accumulators per row tile, so
//                the next tile's scores are computed meanwhile; the weights go
//                back over the accumulator they came from, as the left operand
//                of the output product.
//   warps 8..13  bring codes and scales from the pages, dequantise and store,
//                three warps for even tiles of positions and three for odd ones
//                (K and V apart, four stages each).
//   warps 14, 15 issue the products of a row tile each: the output's of tile i
//                and the scores' of tile i + 2 when tile i's weights are there.
// (48 positions rather than 64: three warps fill them, two threads to each, and
// a row's scores stay in 128 registers.)
//
// Measured: 1024 tokens of each of 2 sequences of up to 6,000, 8 K/V heads of 4
// query heads of 128, 4 bits: 253 us (floor 73 at 1.72 PFLOP/s).  128 rows per
// CTA 284 us, one warp issuing for both row tiles 296 (beside 250 at the time).  About 18 us are a CTA's
// start and end, and 1.5 waves of CTAs leave a quarter of the SMs' time unused.
// Rows that do not see a position must not meet its NaN: a V group that holds
// one is stored as zeros, and the rows that see it end as NaN.  That and pages
// that are missing are found in the first look; only then do the softmax warps
// ask for them, tile by tile.
#include "kv_prompt.cuh"
#include "tmap.cuh"

namespace icx {

constexpr int kB16Keys = 48;   // positions per tile: what three warps dequantise, two threads to each
constexpr int kB16Threads = 512, kB16Stages = 4;
constexpr float kWeightUp = 7.0f;   // scores pass the reference by 8 at most
constexpr int kB16Cols = 64;   // tensor memory columns of an accumulator

template <int D>
struct PromptB16Config {
  static constexpr int G = D / kPrGroup;
  static constexpr int kQ = G * kPrRows * 128;        // of a row tile
  static constexpr int kTile = G * kB16Keys * 128;    // K or V of a stage
  static constexpr int kSmem = 1024 + 2 * kQ + 2 * kB16Stages * kTile;
  // per row tile two score accumulators, then per row tile the output
  static constexpr int kTmemCols = 512;
  static constexpr int kOutCol = 4 * kB16Cols;
};


__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// E for groups with scales up to s_top and low ends up to lo_top: codes x s 2^-E
// and lo 2^-E stay below 2^14 each, their sum below 2^15.
template <int BITS>
__device__ __forceinline__ int unit_for(uint32_t s_top, uint32_t lo_top) {
  const int s = (int)(s_top >> 23) - 126, lo = (int)(lo_top >> 23) - 126;   // below 2^s, 2^lo
  return min(max(max(s + BITS - 14, lo - 14), -100), 120);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Scale (of codes, and of sixteen times codes) and low end of a group in f16.
struct GroupF16 {
  __half2 s, s16, lo;
  __device__ __forceinline__ GroupF16(uint32_t p, float down, bool zero) {
    const float a = zero ? 0.0f : param_scale(p) * down, b = zero ? 0.0f : param_low(p) * down;
    s = __float2half2_rn(a);
    s16 = __float2half2_rn(a * 0.0625f);
    lo = __float2half2_rn(b);
  }
};

// Eight dequantised values of a 16-byte piece, one rounding each (beside the scale's).
template <int BITS>
__device__ __forceinline__ uint4 dequantize(uint32_t w0, uint32_t w1, const GroupF16& g) {
  uint4 u = spread<BITS>(w0, w1);
  uint32_t* v = reinterpret_cast<uint32_t*>(&u);
  const __half2 k1024 = __float2half2_rn(1024.0f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = v[i] | 0x64006400u;   // 1024 + code
    const __half2 code = __hsub2(*reinterpret_cast<const __half2*>(&x), k1024);
    const __half2 y = __hfma2(code, times16<BITS>(2 * i) ? g.s16 : g.s, g.lo);
    v[i] = *reinterpret_cast<const uint32_t*>(&y);
  }
  return u;
}

template <int D, int BITS>
__global__ void __launch_bounds__(kB16Threads, 1)
    kv_prompt_bf16_kernel(const __grid_constant__ KvView c, const __grid_constant__ KvTokens w,
                          const __grid_constant__ AttendArgs a, int rows_per_cta, int splits) {
  using T = __nv_bfloat16;
  using C = PromptB16Config<D>;
  constexpr int G = C::G;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  auto s_k = [&](int n) { return smem + 2 * C::kQ + n * C::kTile; };
  auto s_v = [&](int n) { return smem + 2 * C::kQ + (kB16Stages + n) * C::kTile; };
  __shared__ __align__(8) uint64_t bars[4 * kB16Stages + 14];
  uint64_t *k_full = bars, *k_empty = k_full + kB16Stages, *v_full = k_empty + kB16Stages, *v_empty = v_full + kB16Stages;
  uint64_t *s_full = v_empty + kB16Stages, *p_full = s_full + 4;   // [row tile][accumulator]
  uint64_t *q_full = p_full + 4, *o_full = q_full + 1, *o_done = o_full + 1;   // o_done: as s_full
  __shared__ uint32_t s_look[5];   // largest s and |lo| of K, of V; whether anything is special
  __shared__ uint32_t tmem_slot;
  __shared__ int s_seq, s_tile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = a.q_heads / c.heads;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 5; ++i) s_look[i] = 0u;
    for (int i = 0; i < kB16Stages; ++i) {
      mbar_init(&k_full[i], 3);    // one arrival per warp
      mbar_init(&v_full[i], 3);
      mbar_init(&k_empty[i], 2);   // one per row tile
      mbar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(q_full, 8);
    mbar_init(o_full, 2);
    fence_barrier_init();
  }
  if (warp == 14) {
    tmem_alloc(&tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  if (warp == 0) find_row_tile(c, w, share, rows_per_cta, blockIdx.x, &s_seq, &s_tile);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int seq = s_seq, head = blockIdx.y;
  if (seq >= 0) {
    const SeqUnits su = seq_units(c, w, share, rows_per_cta, seq);
    const int r0 = s_tile * rows_per_cta, nrows = min(rows_per_cta, su.rows - r0);
    const int row_tiles = nrows > kPrRows ? 2 : 1;
    const int64_t first_pos = (int64_t)su.len - su.n;
    const int reach = (int)min((int64_t)su.len, (int64_t)w.width << c.page_shift);
    const int see_any = (int)max((int64_t)0, min(first_pos + (r0 + nrows - 1) / share + 1, (int64_t)reach));
    const PromptShare part(see_any, kB16Keys, splits);
    const int tiles = part.tiles, p0 = part.first, p_end = part.end;
    if (threadIdx.x == 0 && su.len > reach) record_bad_page();

    // the first look
    {
      uint32_t top[4] = {0, 0, 0, 0}, special = 0;
#pragma unroll 4
      for (int pos = p0 + threadIdx.x; pos < p_end; pos += kB16Threads) {
        const int64_t page = kv_page(c, w, seq, pos);
        if (page < 0) {
          special = 1;
          record_bad_page();
          continue;
        }
        uint32_t prm[2][G];
        const int64_t row = kv_row(c, page, head, pos) * G;
        load_words(c.params[0] + row, prm[0]);
        load_words(c.params[1] + row, prm[1]);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int k = 0; k < G; ++k) {
            const float sc = param_scale(prm[x][k]), lo = fabsf(param_low(prm[x][k]));
            if (isnan(sc)) {
              special |= x;
            } else {
              top[2 * x] = max(top[2 * x], __float_as_uint(sc));
              top[2 * x + 1] = max(top[2 * x + 1], __float_as_uint(lo));
            }
          }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        top[x] = __reduce_max_sync(0xffffffffu, top[x]);
        if (lane == 0) atomicMax(&s_look[x], top[x]);
      }
      if (special) s_look[4] = 1u;
      __syncthreads();
    }
    const int k_exp = unit_for<BITS>(s_look[0], s_look[1]), v_exp = unit_for<BITS>(s_look[2], s_look[3]);
    const bool special = s_look[4] != 0u;

    if (warp >= 14) {
      // ---------------------------------------------------------- products
      const int h = warp - 14;   // row tile
      if (h < row_tiles && elect_one()) {
        constexpr uint32_t id_s = prompt_idesc(kB16Keys, false), id_o = prompt_idesc(kPrGroup, true);
        const uint64_t q_desc = smem_desc_k128(smem_addr(s_q + h * C::kQ));
        const uint64_t k_desc = smem_desc_k128(smem_addr(s_k(0))), v_desc = smem_desc_k128(smem_addr(s_v(0)));
        const uint32_t t_acc = tmem + (uint32_t)(2 * h * kB16Cols), t_out = tmem + (uint32_t)(C::kOutCol + h * 128);
        // a stage is free when both row tiles' products have read it
        auto done = [&](uint64_t* bar) {
          mma_commit(bar);
          if (row_tiles == 1) mma_commit(bar);
        };
        // scores of tile i into accumulator i & 1 (its weights of two tiles ago
        // have been issued to the output product before)
        auto scores = [&](int i) {
          const int st = i % kB16Stages;
          if (!mbar_wait(&k_full[st], (uint32_t)(i / kB16Stages & 1), ICX_DEVICE_TIMEOUT_MMA)) return false;
          tc_fence_after();
          const uint64_t kb = k_desc + (uint64_t)(st * (C::kTile >> 4));
#pragma unroll
          for (int k = 0; k < G; ++k)
#pragma unroll
            for (int n = 0; n < kPrGroup / 16; ++n)
              mma_f16_ss(t_acc + (uint32_t)((i & 1) * kB16Cols), q_desc + (uint64_t)(k * (kPrRows * 128 >> 4) + n * 2),
                         kb + (uint64_t)(k * (kB16Keys * 128 >> 4) + n * 2), id_s, k > 0 || n > 0);
          mma_commit(&s_full[2 * h + (i & 1)]);
          done(&k_empty[st]);
          return true;
        };
        bool ok = tiles > 0 && mbar_wait(q_full, 0, ICX_DEVICE_TIMEOUT_MMA);
        for (int i = 0; i < 2 && i < tiles && ok; ++i) ok = scores(i);
        for (int i = 0; i < tiles && ok; ++i) {
          const int st = i % kB16Stages;
          ok = mbar_wait(&v_full[st], (uint32_t)(i / kB16Stages & 1), ICX_DEVICE_TIMEOUT_MMA) &&
               mbar_wait(&p_full[2 * h + (i & 1)], (i >> 1) & 1, ICX_DEVICE_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vb = v_desc + (uint64_t)(st * (C::kTile >> 4));
#pragma unroll
          for (int k = 0; k < G; ++k)
#pragma unroll
            for (int n = 0; n < kB16Keys / 16; ++n)
              mma_f16_ts(t_out + (uint32_t)(k * kPrGroup), t_acc + (uint32_t)((i & 1) * kB16Cols + n * 8),
                         vb + (uint64_t)(k * (kB16Keys * 128 >> 4) + n * 128), id_o, i > 0 || n > 0);
          done(&v_empty[st]);
          mma_commit(&o_done[2 * h + (i & 1)]);
          if (i + 2 < tiles) ok = scores(i + 2);
          if (ok && i + 1 == tiles) done(o_full);
        }
      }
      __syncwarp();
    } else if (warp >= 8) {
      // ------------------------------------------------------ dequantising
      const int set = (warp - 8) / 3, p = threadIdx.x - 256 - set * 96, key = p >> 1, half = p & 1;   // set: tiles set, set + 2, ..
      // the next tile's K codes and scales are fetched when this one's are
      // stored, its V codes likewise
      RawCodes<D, BITS> raw;
      uint32_t kp[G], vp[G];
      int64_t row = -1, row_next = -1;   // cache row of this thread's position, or -1
      auto find = [&](int i) {
        const int pos = p0 + i * kB16Keys + key;
        const int64_t page = pos < p_end ? kv_page(c, w, seq, pos) : -1;
        row_next = page >= 0 ? kv_row(c, page, head, pos) : -1;
      };
      // (a tile is a multiple of 16 positions: the swizzle of the thread's row
      // is the same in all of them)
      auto fetch_k = [&]() {
        if (row_next < 0) return;
        raw.load_k(c, row_next, key, half);
        load_words(c.params[0] + row_next * G, kp);
        load_words(c.params[1] + row_next * G, vp);
      };
      auto fetch_v = [&]() {
        if (row >= 0) raw.load_v(c, row, key, half);
      };
      const float k_down = power_of_two(-k_exp), v_down = power_of_two(-v_exp);
      bool ok = true;
      if (set < tiles) {
        find(set);
        fetch_k();
        row = row_next;
        fetch_v();
        if (set + 2 < tiles) find(set + 2);
      }
      for (int i = set; i < tiles; i += 2) {
        const int st = i % kB16Stages;
        const uint32_t free = (uint32_t)(i / kB16Stages & 1) ^ 1;
        uint32_t vq[G];
#pragma unroll
        for (int k = 0; k < G; ++k) vq[k] = vp[k];
        if (ok) ok = wait_warp(&k_empty[st], free, ICX_DEVICE_TIMEOUT_PRODUCER);
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const GroupF16 g(kp[k], k_down, row < 0);
          uint8_t* kr = s_k(st) + k * kB16Keys * 128 + key * 128;
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const int piece = 2 * (2 * half + x) + n, at = BITS == 4 ? 2 * k + n : 4 * k + 2 * n;
              *reinterpret_cast<uint4*>(kr + ((piece ^ (key & 7)) << 4)) =
                  dequantize<BITS>(raw.k[x][at], raw.k[x][BITS == 4 ? at : at + 1], g);
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[st]);
        if (i + 2 < tiles) fetch_k();
        if (ok) ok = wait_warp(&v_empty[st], free, ICX_DEVICE_TIMEOUT_PRODUCER);
#pragma unroll
        for (int k = 0; k < G; ++k) {
          const GroupF16 g(vq[k], v_down, row < 0 || isnan(param_scale(vq[k])));
          uint8_t* vr = s_v(st) + k * kB16Keys * 128 + key * 128;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int piece = 4 * half + x;
            *reinterpret_cast<uint4*>(vr + ((piece ^ (key & 7)) << 4)) =
                dequantize<BITS>(raw.v[k][BITS / 4 * x], raw.v[k][BITS == 4 ? x : 2 * x + 1], g);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
        row = row_next;
        if (i + 2 < tiles) fetch_v();
        if (i + 4 < tiles) find(i + 4);
      }
    } else {
      // ---------------------------------------------------------- softmax
      const int row = threadIdx.x, r = r0 + row;   // this thread's row = TMEM lane of its row tile
      const bool mine = row < nrows;
      const int see = mine ? (int)max((int64_t)0, min(first_pos + r / share + 1, (int64_t)reach)) : 0;
      const int h = warp >> 2;                     // row tile
      const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16, t_o = tmem + (uint32_t)(C::kOutCol + h * 128);
      // positions that every row of the tile sees
      const int see_all = (int)max((int64_t)0, min(first_pos + (r0 + h * kPrRows) / share + 1, (int64_t)reach));
      bool ok = true;
      const T* q = static_cast<const T*>(a.q) + (int64_t)(su.from + (mine ? r / share : 0)) * a.q_token_stride +
                   (int64_t)(head * share + (mine ? r % share : 0)) * a.q_head_stride;
      float f, qsum[G];
      put_query<T, G, BITS, false>(a, q, mine, row & (kPrRows - 1), s_q + h * C::kQ, &f, qsum);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      const float ft = fminf(fmaxf(f * power_of_two(k_exp), 1e-37f), 1e37f);   // neither 0 nor infinity beside a masked -infinity
      float m = kNoScore, l = 0.0f;   // m: in powers of two
      bool vnan[G];
#pragma unroll
      for (int k = 0; k < G; ++k) vnan[k] = false;
      for (int i = 0; i < tiles && ok && h < row_tiles; ++i) {
        const int st = i & 1;
        ok = wait_warp(&s_full[2 * h + st], (i >> 1) & 1, ICX_DEVICE_TIMEOUT_EPILOGUE);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_s = tmem + t_lane + (uint32_t)((2 * h + st) * kB16Cols);
        uint32_t x0[32], x1[16];
        tmem_ld_32x32b_x32(t_s, x0);
        tmem_ld_32x32b_x16(t_s + 32, x1);
        tmem_ld_wait_regs(x0);
        tmem_ld_wait_regs16(x1);
        float s[kB16Keys];
#pragma unroll
        for (int j = 0; j < kB16Keys; ++j) s[j] = __uint_as_float(j < 32 ? x0[j & 31] : x1[j & 15]);
        if (p0 + (i + 1) * kB16Keys > see_all) {
#pragma unroll
          for (int j = 0; j < kB16Keys; ++j)
            if (p0 + i * kB16Keys + j >= see) s[j] = -INFINITY;
        }
        if (special) {
#pragma unroll
          for (int j = 0; j < kB16Keys; ++j) {
            const int pos = p0 + i * kB16Keys + j;
            if (pos >= see) continue;
            const int64_t page = kv_page(c, w, seq, pos);
            if (page < 0) {
              s[j] = -INFINITY;
              continue;
            }
#pragma unroll
            for (int k = 0; k < G; ++k)
              vnan[k] |= isnan(param_scale(c.params[1][kv_row(c, page, head, pos) * G + k]));
          }
        }
        float tops[4] = {s[0], s[1], s[2], s[3]};   // four chains
#pragma unroll
        for (int j = 4; j < kB16Keys; j += 4)
#pragma unroll
          for (int x = 0; x < 4; ++x) tops[x] = fmaxf(tops[x], s[j + x]);
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * ft;
        const bool move = top > m + 8.0f;
        if (__any_sync(0xffffffffu, move)) {
          const float nm = move ? top : m;
          const float alpha = ex2(m - nm);
          m = nm;
          l *= alpha;
          if (i > 0) {
            // The output so far: this row tile's product of tile i - 1 has to be
            // there.  The barrier's phase before belongs to tile i - 3, whose product
            // the scores of tile i come behind.  (The stages' barriers do not serve:
            // they count the other row tile too, which may be five tiles behind, and
            // then the phase before lets this wait pass.)
            ok = wait_warp(&o_done[2 * h + (st ^ 1)], (uint32_t)((i - 1) >> 1 & 1), ICX_DEVICE_TIMEOUT_EPILOGUE);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int n = 0; n < D; n += 16) {
              uint32_t x[16];
              tmem_ld_32x32b_x16(t_o + t_lane + (uint32_t)n, x);
              tmem_ld_wait_regs16(x);
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * alpha);
              tmem_st_32x32b_x16(t_o + t_lane + (uint32_t)n, x);
            }
          }
        }
        // weights 2^7 times as large, up to 2^15: f16 keeps those 2^-39 of that
        const float m_use = kWeightUp - fmaxf(m, -3e38f);
        const F2 f_2 = f2(ft, ft), m_2 = f2(m_use, m_use);
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
        if (lane == 0) mbar_arrive(&p_full[2 * h + st]);
      }
      // ----------------------------------------------------------- output
      if (tiles > 0 && ok) ok = wait_warp(o_full, 0, ICX_DEVICE_TIMEOUT_EPILOGUE);
      tc_fence_after();
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      const float up = power_of_two(v_exp);
      const int64_t out_row = (int64_t)(su.from + (mine ? r / share : 0)) * a.q_heads + head * share + (mine ? r % share : 0);
      const PromptOut<T, D> out(a, w, splits, out_row);
      if (ok && h < row_tiles) {
#pragma unroll 1
        for (int k = 0; k < G; ++k) {
          bool bad = vnan[0];
#pragma unroll
          for (int kk = 1; kk < G; ++kk) bad = k == kk ? vnan[kk] : bad;
#pragma unroll 1
          for (int n = 0; n < 2; ++n) {   // dimensions 32 n .. 32 n + 31 of the group
            uint32_t x[32];
            if (tiles > 0) {
              tmem_ld_32x32b_x32(t_o + t_lane + (uint32_t)(k * kPrGroup + 32 * n), x);
              tmem_ld_wait_regs(x);
            }
            float y[4][8];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float o = tiles > 0 ? __uint_as_float(x[8 * j + e]) : 0.0f;
                const int d = v_dim<BITS>(j, e);
                y[d >> 3][d & 7] = bad ? NAN : l != 0.0f ? o * inv * up : 0.0f;
              }
            if (mine) out.put(k * kPrGroup + 32 * n, y);
          }
        }
        if (mine) out.put_weight(m, l);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 14) tmem_dealloc(tmem, C::kTmemCols);
}

template <int D, int BITS>
static int launch_kernel(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, const PromptPlan& p) {
  using C = PromptB16Config<D>;
  auto kern = kv_prompt_bf16_kernel<D, BITS>;
  static SharedMemoryOnce once;
  ICX_CUDA(once.allow(kern, C::kSmem));
  ICX_CUDA(launch_pdl(kern, prompt_grid(c, w, a, p), dim3(kB16Threads), C::kSmem, s, c, w, a, p.rows, p.splits));
  return launch_prompt_join<__nv_bfloat16, D>(s, w, a, p);
}

int launch_prompt_bf16(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, const PromptPlan& p) {
  if (c.dim == 64) return c.bits == 4 ? launch_kernel<64, 4>(s, c, w, a, p) : launch_kernel<64, 8>(s, c, w, a, p);
  return c.bits == 4 ? launch_kernel<128, 4>(s, c, w, a, p) : launch_kernel<128, 8>(s, c, w, a, p);
}

}  // namespace icx
