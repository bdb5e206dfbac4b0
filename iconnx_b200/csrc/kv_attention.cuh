// Attention of few query rows over the quantised K/V cache (decoding).
//
// The cache is read once, D bits / 4 + 8 D / group bytes per position and K/V
// head (144 for 128 dimensions of 4 bits in groups of 64), so HBM sets the floor.
// At 4 bits a warp takes about 450 instructions for 16 positions, and at 128
// registers an SM holds 16 warps: an instruction issues in 53% of the cycles, with
// one of a scheduler's four warps ready and most others waiting for the result
// before (integer pipe 50% busy, matrix pipe 23%, HBM 35%): too few warps for so
// many dependent instructions.  Codes are therefore never dequantised: with
// K[p] = c s + lo per group of dimensions,
//     q . K[p] = sum_groups  s (q . c) + lo sum(q)
//     sum_p w_p V[p] = sum_p (w_p s_p) c_p + sum_p w_p lo_p
// and the two contractions run on m16n8k16 matrix instructions whose left
// operand is the codes themselves.  A code c in the low bits of a half word
// *is* the f16 number c * 2^-24 (a subnormal, which the matrix units take at
// full precision), so one mask per two codes makes an operand; a code left in
// bits 4..7 is 16 times that, which the other operand (q) or the final scaling
// (output rows) undoes.  The positions (scores) and the dimensions (output)
// are the 16-row side, the query rows that share a K/V head the 8-column side.
//
// Right operands: q is scaled per row by a power of two into f16's range and
// split into f16 + f16 where it has more than 11 bits (f32 input); w s is scaled
// per group by a power of two that follows the largest s met so far, and split
// into f16 + f16 for every output type: what is rounded there is w s c, and the
// value is what w lo leaves of it, so that beside one strong dimension in a group
// (-50 among values of order 1) a single f16 was off by several steps of bf16.
// The split keeps 22 bits of the largest s's weights, and of smaller ones what
// lies above 2^-25 in its units: an s 2^-13 of the largest keeps about 17 bits, one
// of 2^-20 about 10, beside the weighted low ends, which are f32.
//
// Sums: f32, but matrix units cut off what falls below an f32 sum's last bit
// instead of rounding it, and sums of codes only grow, so that over a warp's share
// of thousands of positions they drifted (9 tokens of each of 115 sequences of up
// to 10,500: f16 outputs off by 1.28e-3 of their norm, where their own rounding is
// 2.07e-4; f32 2.6e-5).  So matrix units sum pieces of 8 steps, and the pieces are
// added in rounded f32 (2.30e-4; 1.3e-6; pieces of 4: 2.26e-4, 1.0e-6).  Earlier
// pieces stand in shared memory, whose third ring stage was worth nothing; in local
// memory, which misses L1, pieces of 8 cost 92 us where they cost 8 now.
//
// Softmax: one pass.  Weights are taken relative to a reference m that only
// moves (rescaling the sums) when a score passes m + 8, so that most tiles
// need one vote and no exchange between lanes: 2^8 more range costs f16
// nothing.  Each lane adds its own positions' weights; lanes are joined once
// per run of positions.
//
// Work: a unit is 16 or 32 positions of one (sequence, K/V head, tile of query
// rows); each warp takes an equal, contiguous share of all units, found on the
// device from seq_lens and cu_tokens, so ragged batches balance and a captured
// call can be replayed with other lengths.  Warps meet nowhere (but at the end of
// the short form, kSplitCta): one that runs into another sequence or head starts
// on it while the other fifteen of the SM keep its pipes busy.  Rows whose units went to several warps leave (m, l, o)
// in the workspace for the join kernel.  All joins run in a fixed order, so
// equal calls give equal results.
//
// Measured: 64 sequences of up to 16,000 positions, one token, 8 K/V heads of 4
// query heads of 128, bf16: 4 bits 220 us (3.5 TB/s; floor 118 us at 6.46 TB/s),
// 8 bits 292 us (4.9 TB/s; floor 222); 212 and 278 in one sum, 197 and 263 with one
// f16 for w s besides.  One sequence of 500, 12 heads of 64, f32, 8 bits: 10 us, latency.
#pragma once

#include <type_traits>

#include "capi.cuh"
#include "common.cuh"
#include "kv_cache.cuh"

namespace icx {

constexpr int kAttWarps = 8;

// Tiles of 16 positions that a warp takes at once: two where codes and sums are
// small enough, which halves what a step costs beside its arithmetic.
__host__ __device__ constexpr int att_subtiles(int dim, int bits, int R) { return dim * bits <= 512 && R <= 8 ? 2 : 1; }
__host__ __device__ constexpr int att_step(int dim, int bits, int R) { return 16 * att_subtiles(dim, bits, R); }
constexpr float kNoScore = -1.7e38f;        // m before the first score

// CTAs per SM: two where 128 registers hold the sums, and shared memory two
// rings beside their queries.
__host__ __device__ constexpr int att_resident(int dim, int nt, int q_bytes) {
  return dim * nt <= 128 && !(q_bytes == 4 && dim == 128) ? 2 : 1;
}

// 8 or 16 query rows per tile.  16 read the cache half as often but take twice
// the registers and instructions, which a warp with few steps has to fetch: they
// pay for long runs in f32 alone (4 tokens of each of 64 sequences of up to 8,000, 8
// K/V heads of 4 query heads of 128, 4 bits: 277 -> 263 us), not in 16 bits (bf16:
// 203 -> 226 us) nor in short runs (6 sequences of up to 5,300, bf16: 42 -> 44 us).
template <typename T>
constexpr int att_most_nt(int dim) {
  return sizeof(T) == 4 && dim <= 128 ? 2 : 1;
}

// What a row's positions are shared out to: one warp; any warps, which leave
// their parts in the workspace; the warps of one CTA, which join in shared memory
// (one launch, no workspace: 1 token on 500 positions, 12 heads of 64, f32: 12.5 -> 10.0
// us; 16 sequences of up to 500, 8 K/V heads of 4 query heads of 128, bf16: 18.6 ->
// 13.8, and 14.4 since w s is two f16).
enum AttendSplit { kSplitNone, kSplitAny, kSplitCta };

struct AttendArgs {
  const void* q;
  int64_t q_token_stride, q_head_stride;
  int q_heads;
  int q_vec;        // four elements of q can be read in one access
  float scale;      // of the scores, times log2(e)
  void* out;
  int64_t* prefix;  // workspace: units before each sequence [batch + 1]
  float* partial;   // workspace: two slots per warp of R x (D + 2) floats
  int split;        // AttendSplit
  int unit;         // positions per unit
};

// Units of a sequence: its row tiles x K/V heads x blocks of positions.
struct SeqUnits {
  int from, n, len, rows, tiles, blocks;
  int64_t units;
};

__device__ __forceinline__ SeqUnits seq_units(const KvView& c, const KvTokens& w, int share, int R, int b,
                                              int unit = 1 << 30) {
  SeqUnits u;
  u.from = b;
  u.n = 1;
  if (w.cu) {
    // rows outside the packed operands do not exist, whatever cu holds
    const int64_t from = max((int64_t)w.cu[b], (int64_t)0);
    const int64_t to = min((int64_t)w.cu[b + 1], w.tokens);
    u.from = (int)from;
    u.n = to > from ? (int)(to - from) : 0;
  }
  u.len = max(w.lens[b], 0);
  u.rows = u.n * share;
  u.tiles = (u.rows + R - 1) / R;
  const int reach = (int)min((int64_t)u.len, (int64_t)w.width << c.page_shift);
  u.blocks = max(1, (int)(((int64_t)reach + unit - 1) / unit));
  u.units = (int64_t)u.tiles * c.heads * u.blocks;
  return u;
}

// How many of the warps get units: all of them, or one per unit.
__device__ __forceinline__ int64_t working_warps(int64_t total, int64_t warps) {
  return max(min(warps, total), (int64_t)1);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

// W consecutive words, W a power of two, naturally aligned up to 16 bytes.
template <int W>
__device__ __forceinline__ void load_words(const uint32_t* p, uint32_t (&r)[W]) {
  if constexpr (W >= 4) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i];
      r[4 * i] = u.x;
      r[4 * i + 1] = u.y;
      r[4 * i + 2] = u.z;
      r[4 * i + 3] = u.w;
    }
  } else if constexpr (W == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    r[0] = u.x;
    r[1] = u.y;
  } else {
    r[0] = *p;
  }
}

// Contiguous global -> shared copy (16-byte aligned, a multiple of 16 bytes),
// counted on `bar`.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_addr(dst)),
               "l"(src), "r"(bytes), "r"(smem_addr(bar))
               : "memory");
}

// Four 8 x 8 matrices of half words, transposed: lane (g, t) gets column g,
// rows 2t and 2t+1 of each.  Lane i gives the address of row i % 8 of matrix
// i / 8.
__device__ __forceinline__ void load_transposed(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// The factor from products of a row scaled by 2^e with codes that count 1 / unit
// to scores in powers of two: above 0, which a masked score's -infinity must not
// meet (below f32's normal numbers all weights are equal anyway).
__device__ __forceinline__ float score_factor(float scale, float unit, int e) {
  return scale != 0.0f ? fmaxf(fabsf(scale) * unit * __uint_as_float((uint32_t)(127 - e) << 23), 1.17549435e-38f) : 1.0f;
}

// Two codes as f16 for a matrix operand: as they stand (subnormals), or as numbers
// around zero: 1024 + code less 1024 + middle.  HIGH: in bits 4..7, sixteen times.
template <bool CENTRE, int BITS, bool HIGH>
__device__ __forceinline__ uint32_t code_operand(uint32_t codes) {
  if constexpr (!CENTRE) return codes;
  constexpr uint32_t zero = BITS == 4 && !HIGH ? 0x64086408u : 0x64806480u;   // 1032, 1152
  uint32_t x = codes | 0x64006400u;
  const __half2 y = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&zero));
  return *reinterpret_cast<const uint32_t*>(&y);
}

template <typename T, int D, int BITS, int GROUP, int NT>
struct AttConfig {
  static constexpr bool QLO = sizeof(T) == 4;
  // f32: codes as f16 integers less kMiddle (one more instruction per operand
  // word), so that the two parts of a sum, s c and lo, do not cancel: with K and V
  // around zero they are some forty times the output (error 3.4e-6 of it without).
  // A code counts 1 then, not 2^-24.  16-bit outputs, with half steps of 2^-11 and
  // 2^-8, go without (64 sequences of up to 16,000 as above, before the pieces: 212
  // -> 265 us with it).
  static constexpr bool CENTRE = sizeof(T) == 4;
  static constexpr float kMiddle = CENTRE ? (float)(1 << (BITS - 1)) : 0.0f;
  static constexpr float kUnit = CENTRE ? 1.0f : 16777216.0f;
  static constexpr int R = 8 * NT;
  static constexpr int G = D / GROUP;
  static constexpr int kMinBlocks = att_resident(D, NT, sizeof(T));
  // q stays in registers where it takes at most 16
  static constexpr bool kQReg = NT == 1 && (D / 16) * 2 * (QLO ? 2 : 1) <= 16;
  static constexpr int kRowFloats = D + 2;
  // a warp's ring: per stage SUB tiles of 16 positions, each K codes, K
  // parameters, V codes, V parameters
  static constexpr int ROW = D * BITS / 8, SUB = att_subtiles(D, BITS, R);
  static constexpr int kCodes = 16 * ROW, kParams = 16 * G * 4;
  static constexpr int kTile = 2 * (kCodes + kParams), kStage = SUB * kTile;
  // a warp's query operand
  static constexpr int kQBytes = kQReg ? 0 : NT * (D / 16) * (QLO ? 2 : 1) * 32 * 8;
  // a warp's sums of earlier pieces, in shared memory where that leaves two
  // stages (not beside 256 dimensions of 8 bits: local memory and larger pieces;
  // 32 sequences of up to 16,000, 8 K/V heads of 4 query heads: 236 -> 272 us)
  static constexpr int kRoom = (kMinBlocks == 2 ? 108 : 220) * 1024 / kAttWarps - kQBytes;
  static constexpr bool kSharedSums = kRoom - R * D * 4 >= 2 * kStage;
  static constexpr int kSumBytes = kSharedSums ? R * D * 4 : 0;
  static constexpr int kPiece = kSharedSums ? 8 : 32;   // steps
  static constexpr int kFit = (kRoom - kSumBytes) / kStage;
  static constexpr int kStages = kFit > 4 ? 4 : kFit < 2 ? 2 : kFit;
  static constexpr int kRing = kAttWarps * kStages * kStage;
  static constexpr int kSums = kRing + kAttWarps * kQBytes;   // where the sums stand
  static constexpr int kSmem = kSums + kAttWarps * kSumBytes;
  static_assert(kSmem * kMinBlocks <= 224 * 1024, "shared memory");
};

template <typename T, int D, int BITS, int GROUP, int NT>
__global__ void __launch_bounds__(32 * kAttWarps, (AttConfig<T, D, BITS, GROUP, NT>::kMinBlocks))
    kv_attend_rows_kernel(const __grid_constant__ KvView c, const __grid_constant__ KvTokens w,
                          const __grid_constant__ AttendArgs a) {
  using C = AttConfig<T, D, BITS, GROUP, NT>;
  constexpr int G = C::G, R = C::R, KS = D / 16, SG = GROUP / 16, MT = D / 16;
  constexpr int KW = D * BITS / 128;   // words of a K chunk
  constexpr int ROW = C::ROW, SUB = C::SUB, kStep = att_step(D, BITS, R);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kAttWarps][C::kStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int share = a.q_heads / c.heads;
  if (lane < C::kStages) mbar_init(&full[warp][lane], 1);
  fence_barrier_init();
  pdl_wait();
  pdl_trigger();

  // this warp's units [u0, u1) of all
  int64_t total = 0;
  for (int b = lane; b < w.batch; b += 32) total += seq_units(c, w, share, R, b, a.unit).units;
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const int64_t all = (int64_t)gridDim.x * kAttWarps, warps = working_warps(total, all);
  // few working warps: one per CTA first
  const int64_t me = warps < all ? (int64_t)warp * gridDim.x + blockIdx.x : (int64_t)blockIdx.x * kAttWarps + warp;
  const bool cta = a.split == kSplitCta;   // a unit (row tile) per CTA
  const int64_t u0 = cta ? min((int64_t)blockIdx.x, total) : min(total * me / warps, total);
  const int64_t u1 = cta ? min((int64_t)blockIdx.x + 1, total) : min(total * (me + 1) / warps, total);
  const bool write = a.split == kSplitAny && me == 0;   // the first warp leaves the prefix sums
  int seq = w.batch;
  int64_t base = 0, before = 0;
  for (int b0 = 0; b0 < w.batch; b0 += 32) {
    const int b = b0 + lane;
    const int64_t n = b < w.batch ? seq_units(c, w, share, R, b, a.unit).units : 0;
    int64_t inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    if (write && b < w.batch) a.prefix[b + 1] = before + inc;
    const uint32_t hit = __ballot_sync(0xffffffffu, before + inc > u0);
    if (hit && seq == w.batch) {
      const int l = __ffs(hit) - 1;
      seq = b0 + l;
      base = before + __shfl_sync(0xffffffffu, inc - n, l);
      if (!write) break;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (write && lane == 0) a.prefix[0] = 0;
  if (u0 >= u1) return;
  SeqUnits su = seq_units(c, w, share, R, seq, a.unit);
  __syncwarp();
  uint32_t phase = 0;   // parity of each stage's barrier
  bool ok = true;       // false once a bounded wait gave up

  for (int64_t u = u0; u < u1;) {
    while (u >= base + su.units) {
      base += su.units;
      su = seq_units(c, w, share, R, ++seq, a.unit);
    }
    const int64_t in = u - base;
    const int block0 = (int)(in % su.blocks);
    const int block1 = (int)min((int64_t)su.blocks, block0 + (u1 - u));
    const int rest = (int)(in / su.blocks);
    const int head = rest / su.tiles, r0 = (rest % su.tiles) * R;
    u += block1 - block0;
    const int row_base = su.from;   // packed row of the sequence's first new token
    const int64_t first_pos = (int64_t)su.len - su.n;
    const int nrows = min(R, su.rows - r0);
    // positions that some row of the tile sees, and that every row sees
    const int reach = (int)min((int64_t)su.len, (int64_t)w.width << c.page_shift);
    const int see_any = (int)max((int64_t)0, min(first_pos + (r0 + nrows - 1) / share + 1, (int64_t)reach));
    const int see_all = (int)max((int64_t)0, min(first_pos + r0 / share + 1, (int64_t)reach));
    if (lane == 0 && su.len > reach) record_bad_page();

    // ------------------------------------------------------- codes on their way
    uint8_t* ring = smem + warp * C::kStages * C::kStage;
    int end = (int)min((int64_t)block1 * a.unit, (int64_t)see_any), p0 = block0 * a.unit;
    if (cta) {
      const int steps = (end + kStep - 1) / kStep;
      p0 = steps * warp / kAttWarps * kStep;
      end = min(end, steps * (warp + 1) / kAttWarps * kStep);
    }
    const int tiles = p0 < end ? (end - p0 + kStep - 1) / kStep : 0;   // steps of SUB tiles
    // lane i < 4 SUB brings piece i % 4 (K codes, K parameters, V codes, V
    // parameters) of tile i / 4
    const int my_piece = lane & 3, my_sub = (lane >> 2) & (SUB - 1);
    const uint32_t my_bytes = (my_piece & 1) ? C::kParams : C::kCodes;
    const int64_t my_row = (my_piece & 1) ? G * 4 : ROW;
    const uint8_t* my_src = ((my_piece & 1) ? reinterpret_cast<const uint8_t*>(c.params[my_piece >> 1]) : c.codes[my_piece >> 1]) +
                            ((int64_t)head << c.page_shift) * my_row;
    const int64_t my_page_bytes = ((int64_t)c.heads << c.page_shift) * my_row;
    const int my_dst = my_sub * C::kTile + (my_piece >> 1) * (C::kCodes + C::kParams) + (my_piece & 1) * C::kCodes;
    // lane i holds the page of this warp's i-th tile of the current 32
    int my_page = -1;
    auto fetch_pages = [&](int from) {   // from: a tile, a multiple of 32
      const int i = from + lane, p = p0 + i / SUB * kStep + i % SUB * 16;
      my_page = p < end ? (int)kv_page(c, w, seq, p) : -1;
      if (p < end && my_page < 0) record_bad_page();
    };
    // bits SUB st ..: which tiles of stage st have a page and positions
    uint32_t there = 0;
    int filled = 0, fill = 0;   // steps brought so far, and the next one's stage
    auto advance = [&]() {
      if (filled >= tiles || !ok) return;
      const int first = filled * SUB & 31;
      if (first == 0) fetch_pages(filled * SUB);
      const int page = __shfl_sync(0xffffffffu, my_page, first + my_sub);
      const uint32_t pages = __ballot_sync(0xffffffffu, my_page >= 0) >> first & ((1u << SUB) - 1);
      there = (there & ~(((1u << SUB) - 1) << (fill * SUB))) | pages << (fill * SUB);
      if (pages != 0) {
        uint64_t* bar = &full[warp][fill];
        if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)__popc(pages) * C::kTile);
        __syncwarp();
        if (lane < 4 * SUB && page >= 0) {
          const int in_page = (p0 + my_sub * 16 + filled * kStep) & ((1 << c.page_shift) - 1);
          bulk_load(ring + fill * C::kStage + my_dst, my_src + page * my_page_bytes + in_page * my_row, my_bytes, bar);
        }
      }
      ++filled;
      fill = fill + 1 == C::kStages ? 0 : fill + 1;
    };
    // the ring holds the next kStages - 1 steps
    for (int i = 0; i < C::kStages - 1; ++i) advance();

    // ------------------------------------------------------ query operand
    // column g of tile x is row r0 + 8 x + g; step j's contraction index of
    // this thread is dimensions 16 j + 4 t + {0,1} and {2,3}
    constexpr int QP = C::QLO ? 2 : 1;   // f16 parts of q
    uint32_t qr[C::kQReg ? KS : 1][QP][2];
    uint2* q_smem = reinterpret_cast<uint2*>(smem + C::kRing + warp * C::kQBytes) + lane;   // [NT][KS][QP][32], own lane's
    float qsum[NT][G][2], qf[NT][2], step[NT][2];   // per column 2t and 2t+1: sums by group, score factor, 8 / factor
    int see[NT][2];                    // positions that row sees
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int r = r0 + 8 * x + g;
      const bool ok = r < su.rows;
      const T* q = static_cast<const T*>(a.q) + (int64_t)(row_base + (ok ? r / share : 0)) * a.q_token_stride +
                   (int64_t)(head * share + (ok ? r % share : 0)) * a.q_head_stride;
      float peak = 0.0f, v[4];
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        load_f32<T, 4>(q + 16 * j + 4 * t, v, a.q_vec);
#pragma unroll
        for (int i = 0; i < 4; ++i) peak = fmaxf(peak, ok ? fabsf(v[i]) : 0.0f);
      }
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
      peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
      // 2^e with peak * 2^e in [2^14, 2^15)
      const int e = peak > 0.0f ? max(-60, min(C::CENTRE ? 96 : 120, 14 - (int)((__float_as_uint(peak) >> 23) & 255) + 127)) : 0;
      // scores are held in units of 1 / f, f > 0: a negative scale turns q round
      const float up = a.scale != 0.0f ? copysignf(__uint_as_float((uint32_t)(e + 127) << 23), a.scale) : 0.0f;
      float sums[G] = {};
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        load_f32<T, 4>(q + 16 * j + 4 * t, v, a.q_vec);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = ok && up != 0.0f ? v[i] * up : 0.0f;
          sums[j / SG] += v[i];
          if (BITS == 4 && (j & 1)) v[i] *= 0.0625f;
        }
        uint32_t part[2][2];
        part[0][0] = pack_f16(v[0], v[1]);
        part[0][1] = pack_f16(v[2], v[3]);
        const float2 h0 = unpack_f16(part[0][0]), h1 = unpack_f16(part[0][1]);
        part[1][0] = pack_f16(v[0] - h0.x, v[1] - h0.y);
        part[1][1] = pack_f16(v[2] - h1.x, v[3] - h1.y);
#pragma unroll
        for (int i = 0; i < QP; ++i) {
          if constexpr (C::kQReg) {
            qr[j][i][0] = part[i][0];
            qr[j][i][1] = part[i][1];
          } else {
            q_smem[((x * KS + j) * QP + i) * 32] = make_uint2(part[i][0], part[i][1]);
          }
        }
      }
      const float f = score_factor(a.scale, C::kUnit, e);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int from = (2 * t + h) * 4;   // a lane that holds column 2t + h
        qf[x][h] = __shfl_sync(0xffffffffu, f, from);
        step[x][h] = 8.0f / qf[x][h];
        const int rr = r0 + 8 * x + 2 * t + h;
        see[x][h] = rr < su.rows ? (int)max((int64_t)0, min(first_pos + rr / share + 1, (int64_t)reach)) : 0;
      }
#pragma unroll
      for (int k = 0; k < G; ++k) {
        float s = sums[k];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s *= 1.0f / C::kUnit;   // in units of a code
        qsum[x][k][0] = __shfl_sync(0xffffffffu, s, 8 * t);
        qsum[x][k][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
      }
    }

    // -------------------------------------------------------- running sums
    float o[NT][MT][4] = {};
    float m[NT][2], l[NT][2], vlo[NT][G][2];
    float4 local_sums[C::kSharedSums ? 1 : NT * MT];
    // the sums of the pieces before this one, [NT][MT], own lane's
    constexpr int kNext = C::kSharedSums ? 32 : 1;
    float4* sums = C::kSharedSums ? reinterpret_cast<float4*>(smem + C::kSums + warp * C::kSumBytes) + lane : local_sums;
    bool pieces = false;   // whether there are any
    auto scale_sums = [&](int i, int n, float f0, float f1) {   // columns 2t and 2t + 1
#pragma unroll 1
      for (float4* v = sums + i * kNext; n > 0; --n, v += kNext) *v = make_float4(v->x * f0, v->y * f1, v->z * f0, v->w * f1);
    };
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        m[x][h] = kNoScore;   // in units of 1 / f
        l[x][h] = 0.0f;
#pragma unroll
        for (int k = 0; k < G; ++k) vlo[x][k][h] = 0.0f;
      }
    // w s is held times 2^-ve, with the largest s at most 2^7 (w at most 2^8)
    float vmax[G], vdown[G];
#pragma unroll
    for (int k = 0; k < G; ++k) {
      vmax[k] = 0.0f;
      vdown[k] = 0.0f;
    }

    // One step: SUB tiles of 16 positions.  EDGE: some row does not see some of
    // them, or a tile has no page.
    auto process = [&](auto edge_tag, int stage, int pos, uint32_t pages) {
      constexpr bool EDGE = decltype(edge_tag)::value;
      const uint8_t* base = ring + stage * C::kStage;
      // -- scores: positions g, g + 8 of each tile (rows) x columns 2t, 2t+1
      float s[SUB][NT][4];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const uint8_t* kc = base + u * C::kTile;
        const uint32_t* kprm = reinterpret_cast<const uint32_t*>(kc + C::kCodes);
        uint32_t kw[2][KW], kp[2][G];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = g + 8 * h;
          if constexpr (KW >= 4) {
#pragma unroll
            for (int i = 0; i < KW; i += 4) {
              const uint4 x = *reinterpret_cast<const uint4*>(kc + at * ROW + k_word_at<ROW>(at, t, i));
              kw[h][i] = x.x;
              kw[h][i + 1] = x.y;
              kw[h][i + 2] = x.z;
              kw[h][i + 3] = x.w;
            }
          } else {
            load_words(reinterpret_cast<const uint32_t*>(kc + at * ROW + k_word_at<ROW>(at, t, 0)), kw[h]);
          }
          load_words(kprm + at * G, kp[h]);
        }
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][x][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < G; ++k) {
          float acc[NT][4] = {};
#pragma unroll
          for (int js = 0; js < SG; ++js) {
            const int j = k * SG + js;
            uint32_t A[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (BITS == 4) {
                const uint32_t word = kw[h][j >> 1];
                if (j & 1) {
                  A[h] = code_operand<C::CENTRE, 4, true>(word & 0x00f000f0u);
                  A[2 + h] = code_operand<C::CENTRE, 4, true>((word >> 8) & 0x00f000f0u);
                } else {
                  A[h] = code_operand<C::CENTRE, 4, false>(word & 0x000f000fu);
                  A[2 + h] = code_operand<C::CENTRE, 4, false>((word >> 8) & 0x000f000fu);
                }
              } else {
                const uint32_t word = kw[h][j];
                A[h] = code_operand<C::CENTRE, 8, false>(word & 0x00ff00ffu);
                A[2 + h] = code_operand<C::CENTRE, 8, false>((word >> 8) & 0x00ff00ffu);
              }
            }
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
              for (int i = 0; i < QP; ++i) {
                if constexpr (C::kQReg) {
                  mma_f16(acc[x], A, qr[j][i][0], qr[j][i][1]);
                } else {
                  const uint2 b = q_smem[((x * KS + j) * QP + i) * 32];
                  mma_f16(acc[x], A, b.x, b.y);
                }
              }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float sc = param_scale(kp[h][k]), lo = C::CENTRE ? fmaf(C::kMiddle, sc, param_low(kp[h][k])) : param_low(kp[h][k]);
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float& v = s[u][x][2 * h + i];
                v = k == 0 ? lo * qsum[x][k][i] : fmaf(lo, qsum[x][k][i], v);
                v = fmaf(sc, acc[x][2 * h + i], v);
              }
          }
        }
        if (EDGE) {
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!(pages >> u & 1u) || pos + 16 * u + g + 8 * (i >> 1) >= see[x][i & 1]) s[u][x][i] = -INFINITY;
        }
      }
      // -- the reference follows the scores in steps of at least 8
      bool move = false;
      float top[NT][2];
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[x][h] = fmaxf(s[0][x][h], s[0][x][2 + h]);
#pragma unroll
          for (int u = 1; u < SUB; ++u) top[x][h] = fmaxf(top[x][h], fmaxf(s[u][x][h], s[u][x][2 + h]));
          move |= top[x][h] > m[x][h] + step[x][h];
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          float moved[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v = top[x][h];
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
            v = fmaxf(v, m[x][h]);
            const float f = ex2((m[x][h] - v) * qf[x][h]);
            m[x][h] = v;
            moved[h] = f;
            l[x][h] *= f;
#pragma unroll
            for (int k = 0; k < G; ++k) vlo[x][k][h] *= f;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[x][i][h] *= f;
              o[x][i][2 + h] *= f;
            }
          }
          if (pieces) scale_sums(x * MT, MT, moved[0], moved[1]);
        }
      }
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float mf = fmaxf(m[x][h] * qf[x][h], -3e38f);   // finite before the first score
#pragma unroll
          for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int i = h; i < 4; i += 2) {
              s[u][x][i] = ex2(fmaf(s[u][x][i], qf[x][h], -mf));
              l[x][h] += s[u][x][i];
            }
        }
      // -- the scale of w s follows the largest s
      bool grow = false;
      uint32_t vp[SUB][2][G];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          load_words(reinterpret_cast<const uint32_t*>(base + u * C::kTile + 2 * C::kCodes + C::kParams) + (g + 8 * h) * G,
                     vp[u][h]);
#pragma unroll
          for (int k = 0; k < G; ++k) {
            // positions behind the last hold whatever the page held before
            if (EDGE && (!(pages >> u & 1u) || pos + 16 * u + g + 8 * h >= see_any)) vp[u][h][k] = 0u;
            grow |= param_scale(vp[u][h][k]) > vmax[k];
          }
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int k = 0; k < G; ++k) {
          float v = vmax[k];
#pragma unroll
          for (int u = 0; u < SUB; ++u) v = fmaxf(v, fmaxf(param_scale(vp[u][0][k]), param_scale(vp[u][1][k])));
          v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
          if (!(v > vmax[k])) continue;
          // v in [2^(E-1), 2^E): 2^(5-E) leaves it below 2^5, with room for 4 times as much
          const int E = min(max((int)(__float_as_uint(v) >> 23) - 126, -90), 128);
          const float down = __uint_as_float((uint32_t)(5 - E + 127) << 23);
          const float f = vmax[k] > 0.0f ? down / vdown[k] : 0.0f;
          vmax[k] = __uint_as_float((uint32_t)(min(E + 2, 127) + 127) << 23);
          vdown[k] = down;
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int i = 0; i < GROUP / 16; ++i)
#pragma unroll
              for (int q = 0; q < 4; ++q) o[x][k * (GROUP / 16) + i][q] *= f;
          if (pieces)
#pragma unroll
            for (int x = 0; x < NT; ++x) scale_sums(x * MT + k * (GROUP / 16), GROUP / 16, f, f);
        }
      }
      // -- output: rows are dimensions, the contraction runs over the positions
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        uint32_t ph[G][NT][2], pl[G][NT][2];
#pragma unroll
        for (int k = 0; k < G; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float sv = param_scale(vp[u][h][k]) * vdown[k];
            const float lo = C::CENTRE ? fmaf(C::kMiddle, param_scale(vp[u][h][k]), param_low(vp[u][h][k])) : param_low(vp[u][h][k]);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              const float e0 = s[u][x][2 * h], e1 = s[u][x][2 * h + 1];
              float w0 = e0 * sv, w1 = e1 * sv;
              if (EDGE) {   // a position that a row does not see gives it nothing, NaN or not
                const int at = pos + 16 * u + g + 8 * h;
                if (at >= see[x][0]) w0 = 0.0f;
                else vlo[x][k][0] = fmaf(e0, lo, vlo[x][k][0]);
                if (at >= see[x][1]) w1 = 0.0f;
                else vlo[x][k][1] = fmaf(e1, lo, vlo[x][k][1]);
              } else {
                vlo[x][k][0] = fmaf(e0, lo, vlo[x][k][0]);
                vlo[x][k][1] = fmaf(e1, lo, vlo[x][k][1]);
              }
              const uint32_t hi = pack_f16(w0, w1);
              ph[k][x][h] = transpose_8x8(hi);
              const float2 f = unpack_f16(hi);
              pl[k][x][h] = transpose_8x8(pack_f16(w0 - f.x, w1 - f.y));
            }
          }
        // lane's row: position lane % 16, piece lane / 16 of a pair
        const int vr = lane & 15;
        const uint32_t v_at = smem_addr(base + u * C::kTile + C::kCodes + C::kParams) + vr * ROW;
        const int v_x = (lane >> 4) ^ v_swizzle<ROW>(vr);
#pragma unroll
        for (int pp = 0; pp < ROW / 16; pp += 2) {
          uint32_t r[4];   // pieces pp and pp + 1: positions 2t, 2t+1 and 2t+8, 2t+9
          load_transposed(v_at + ((v_x ^ pp) << 4), r);
          constexpr int kPerPiece = 8 / BITS;   // row tiles
#pragma unroll
          for (int q = 0; q < 2 * kPerPiece; ++q) {
            const int mt = pp * kPerPiece + q, k = mt / (GROUP / 16);
            const uint32_t lo8 = r[q / kPerPiece * 2], hi8 = r[q / kPerPiece * 2 + 1];
            uint32_t A[4];
            if (BITS == 4) {
              const uint32_t a0 = (q & 1) ? lo8 >> 8 : lo8, a1 = (q & 1) ? hi8 >> 8 : hi8;
              A[0] = code_operand<C::CENTRE, 4, false>(a0 & 0x000f000fu);
              A[1] = code_operand<C::CENTRE, 4, true>(a0 & 0x00f000f0u);
              A[2] = code_operand<C::CENTRE, 4, false>(a1 & 0x000f000fu);
              A[3] = code_operand<C::CENTRE, 4, true>(a1 & 0x00f000f0u);
            } else {
              A[0] = code_operand<C::CENTRE, 8, false>(lo8 & 0x00ff00ffu);
              A[1] = code_operand<C::CENTRE, 8, false>((lo8 >> 8) & 0x00ff00ffu);
              A[2] = code_operand<C::CENTRE, 8, false>(hi8 & 0x00ff00ffu);
              A[3] = code_operand<C::CENTRE, 8, false>((hi8 >> 8) & 0x00ff00ffu);
            }
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              mma_f16(o[x][mt], A, ph[k][x][0], ph[k][x][1]);
              mma_f16(o[x][mt], A, pl[k][x][0], pl[k][x][1]);
            }
          }
        }
      }
    };

    // ------------------------------------------------------ the positions
    int stage = 0;
    for (int pos = p0; pos < p0 + tiles * kStep; pos += kStep) {
      __syncwarp();   // every lane is done with the stage that is filled next
      advance();
      const uint32_t pages = there >> (stage * SUB) & ((1u << SUB) - 1);
      if (pages != 0) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][stage], phase >> stage & 1, ICX_DEVICE_TIMEOUT_CACHE));
        phase ^= 1u << stage;
        if (ok) {
          if (pos + 16 * SUB > see_all || pages != (1u << SUB) - 1) process(std::true_type{}, stage, pos, pages);
          else process(std::false_type{}, stage, pos, pages);
        }
      }
      stage = stage + 1 == C::kStages ? 0 : stage + 1;
      if (((pos - p0) / kStep & (C::kPiece - 1)) == C::kPiece - 1) {   // the end of a piece
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            float(&v)[4] = o[x][i];
            float4& sum = sums[(x * MT + i) * kNext];
            if (pieces) sum = make_float4(sum.x + v[0], sum.y + v[1], sum.z + v[2], sum.w + v[3]);
            else sum = make_float4(v[0], v[1], v[2], v[3]);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = 0.0f;
          }
        pieces = true;
      }
    }
    if (pieces) {
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const float4 sum = sums[(x * MT + i) * kNext];
          o[x][i][0] += sum.x;
          o[x][i][1] += sum.y;
          o[x][i][2] += sum.z;
          o[x][i][3] += sum.w;
        }
    }

    // ---------------------------------------------- join lanes, and write
    const bool whole = !cta && block0 == 0 && block1 == su.blocks;
    static_assert(C::kStages * C::kStage >= R * C::kRowFloats * 4, "a warp's ring holds its part");
    float* slot = cta ? reinterpret_cast<float*>(ring) : a.partial + (me * 2 + (block0 == 0 ? 1 : 0)) * R * C::kRowFloats;
    __syncwarp();   // the ring has been read by all lanes
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        m[x][h] = fmaxf(m[x][h] * qf[x][h], kNoScore);   // in powers of two from here
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[x][h] += __shfl_xor_sync(0xffffffffu, l[x][h], d);
        const float inv = !whole ? 1.0f : l[x][h] != 0.0f ? 1.0f / l[x][h] : 0.0f;
        const int r = r0 + 8 * x + 2 * t + h;
        T* out = static_cast<T*>(a.out) +
                 ((int64_t)(row_base + r / share) * a.q_heads + head * share + r % share) * D + 2 * g;
        float* part = slot + (r - r0) * C::kRowFloats + 2 * g;
#pragma unroll
        for (int k = 0; k < G; ++k) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) vlo[x][k][h] += __shfl_xor_sync(0xffffffffu, vlo[x][k][h], d);
          // o in units of the cached values
          const float up = vdown[k] > 0.0f ? 1.0f / vdown[k] : 0.0f;
#pragma unroll
          for (int i = 0; i < GROUP / 16; ++i) {
            const int mt = k * (GROUP / 16) + i;
            const float v[2] = {fmaf(o[x][mt][h] * C::kUnit, up, vlo[x][k][h]) * inv,
                                fmaf(o[x][mt][2 + h] * (BITS == 4 ? C::kUnit * 0.0625f : C::kUnit), up, vlo[x][k][h]) * inv};
            if (r >= su.rows) continue;
            if (whole) store_f32<T, 2>(out + 16 * mt, v);
            else *reinterpret_cast<float2*>(part + 16 * mt) = make_float2(v[0], v[1]);
          }
        }
        if (!whole && g == 0 && r < su.rows) *reinterpret_cast<float2*>(part + D) = make_float2(m[x][h], l[x][h]);
      }
    if (cta) {   // the only pass of this loop, in all warps
      __syncthreads();
      for (int i = threadIdx.x; i < nrows * (D / 2); i += 32 * kAttWarps) {
        const int row = i / (D / 2), d = i % (D / 2) * 2;
        auto at = [&](int z) { return reinterpret_cast<const float*>(smem + z * C::kStages * C::kStage) + row * C::kRowFloats; };
        float top = kNoScore, sum = 0.0f, v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int z = 0; z < kAttWarps; ++z) top = fmaxf(top, at(z)[D]);
#pragma unroll
        for (int z = 0; z < kAttWarps; ++z) {
          const float2 ml = *reinterpret_cast<const float2*>(at(z) + D), y = *reinterpret_cast<const float2*>(at(z) + d);
          const float f = ex2(ml.x - top);
          sum = fmaf(ml.y, f, sum);
          v[0] = fmaf(y.x, f, v[0]);
          v[1] = fmaf(y.y, f, v[1]);
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        v[0] *= inv;
        v[1] *= inv;
        const int r = r0 + row;
        store_f32<T, 2>(static_cast<T*>(a.out) + ((int64_t)(row_base + r / share) * a.q_heads + head * share + r % share) * D + d, v);
      }
    }
  }
}

// Joins the rows whose units went to several warps: `per_row` (1 or 8) warps per
// (token, query head), each taking every per_row-th part, then in order.
template <typename T, int D>
__global__ void __launch_bounds__(256)
    kv_attend_join_kernel(const __grid_constant__ KvView c, const __grid_constant__ KvTokens w,
                          const __grid_constant__ AttendArgs a, int R, int warps, int per_row) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = D / 32;
  __shared__ float s_o[8][D + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mine = warp % per_row;
  const int64_t item = (int64_t)blockIdx.x * (8 / per_row) + warp / per_row;
  const int share = a.q_heads / c.heads;
  const int64_t token = item / a.q_heads;
  const int hq = (int)(item % a.q_heads);
  const int b = item < w.tokens * a.q_heads ? kv_sequence(w, token) : -1;
  int first = 0, last = 0, r = 0;
  if (b >= 0) {
    const SeqUnits su = seq_units(c, w, share, R, b, a.unit);
    r = (int)(token - su.from) * share + hq % share;
    const int64_t total = a.prefix[w.batch], working = working_warps(total, warps);
    const int64_t s0 = a.prefix[b] + ((int64_t)(hq / share) * su.tiles + r / R) * su.blocks, s1 = s0 + su.blocks;
    // the warp that holds unit s is the last with total * warp / working <= s
    if (total > 0) {
      first = (int)(((s0 + 1) * working - 1) / total);
      last = (int)((s1 * working - 1) / total);
    }
  }
  // first == last: written whole, or nothing there
  float m = kNoScore, l = 0.0f, o[E] = {};
  if (first < last) {
    auto part = [&](int i) { return a.partial + (((int64_t)i * 2 + (i == first ? 1 : 0)) * R + r % R) * (D + 2); };
    // 32 parts at a time: a lane each for their factors, then all lanes for each
    for (int i0 = first + mine; i0 <= last; i0 += 32 * per_row) {
      const int n = min(32, (last - i0) / per_row + 1);
      float2 ml = make_float2(kNoScore, 0.0f);
      if (lane < n) ml = *reinterpret_cast<const float2*>(part(i0 + lane * per_row) + D);
      float top = fmaxf(m, ml.x);
#pragma unroll
      for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float moved = ex2(m - top), f = ex2(ml.x - top);
      float sum = ml.y * f;
#pragma unroll
      for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      m = top;
      l = l * moved + sum;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= moved;
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const float fj = __shfl_sync(0xffffffffu, f, j);
        const float* p = part(i0 + j * per_row) + lane * E;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 v = *reinterpret_cast<const float2*>(p + e);
          o[e] = fmaf(v.x, fj, o[e]);
          o[e + 1] = fmaf(v.y, fj, o[e + 1]);
        }
      }
    }
  }
  if (per_row > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
    if (lane == 0) {
      s_o[warp][D] = m;
      s_o[warp][D + 1] = l;
    }
    __syncthreads();
    if (warp != 0) return;
    for (int i = 1; i < per_row; ++i) {
      const float mi = s_o[i][D], li = s_o[i][D + 1];
      const float top = fmaxf(m, mi), fa = ex2(m - top), fb = ex2(mi - top);
      m = top;
      l = l * fa + li * fb;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * fa + s_o[i][lane * E + e] * fb;
    }
  }
  if (first == last) return;
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  T* out = static_cast<T*>(a.out) + (token * a.q_heads + hq) * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const float v[2] = {o[e] * inv, o[e + 1] * inv};
    store_f32<T, 2>(out + e, v);
  }
}

// Which kernel, on how many CTAs.
struct AttendPlan {
  int nt;      // query rows per tile / 8
  int ctas;
  int unit;    // positions per unit
  int split;   // AttendSplit
  size_t prefix_bytes, bytes;   // workspace
};

AttendPlan plan_attend(const KvView& c, const KvTokens& w, int q_heads, int type);

// Many rows per sequence: the tensor-memory kernel (kv_prompt.cu).
bool prompt_preferred(const KvView& c, const KvTokens& w, int q_heads, int type);
int launch_prompt(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, int type);

// Rows per CTA, shares of the positions, and the workspace these need.
struct PromptPlan {
  int rows, splits;
  size_t bytes;
};
PromptPlan plan_prompt(const KvView& c, const KvTokens& w, int q_heads, int type);

template <typename T>
int launch_attend(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, const AttendPlan& p);

template <>
int launch_attend<float>(cudaStream_t, const KvView&, const KvTokens&, const AttendArgs&, const AttendPlan&);
template <>
int launch_attend<__half>(cudaStream_t, const KvView&, const KvTokens&, const AttendArgs&, const AttendPlan&);
template <>
int launch_attend<__nv_bfloat16>(cudaStream_t, const KvView&, const KvTokens&, const AttendArgs&, const AttendPlan&);

template <typename T, int D, int BITS, int GROUP, int NT>
int launch_attend_rows(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a,
                       const AttendPlan& p) {
  using C = AttConfig<T, D, BITS, GROUP, NT>;
  auto kern = kv_attend_rows_kernel<T, D, BITS, GROUP, NT>;
  static SharedMemoryOnce once;
  if (C::kSmem > 40 * 1024)   // beside the static part
    ICX_CUDA(once.allow(kern, C::kSmem));
  ICX_CUDA(launch_pdl(kern, dim3(p.ctas), dim3(32 * kAttWarps), C::kSmem, s, c, w, a));
  if (p.split == kSplitAny) {
    // few rows have many parts each
    const int64_t rows = w.tokens * a.q_heads;
    const int per_row = rows <= 1024 ? 8 : 1;
    ICX_CUDA(launch_pdl(kv_attend_join_kernel<T, D>, dim3((unsigned)((rows * per_row + 7) / 8)), dim3(256), 0, s, c, w, a,
                        C::R, p.ctas * kAttWarps, per_row));
  }
  return ICX_OK;
}

template <typename T, int D, int BITS, int GROUP>
int launch_attend_nt(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, const AttendPlan& p) {
  if constexpr (att_most_nt<T>(D) == 2)
    if (p.nt == 2) return launch_attend_rows<T, D, BITS, GROUP, 2>(s, c, w, a, p);
  return launch_attend_rows<T, D, BITS, GROUP, 1>(s, c, w, a, p);
}

template <typename T, int D>
int launch_attend_dim(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a, const AttendPlan& p) {
  if (c.bits == 4)
    return c.group == 32 ? launch_attend_nt<T, D, 4, 32>(s, c, w, a, p) : launch_attend_nt<T, D, 4, 64>(s, c, w, a, p);
  return c.group == 32 ? launch_attend_nt<T, D, 8, 32>(s, c, w, a, p) : launch_attend_nt<T, D, 8, 64>(s, c, w, a, p);
}

#define ICX_ATTEND_INSTANCE(T)                                                                             \
  template <>                                                                                              \
  int launch_attend<T>(cudaStream_t s, const KvView& c, const KvTokens& w, const AttendArgs& a,            \
                       const AttendPlan& p) {                                                              \
    return c.dim == 64    ? launch_attend_dim<T, 64>(s, c, w, a, p)                                        \
           : c.dim == 128 ? launch_attend_dim<T, 128>(s, c, w, a, p)                                       \
                          : launch_attend_dim<T, 256>(s, c, w, a, p);                                      \
  }

}  // namespace icx
