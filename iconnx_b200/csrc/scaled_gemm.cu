// Scaled int8 product on the 5th-generation tensor cores:
//   out[m,n] = (sum_k q[m,k] w[n,k]) * q_scale[m] * w_scale[n] [+ bias[n]]
//              [+ residual[m,n]],  rounded once to f32 / f16 / bf16.
// The s32 sum is exact (tcgen05.mma kind::i8, K <= 131071) and stays in tensor
// memory; the rest happens in registers on its way out.  Three kernels:
//
//   scaled_rows_kernel    many tokens: 128 (one CTA) or 256 (a CTA pair,
//                         cta_group::2) tokens x 128 / 256 channels per tile,
//                         persistent, bound by the tensor cores (8192 tokens,
//                         K = 4096, N = 14336: 307 us, 3.1 POPS).
//   scaled_stream_kernel  up to 32 tokens, and up to 128 where K is long: the
//                         weight is the 128-row operand and the tokens the
//                         narrow one, so that nothing is padded to 128 tokens; bound by reading the weight
//                         once, which all SMs share by splitting K over the
//                         CTAs of a cluster, summed in s32 through distributed
//                         shared memory (exact, so in any order).  4 tokens,
//                         K = N = 4096: 5.9 us, 2.8 TB/s, latency.
//   scaled_tile_kernel    any K and alignment (TMA needs K % 16 == 0 and
//                         16-byte bases): mma.sync on 64 x 64 tiles.
#include <type_traits>

#include "capi.cuh"
#include "common.cuh"
#include "floats.cuh"
#include "tmap.cuh"

namespace icx {

struct ScaledArgs {
  const int8_t* q;
  const float* q_scale;
  const int8_t* wt;  // [N, K]
  int M, K, N;
  const float* w_scale;
  const float* bias;      // nullable
  const void* residual;   // nullable, out type
  void* out;
};

// One rounding per operation: the product with the token's scale, then with
// the channel's (fused with the bias), then the residual's sum.
__device__ __forceinline__ float scaled_value(int acc, float sa, float sw, float bias) {
  return fmaf(__int2float_rn(acc) * sa, sw, bias);
}

// ------------------------------------------------- any K and any alignment
// 64 tokens x 64 channels per CTA, 128 bytes of K per step, on m16n8k32 matrix
// instructions.  A row may start at any byte, so it is fetched as the aligned
// words that hold it and shifted into place; the next step's words are on their
// way meanwhile.  Where the tiles are few, the CTAs of a cluster (up to eight)
// share out K and sum in s32 through distributed shared memory.  Bound by the
// instructions of the shifts (8 tokens, K = 7425, N = 7424: 89 us, 205 us with
// byte loads and dp4a; 5288 tokens, K = 7816, N = 64: 76 us, 227).
constexpr int kAnyTile = 64, kAnyStep = 128, kAnyRow = kAnyStep / 4 + 4;   // words of a row in shared memory, padded

// The aligned words that hold bytes [at, at + 64) of [from, to), zero outside;
// *shift tells where they start.
__device__ __forceinline__ void fetch_any(const int8_t* from, const int8_t* to, const int8_t* at, bool there,
                                          uint32_t (&w)[17], int* shift) {
  const int8_t* a = reinterpret_cast<const int8_t*>(reinterpret_cast<uintptr_t>(at) & ~uintptr_t(3));
  *shift = (int)(at - a) * 8;
  if (there && a >= from && a + 68 <= to) {
#pragma unroll
    for (int i = 0; i < 17; ++i) w[i] = *reinterpret_cast<const uint32_t*>(a + 4 * i);
  } else {   // a row that does not exist, or the operand's first or last bytes
#pragma unroll 1
    for (int i = 0; i < 17; ++i) {
      uint32_t x = 0;
      if (there)
        for (int b = 0; b < 4; ++b)
          if (a + 4 * i + b >= from && a + 4 * i + b < to) x |= (uint32_t)(uint8_t)a[4 * i + b] << (8 * b);
#pragma unroll
      for (int n = 0; n < 17; ++n) w[n] = n == i ? x : w[n];
    }
  }
}

__device__ __forceinline__ int ld_cluster_s32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ int4 ld_cluster_s32x4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <typename T>
__global__ void __launch_bounds__(256) scaled_tile_kernel(const ScaledArgs p, int split) {
  __shared__ __align__(16) uint32_t s_ab[2][2 * kAnyTile][kAnyRow];   // rows: tokens, then channels
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int m0 = blockIdx.y * kAnyTile, n0 = (int)(blockIdx.x / split) * kAnyTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wm = (warp & 1) * 32, wn = kAnyTile + (warp >> 1) * 16;   // this warp's tokens and channels
  // this thread brings half a row per step
  const int row = threadIdx.x >> 1, half = threadIdx.x & 1;
  const bool token = row < kAnyTile;
  const int index = token ? m0 + row : n0 + row - kAnyTile;
  const bool there = index < (token ? p.M : p.N);
  const int8_t* from = token ? p.q : p.wt;
  const int8_t* to = from + (size_t)(token ? p.M : p.N) * p.K;
  const int8_t* src = from + (size_t)(there ? index : 0) * p.K + half * 64;
  const int steps = (p.K + kAnyStep - 1) / kAnyStep;
  const int k0 = steps * rank / split, k1 = steps * (rank + 1) / split;
  pdl_wait();
  pdl_trigger();
  int acc[2][2][4] = {};
  uint32_t w[17];
  int shift = 0;
  if (k0 < k1) fetch_any(from, to, src + k0 * kAnyStep, there, w, &shift);
  for (int k = k0; k < k1; ++k) {
    uint32_t(*ab)[kAnyRow] = s_ab[(k - k0) & 1];
    // bytes of K that this half row has: what lies behind them meets zeros of q
    const int left = p.K - k * kAnyStep - half * 64;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      uint32_t v[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v[x] = __funnelshift_r(w[i + x], w[i + x + 1], shift);
        const int n = left - 4 * (i + x);
        if (token && n < 4) v[x] &= n <= 0 ? 0u : (1u << (8 * n)) - 1u;
      }
      *reinterpret_cast<uint4*>(&ab[row][half * 16 + i]) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    __syncthreads();   // the other buffer is free then, too: all have passed its products
    if (k + 1 < k1) fetch_any(from, to, src + (k + 1) * kAnyStep, there, w, &shift);
#pragma unroll
    for (int kk = 0; kk < kAnyStep / 4; kk += 8) {
      uint32_t b[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        b[j][0] = ab[wn + 8 * j + g][kk + t];
        b[j][1] = ab[wn + 8 * j + g][kk + t + 4];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t a0 = ab[wm + 16 * i + g][kk + t], a1 = ab[wm + 16 * i + g + 8][kk + t];
        const uint32_t a2 = ab[wm + 16 * i + g][kk + t + 4], a3 = ab[wm + 16 * i + g + 8][kk + t + 4];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
              : "+r"(acc[i][j][0]), "+r"(acc[i][j][1]), "+r"(acc[i][j][2]), "+r"(acc[i][j][3])
              : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[j][0]), "r"(b[j][1]));
      }
    }
  }
  // sums into shared memory; each CTA of the cluster finishes its share of the tokens
  __syncthreads();
  int* sums = reinterpret_cast<int*>(&s_ab[0][0][0]);
  constexpr int kSumRow = kAnyTile + 8;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<int2*>(&sums[(wm + 16 * i + 8 * h + g) * kSumRow + wn - kAnyTile + 8 * j + 2 * t]) =
            make_int2(acc[i][j][2 * h], acc[i][j][2 * h + 1]);
  if (split > 1) cluster_sync();
  else __syncthreads();
  for (int i = threadIdx.x; i < kAnyTile / split * kAnyTile; i += 256) {
    const int r = rank + i / kAnyTile * split, m = m0 + r, n = n0 + i % kAnyTile;
    if (m >= p.M || n >= p.N) continue;
    const int* at = sums + r * kSumRow + i % kAnyTile;
    int sum = split > 1 ? 0 : *at;
    for (int z = 0; split > 1 && z < split; ++z) sum += ld_cluster_s32(cluster_addr(at, (uint32_t)z));
    const size_t o = (size_t)m * p.N + n;
    float v = scaled_value(sum, p.q_scale[m], p.w_scale[n], p.bias ? p.bias[n] : 0.0f);
    if (p.residual) v += to_f32(static_cast<const T*>(p.residual)[o]);
    static_cast<T*>(p.out)[o] = from_f32<T>(v);
  }
  if (split > 1) cluster_sync();   // no CTA leaves while another reads its sums
}

constexpr int kRows = 128;    // rows of the wide operand per CTA
constexpr int kStep = 128;    // K bytes per stage (one 128-byte swizzle atom)

// ------------------------------------------------------------- many tokens
// Warp 0 loads (TMA, 128-byte swizzle), warp 1 issues the matrix
// instructions into two accumulators of BN columns, warps 2..9 finish: each
// takes the 32 tokens of its TMEM quadrant and every other box of 128 output
// bytes per token, which leaves through a swizzled staging box (two per warp)
// by TMA, or row by row where N or the output is not 16-byte aligned.
constexpr int kRowsEpi = 8;
constexpr int kRowsThreads = 64 + 32 * kRowsEpi;

template <int BN, int CG>
struct RowsConfig {
  static constexpr int kABytes = kRows * kStep;
  static constexpr int kBBytes = (BN / CG) * kStep;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = (224 * 1024 - kRowsEpi * (2 * 4096 + 512) - 2048) / kStageBytes;
  static constexpr int kBoxOffset = kStages * kStageBytes;
  static constexpr int kOpOffset = kBoxOffset + kRowsEpi * 2 * 4096;
  static constexpr int kBarOffset = kOpOffset + kRowsEpi * 512;
  static constexpr int kSmem = kBarOffset + 512 + 1024;   // + alignment slack
  static constexpr int kTmemCols = 2 * BN;
  static_assert(kStages >= 3 && (2 * kStages + 4) * 8 + 8 <= 512 && kSmem <= 227 * 1024, "shared memory");
};

template <typename T, int BN, int CG>
__global__ void __launch_bounds__(kRowsThreads, 1)
    scaled_rows_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ ScaledArgs p,
                       int tma_store, int vec_residual) {
  using C = RowsConfig<BN, CG>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::kStages * C::kABytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
  uint64_t* empty = full + C::kStages;
  uint64_t* tfull = empty + C::kStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_n = (p.N + BN - 1) / BN, num_m = (p.M + kRows * CG - 1) / (kRows * CG);
  const int ntiles = num_m * num_n, nk = (p.K + kStep - 1) / kStep;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const int tile0 = CG == 2 ? (int)cluster_id_x() : (int)blockIdx.x;
  const int tstep = CG == 2 ? (int)nclusters_x() : (int)gridDim.x;
  // tiles in bands of 16 token tiles, channel by channel inside a band: the
  // CTAs that run together share few rows of both operands, which stay in L2
  auto tile_at = [&](int t, int& m0, int& n0) {
    const int band = t / (16 * num_n), in = t - band * 16 * num_n;
    const int height = min(16, num_m - band * 16);
    m0 = (band * 16 + in % height) * kRows * CG + (int)rank * kRows;
    n0 = in / height * BN;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], CG * kRowsEpi);   // the leader's counts both CTAs' warps
    }
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (tma_store) tma_prefetch_desc(&tmOut);
  }
  if (warp == 1) {
    if (CG == 2) {
      tmem_alloc_pair(tmem_slot, C::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, C::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if (CG == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = tile0; t < ntiles && ok; t += tstep) {
        int m0, n0;
        tile_at(t, m0, n0);
        n0 += (int)rank * (BN / CG);
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, ICX_DEVICE_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          if (CG == 2) {
            const uint32_t fb = cluster_addr(&full[stage], 0);
            if (rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * C::kStageBytes);
            tma_load_2d_pair(sA + stage * C::kABytes, &tmA, fb, kb * kStep, m0);
            tma_load_2d_pair(sB + stage * C::kBBytes, &tmB, fb, kb * kStep, n0);
          } else {
            mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
            tma_load_2d(sA + stage * C::kABytes, &tmA, &full[stage], kb * kStep, m0);
            tma_load_2d(sB + stage * C::kBBytes, &tmB, &full[stage], kb * kStep, n0);
          }
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = idesc_i8(kRows * CG, BN, true, true);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = tile0; t < ntiles && ok; t += tstep) {
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1, ICX_DEVICE_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(acc * BN);
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait(&full[stage], phase, ICX_DEVICE_TIMEOUT_MMA)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t da = smem_desc_k128(smem_addr(sA + stage * C::kABytes));
          const uint64_t db = smem_desc_k128(smem_addr(sB + stage * C::kBBytes));
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (CG == 2) mma_i8_pair(d, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc, (kb | k) != 0);
            else mma_i8(d, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc, (kb | k) != 0);
          }
          if (CG == 2) {
            mma_commit_pair(cluster_addr(&empty[stage], 0));
            mma_commit_pair(cluster_addr(&empty[stage], 1));
          } else {
            mma_commit(&empty[stage]);
          }
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if (CG == 2) {
          mma_commit_pair(cluster_addr(&tfull[acc], 0));
          mma_commit_pair(cluster_addr(&tfull[acc], 1));
        } else {
          mma_commit(&tfull[acc]);
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
  } else {
    constexpr int CB = 128 / (int)sizeof(T);   // columns of a box
    constexpr int kPiece = 16 / (int)sizeof(T);   // columns of 16 bytes
    const int e = warp - 2, quad = warp & 3, part = e >> 2;
    uint8_t* box0 = smem + C::kBoxOffset + e * 2 * 4096;
    float* ops = reinterpret_cast<float*>(smem + C::kOpOffset + e * 512);   // [CB] scales, [CB] biases
    const T* residual = static_cast<const T*>(p.residual);
    int acc = 0, buf = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    // The residual's box into the places its outputs will take; the box's store
    // of two boxes ago has been read out.
    auto put_residual = [&](uint8_t* box, int mrow0, int nb) {
      if (!residual) return;
      if (tma_store && lane == 0) bulk_wait_read<1>();
      __syncwarp();
      if (vec_residual && nb + CB <= p.N) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = (lane >> 3) + 4 * i;
          v[i] = make_uint4(0, 0, 0, 0);
          if (mrow0 + rr < p.M)
            v[i] = __ldg(reinterpret_cast<const uint4*>(residual + (size_t)(mrow0 + rr) * p.N + nb) + (lane & 7));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int rr = (lane >> 3) + 4 * i;
          *reinterpret_cast<uint4*>(box + rr * 128 + (((lane & 7) ^ (rr & 7)) << 4)) = v[i];
        }
      } else {
        for (int r0 = 0; r0 < 32; r0 += 16) {   // sixteen rows in flight
          T v[16][CB / 32];
#pragma unroll
          for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int x = 0; x < CB / 32; ++x) {
              const int mm = mrow0 + r0 + i, n = nb + x * 32 + lane;
              v[i][x] = mm < p.M && n < p.N ? residual[(size_t)mm * p.N + n] : from_f32<T>(0.0f);
            }
#pragma unroll
          for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int x = 0; x < CB / 32; ++x) {
              const int rr = r0 + i, c = x * 32 + lane;
              *reinterpret_cast<T*>(box + rr * 128 + (((c / kPiece) ^ (rr & 7)) << 4) + c % kPiece * sizeof(T)) = v[i][x];
            }
        }
      }
    };
    for (int t = tile0; t < ntiles; t += tstep) {
      int m0, n0;
      tile_at(t, m0, n0);
      const int mrow0 = m0 + quad * 32, m = mrow0 + lane;
      const float sa = m < p.M ? __ldg(p.q_scale + m) : 0.0f;
      const int nboxes = (min(BN, p.N - n0) + CB - 1) / CB;
      // A warp whose 32 tokens all lie behind the last leaves its boxes alone: they
      // may still be on their way out with the tile before.
      const bool rows_here = mrow0 < p.M;
      // the first box's residual arrives while the products run
      if (rows_here && part < nboxes) put_residual(box0 + buf * 4096, mrow0, n0 + part * CB);
      if (ok) ok = mbar_wait_warp(&tfull[acc], acc_phase, ICX_DEVICE_TIMEOUT_EPILOGUE);
      tc_fence_after();
      const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BN);
      for (int bx = part; ok && rows_here && bx < nboxes; bx += kRowsEpi / 4) {
        const int nb = n0 + bx * CB;
        uint8_t* box = box0 + buf * 4096;
        uint8_t* row = box + lane * 128;
        uint32_t r[32];
        tmem_ld_32x32b_x32(trow + (uint32_t)(bx * CB), r);
        if (bx != part) put_residual(box, mrow0, nb);
        if (tma_store && !residual && lane == 0) bulk_wait_read<1>();
        __syncwarp();
#pragma unroll
        for (int i = 0; i < CB / 32; ++i) {
          const int c = i * 32 + lane, n = nb + c;
          ops[c] = n < p.N ? __ldg(p.w_scale + n) : 0.0f;
          ops[CB + c] = p.bias && n < p.N ? __ldg(p.bias + n) : 0.0f;
        }
        __syncwarp();
#pragma unroll
        for (int half = 0; half < CB / 32; ++half) {
          if (half) tmem_ld_32x32b_x32(trow + (uint32_t)(bx * CB + 32), r);
          tmem_ld_wait_regs(r);
#pragma unroll
          for (int q = 0; q < 32 / kPiece; ++q) {
            const int pc = half * (32 / kPiece) + q;   // piece of the row
            Vec<T, kPiece>* at = reinterpret_cast<Vec<T, kPiece>*>(row + ((pc ^ (lane & 7)) << 4));
            float v[kPiece];
#pragma unroll
            for (int i = 0; i < kPiece; i += 4) {
              const float4 sw = *reinterpret_cast<const float4*>(ops + pc * kPiece + i);
              const float4 bi = *reinterpret_cast<const float4*>(ops + CB + pc * kPiece + i);
              v[i] = scaled_value((int)r[q * kPiece + i], sa, sw.x, bi.x);
              v[i + 1] = scaled_value((int)r[q * kPiece + i + 1], sa, sw.y, bi.y);
              v[i + 2] = scaled_value((int)r[q * kPiece + i + 2], sa, sw.z, bi.z);
              v[i + 3] = scaled_value((int)r[q * kPiece + i + 3], sa, sw.w, bi.w);
            }
            Vec<T, kPiece> u;
            if (residual) {
              u = *at;
#pragma unroll
              for (int i = 0; i < kPiece; ++i) v[i] += to_f32(u.v[i]);
            }
#pragma unroll
            for (int i = 0; i < kPiece; ++i) u.v[i] = from_f32<T>(v[i]);
            *at = u;
          }
        }
        if (tma_store) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmOut, box, nb, mrow0);
            bulk_commit();
          }
          buf ^= 1;
        } else {
          __syncwarp();
          T* out = static_cast<T*>(p.out);
          for (int rr = 0; rr < 32 && mrow0 + rr < p.M; ++rr)
#pragma unroll
            for (int i = 0; i < CB / 32; ++i) {
              const int c = i * 32 + lane;
              if (nb + c < p.N)
                out[(size_t)(mrow0 + rr) * p.N + nb + c] = *reinterpret_cast<const T*>(
                    box + rr * 128 + (((c / kPiece) ^ (rr & 7)) << 4) + c % kPiece * sizeof(T));
            }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) mbar_arrive_cluster(cluster_addr(&tempty[acc], 0));
        else mbar_arrive(&tempty[acc]);
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (tma_store && lane == 0) bulk_wait0();
  }
  tc_fence_before();
  __syncwarp();
  if (CG == 2) cluster_sync();   // neither CTA leaves while the other may still signal or read it
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    if (CG == 2) tmem_dealloc_pair(tmem, C::kTmemCols);
    else tmem_dealloc(tmem, C::kTmemCols);
  }
}

// -------------------------------------------------------------- few tokens
// One tile of 128 channels per cluster; CTA r of the cluster takes its share
// of K.  Warp 0 loads, warp 1 multiplies, and all six finish: the s32 sums go
// through shared memory ([token][channel]), and CTA r sums and writes its
// share of the tokens.
constexpr int kStreamThreads = 192;

template <int TOK>
struct StreamConfig {
  static constexpr int kABytes = kRows * kStep, kBBytes = TOK * kStep;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kFit = (200 * 1024) / kStageBytes;
  static constexpr int kStages = kFit > 8 ? 8 : kFit;
  static constexpr int kBarOffset = kStages * kStageBytes;
  static constexpr int kSmem = kBarOffset + 512 + 1024;
  static constexpr int kTmemCols = TOK < 32 ? 32 : TOK;
  static_assert(TOK * kRows * 4 <= kStages * kStageBytes, "sums over the ring");
};

template <typename T, int TOK>
__global__ void __launch_bounds__(kStreamThreads, 1)
    scaled_stream_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmQ,
                         const __grid_constant__ ScaledArgs p, int split) {
  using C = StreamConfig<TOK>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sQ = smem + C::kStages * C::kABytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
  uint64_t* empty = full + C::kStages;
  uint64_t* done = empty + C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int n0 = (int)blockIdx.x / split * kRows;
  const int nk = (p.K + kStep - 1) / kStep;
  const int kb0 = nk * rank / split, kb1 = nk * (rank + 1) / split;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    fence_barrier_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmQ);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  bool ok = true;
  if (warp == 0) {
    if (elect_one()) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, stage = i % C::kStages;
        if (!mbar_wait(&empty[stage], (uint32_t)(i / C::kStages & 1) ^ 1, ICX_DEVICE_TIMEOUT_PRODUCER)) break;
        mbar_arrive_expect_tx(&full[stage], C::kStageBytes);
        tma_load_2d(sW + stage * C::kABytes, &tmW, &full[stage], kb * kStep, n0);
        tma_load_2d(sQ + stage * C::kBBytes, &tmQ, &full[stage], kb * kStep, 0);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_i8(kRows, TOK, true, true);
      bool good = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, stage = i % C::kStages;
        good = mbar_wait(&full[stage], (uint32_t)(i / C::kStages & 1), ICX_DEVICE_TIMEOUT_MMA);
        if (!good) break;
        tc_fence_after();
        const uint64_t da = smem_desc_k128(smem_addr(sW + stage * C::kABytes));
        const uint64_t db = smem_desc_k128(smem_addr(sQ + stage * C::kBBytes));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_i8(tmem, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc, (i | k) != 0);
        mma_commit(&empty[stage]);
      }
      if (good) mma_commit(done);
    }
  }
  __syncwarp();
  // every warp: its share of the finishing below starts when the sums are whole
  ok = mbar_wait_warp(done, 0, ICX_DEVICE_TIMEOUT_EPILOGUE);
  tc_fence_after();
  int* sums = reinterpret_cast<int*>(smem);   // [TOK][128] over the ring, all of it read by now
  if (warp >= 2 && ok && kb1 > kb0) {
    const int quad = warp & 3;
#pragma unroll
    for (int c0 = 0; c0 < TOK; c0 += 16) {
      if (c0 >= p.M) break;
      uint32_t r[16];
      tmem_ld_32x32b_x16(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)c0, r);
      tmem_ld_wait_regs16(r);
#pragma unroll
      for (int i = 0; i < 16; ++i) sums[(c0 + i) * kRows + quad * 32 + lane] = (int)r[i];
    }
  }
  tc_fence_before();
  if (split > 1) cluster_sync();
  else __syncthreads();
  if (ok) {
    const int m_from = p.M * rank / split, m_to = p.M * (rank + 1) / split;
    // four channels per thread (every CTA of the cluster has steps: nk >= split)
#pragma unroll 2
    for (int i = threadIdx.x; i < (m_to - m_from) * (kRows / 4); i += kStreamThreads) {
      const int m = m_from + i / (kRows / 4), c = i % (kRows / 4) * 4, n = n0 + c;
      if (n >= p.N) continue;
      int4 acc = *reinterpret_cast<const int4*>(sums + m * kRows + c);
      for (int x = 1; x < split; ++x) {   // the others', in any order: s32 sums are exact
        const int4 y = ld_cluster_s32x4(cluster_addr(sums + m * kRows + c, (uint32_t)((rank + x) & (split - 1))));
        acc.x += y.x;
        acc.y += y.y;
        acc.z += y.z;
        acc.w += y.w;
      }
      const int sum[4] = {acc.x, acc.y, acc.z, acc.w};
      const float sa = __ldg(p.q_scale + m);
      const size_t o = (size_t)m * p.N + n;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = 0.0f;
        if (n + e >= p.N) continue;
        v[e] = scaled_value(sum[e], sa, __ldg(p.w_scale + n + e), p.bias ? __ldg(p.bias + n + e) : 0.0f);
        if (p.residual) v[e] += to_f32(static_cast<const T*>(p.residual)[o + e]);
      }
      T* out = static_cast<T*>(p.out) + o;
      if ((reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0 && n + 4 <= p.N) {
        store_f32<T, 4>(out, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.N) out[e] = from_f32<T>(v[e]);
      }
    }
  }
  if (split > 1) cluster_sync();   // no CTA leaves while another reads its sums
  else __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::kTmemCols);
}

// ---------------------------------------------------------------- host side
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
static int make_out_map(CUtensorMap* map, void* out, int M, int N) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) {
    set_error("cuTensorMapEncodeTiled unavailable from the driver");
    return ICX_ERR_CUDA;
  }
  const CUtensorMapDataType type = sizeof(T) == 4                      ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M}, strides[1] = {(cuuint64_t)N * sizeof(T)};
  cuuint32_t box[2] = {128 / sizeof(T), 32}, estr[2] = {1, 1};
  const CUresult r = fn(map, type, 2, out, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled (output) failed (%d) M=%d N=%d", (int)r, M, N);
    return ICX_ERR_CUDA;
  }
  return ICX_OK;
}

// CTA pairs of a kernel that can be resident at once (per device; callers on
// several threads store the same number).
template <typename T, int BN>
static int max_pairs() {
  static std::atomic<int> cached[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 0;
  if (const int known = cached[dev].load(std::memory_order_relaxed)) return known;
  using C = RowsConfig<BN, 2>;
  auto kern = scaled_rows_kernel<T, BN, 2>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * 74);
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return 0;
  }
  cached[dev].store(n, std::memory_order_relaxed);
  return n;
}

template <typename T, int BN, int CG>
static int launch_rows(cudaStream_t s, const ScaledArgs& p, int units) {
  using C = RowsConfig<BN, CG>;
  auto kern = scaled_rows_kernel<T, BN, CG>;
  CUtensorMap ta, tb, to = {};
  int rc = make_tmap(&ta, p.q, p.M, p.K, kRows);
  if (rc) return rc;
  rc = make_tmap(&tb, p.wt, p.N, p.K, BN / CG);
  if (rc) return rc;
  const bool pitch16 = (size_t)p.N * sizeof(T) % 16 == 0;
  const int tma_store = pitch16 && aligned16(p.out);
  if (tma_store) {
    rc = make_out_map<T>(&to, p.out, p.M, p.N);
    if (rc) return rc;
  }
  const int vec_residual = pitch16 && p.residual && aligned16(p.residual);
  static SharedMemoryOnce once;
  ICX_CUDA(once.allow(kern, C::kSmem));
  const long tiles = (long)((p.M + kRows * CG - 1) / (kRows * CG)) * ((p.N + BN - 1) / BN);
  const unsigned grid = (unsigned)(tiles < units ? tiles : units) * CG;
  if (CG == 2)
    ICX_CUDA(launch_pdl_cluster(kern, dim3(grid), dim3(kRowsThreads), C::kSmem, s, 2u, ta, tb, to, p, tma_store,
                                vec_residual));
  else
    ICX_CUDA(launch_pdl(kern, dim3(grid), dim3(kRowsThreads), C::kSmem, s, ta, tb, to, p, tma_store, vec_residual));
  return ICX_OK;
}

// CTAs that share out K for a tile of channels: while the SMs are not all busy
// and a CTA keeps at least four steps.
static int stream_split(const ScaledArgs& p) {
  const int tiles = (p.N + kRows - 1) / kRows, nk = (p.K + kStep - 1) / kStep, sms = sm_count();
  int split = 1;
  while (split < 8 && tiles * split * 2 <= sms && nk / (split * 2) >= 4) split *= 2;
  return split;
}

template <typename T, int TOK>
static int launch_stream(cudaStream_t s, const ScaledArgs& p) {
  using C = StreamConfig<TOK>;
  auto kern = scaled_stream_kernel<T, TOK>;
  CUtensorMap tw, tq;
  int rc = make_tmap(&tw, p.wt, p.N, p.K, kRows);
  if (rc) return rc;
  rc = make_tmap(&tq, p.q, p.M, p.K, TOK);
  if (rc) return rc;
  static SharedMemoryOnce once;
  ICX_CUDA(once.allow(kern, C::kSmem));
  const int tiles = (p.N + kRows - 1) / kRows, split = stream_split(p);
  ICX_CUDA(launch_pdl_cluster(kern, dim3((unsigned)(tiles * split)), dim3(kStreamThreads), C::kSmem, s,
                              (unsigned)split, tw, tq, p, split));
  return ICX_OK;
}

template <typename T>
static int launch_scaled(cudaStream_t s, const ScaledArgs& p) {
  if (p.K == 0 || p.K % 16 != 0 || !aligned16(p.q) || !aligned16(p.wt)) {
    const unsigned tn = (unsigned)((p.N + kAnyTile - 1) / kAnyTile), tm = (unsigned)((p.M + kAnyTile - 1) / kAnyTile);
    // K in shares while that leaves three CTAs per SM or fewer, of two steps or more
    const int steps = (p.K + kAnyStep - 1) / kAnyStep;
    int split = 1;
    while (split < 8 && (int64_t)tn * tm * split * 2 <= 3 * sm_count() && steps / (split * 2) >= 2) split *= 2;
    ICX_CUDA(launch_pdl_cluster(scaled_tile_kernel<T>, dim3(tn * split, tm), dim3(256), 0, s, (unsigned)split, p, split));
    return ICX_OK;
  }
  if (p.M <= 16) return launch_stream<T, 16>(s, p);
  if (p.M <= 32) return launch_stream<T, 32>(s, p);
  // 33 to 128 tokens: the other way round where K is short or hardly shared out
  // (K, N; rows / stream, us: 128 tokens 1472, 768: 6.9 / 10.0; 4096, 14336: 18.2 /
  // 20.9; 8192, 1024: 15.4 / 8.4; 100 tokens 4096, 4096: 11.1 / 9.2; 64 tokens 768,
  // 768: 5.2 / 6.9; 4096, 4096: 10.5 / 7.3)
  if (p.M <= 64 && p.K > 8 * kStep) return launch_stream<T, 64>(s, p);
  if (p.M > 64 && p.M <= 128 && stream_split(p) >= 4) return launch_stream<T, 128>(s, p);
  const int sms = sm_count();
  const long nm = (p.M + kRows - 1) / kRows;
  const int pairs = p.M >= 1024 && p.N > 128 ? max_pairs<T, 256>() : 0;
  // the kernel whose busiest CTA does the least: tiles per CTA x columns of a
  // tile (plus what a tile costs beside its columns); pairs move half the
  // weight bytes per product and win where they keep all SMs busy
  const long c1 = (nm * ((p.N + 127) / 128) + sms - 1) / sms * (128 + 64);
  const long c2 = (nm * ((p.N + 255) / 256) + sms - 1) / sms * (256 + 64);
  const long cp = pairs ? (((nm + 1) / 2) * ((p.N + 255) / 256) + pairs - 1) / pairs * (256 + 32) : c1 + c2;
  if (cp <= c1 && cp <= c2) return launch_rows<T, 256, 2>(s, p, pairs);
  return c2 <= c1 ? launch_rows<T, 256, 1>(s, p, sms) : launch_rows<T, 128, 1>(s, p, sms);
}

}  // namespace icx

using namespace icx;

extern "C" int icx_matmul_integer_scaled(void* stream, const int8_t* d_q, const float* d_q_scale,
                                         const int8_t* d_wt, size_t M, size_t K, size_t N,
                                         const float* d_w_scale, const float* d_bias,
                                         const void* d_residual, int out_type, void* d_out) {
  ICX_REQUIRE(is_float_type(out_type), "MatMulIntegerScaled: output must be Float32, Float16 or BFloat16");
  ICX_REQUIRE(K <= ICX_SCALED_MAX_K, "MatMulIntegerScaled: K %zu above %d, where the s32 sum could wrap", K,
              ICX_SCALED_MAX_K);
  ICX_REQUIRE(M <= 65535ull * 64 && N < (1ull << 22),   // tiles of 64 tokens in grid.y
              "MatMulIntegerScaled: shape too large");
  if (M == 0 || N == 0) return ICX_OK;
  ICX_REQUIRE(d_out && d_q_scale && d_w_scale && (K == 0 || (d_q && d_wt)),
              "MatMulIntegerScaled: null operand");
  const ScaledArgs a{d_q, d_q_scale, d_wt, (int)M, (int)K, (int)N, d_w_scale, d_bias, d_residual, d_out};
  int rc = ICX_OK;
  ICX_FLOAT_DISPATCH(out_type, rc = launch_scaled<T>(as_stream(stream), a));
  return rc;
}
