// Int8 linear layers with a scale per token and per output channel:
// per-token quantisation and the scaled int8 product.
#include "capi.cuh"
#include "common.cuh"
#include "floats.cuh"

namespace icx {

// ------------------------------------------------- per-token quantisation
// s = f32(max|x| / 127); q = clamp(rte(x / s), -127, 127), the quotient exact
// before it is rounded.  |x| is compared by its bits: a NaN's are above
// infinity's, whose are above every finite value's, so one integer maximum
// also finds rows that hold either.
constexpr uint32_t kInfBits = 0x7f800000u;

__device__ __forceinline__ float token_scale(uint32_t peak_bits) {
  return peak_bits >= kInfBits ? __uint_as_float(0x7fc00000u)
                               : __fdiv_rn(__uint_as_float(peak_bits), 127.0f);
}

__device__ __forceinline__ int quantize_exact(float x, float s) {
  const double t = (double)x / (double)s;
  return max(-127, min(127, __double2int_rn(t)));
}

template <typename T>
__global__ void __launch_bounds__(256)
    quantize_token_kernel(const T* __restrict__ x, size_t cols, size_t stride, int8_t* __restrict__ q,
                          float* __restrict__ scale) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t red[8];
  const T* row = x + (size_t)blockIdx.x * stride;
  uint32_t peak = 0;
  for (size_t i = threadIdx.x; i < cols; i += 256) peak = max(peak, __float_as_uint(fabsf(to_f32(row[i]))));
  peak = __reduce_max_sync(0xffffffffu, peak);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = peak;
  __syncthreads();
  peak = red[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) peak = max(peak, red[i]);
  const float s = token_scale(peak);
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
  int8_t* out = q + (size_t)blockIdx.x * cols;
  for (size_t i = threadIdx.x; i < cols; i += 256)
    out[i] = s > 0.0f ? (int8_t)quantize_exact(to_f32(row[i]), s) : (int8_t)0;
}

// ---------------------------------------------------- scaled int8 product
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

template <typename T>
__device__ __forceinline__ float scaled_out(int acc, float sa, float sw, float bias, bool has_bias) {
  const float v = __int2float_rn(acc) * sa;
  return has_bias ? fmaf(v, sw, bias) : v * sw;
}

// Any K and alignment: 64 x 64 outputs per CTA, bytes staged through shared
// memory, four products per dp4a.
template <typename T>
__global__ void __launch_bounds__(256) scaled_tile_kernel(const ScaledArgs p) {
  pdl_wait();
  pdl_trigger();
  __shared__ int sa[64][17], sb[64][17];   // 64 rows of 64 bytes, padded
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 64) {
    for (int i = threadIdx.x; i < 64 * 64; i += 256) {
      const int r = i >> 6, c = i & 63;
      const bool kv = k0 + c < p.K;
      reinterpret_cast<int8_t*>(&sa[r][0])[c] =
          kv && m0 + r < p.M ? p.q[(size_t)(m0 + r) * p.K + k0 + c] : (int8_t)0;
      reinterpret_cast<int8_t*>(&sb[r][0])[c] =
          kv && n0 + r < p.N ? p.wt[(size_t)(n0 + r) * p.K + k0 + c] : (int8_t)0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sa[ty + 16 * i][k], sb[tx + 16 * j][k], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= p.M || n >= p.N) continue;
      const size_t o = (size_t)m * p.N + n;
      float v = scaled_out<T>(acc[i][j], p.q_scale[m], p.w_scale[n], p.bias ? p.bias[n] : 0.0f,
                              p.bias != nullptr);
      if (p.residual) v += to_f32(static_cast<const T*>(p.residual)[o]);
      static_cast<T*>(p.out)[o] = from_f32<T>(v);
    }
}

}  // namespace icx

using namespace icx;

extern "C" int icx_quantize_per_token(void* stream, const void* d_x, int x_type, size_t rows,
                                      size_t cols, size_t row_stride, int8_t* d_q, float* d_scale) {
  ICX_REQUIRE(is_float_type(x_type), "QuantizePerToken: input must be Float32, Float16 or BFloat16");
  ICX_REQUIRE(rows < (1ull << 31) && cols < (1ull << 31), "QuantizePerToken: shape too large");
  ICX_REQUIRE(rows <= 1 || row_stride >= cols, "QuantizePerToken: row stride %zu below the row length %zu",
              row_stride, cols);
  if (rows == 0) return ICX_OK;
  ICX_REQUIRE(d_scale && (cols == 0 || (d_x && d_q)), "QuantizePerToken: null pointer");
  cudaStream_t s = as_stream(stream);
  ICX_FLOAT_DISPATCH(x_type, ICX_CUDA(launch_pdl(quantize_token_kernel<T>, dim3((unsigned)rows), dim3(256), 0, s,
                                                 static_cast<const T*>(d_x), cols, row_stride, d_q, d_scale)));
  return ICX_OK;
}

extern "C" int icx_matmul_integer_scaled(void* stream, const int8_t* d_q, const float* d_q_scale,
                                         const int8_t* d_wt, size_t M, size_t K, size_t N,
                                         const float* d_w_scale, const float* d_bias,
                                         const void* d_residual, int out_type, void* d_out) {
  ICX_REQUIRE(is_float_type(out_type), "MatMulIntegerScaled: output must be Float32, Float16 or BFloat16");
  ICX_REQUIRE(K <= ICX_SCALED_MAX_K, "MatMulIntegerScaled: K %zu above %d, where the s32 sum could wrap", K,
              ICX_SCALED_MAX_K);
  ICX_REQUIRE(M < (1ull << 22) && N < (1ull << 22), "MatMulIntegerScaled: shape too large");
  if (M == 0 || N == 0) return ICX_OK;
  ICX_REQUIRE(d_out && d_q_scale && d_w_scale && (K == 0 || (d_q && d_wt)),
              "MatMulIntegerScaled: null operand");
  ScaledArgs a{d_q, d_q_scale, d_wt, (int)M, (int)K, (int)N, d_w_scale, d_bias, d_residual, d_out};
  cudaStream_t s = as_stream(stream);
  const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
  ICX_FLOAT_DISPATCH(out_type, ICX_CUDA(launch_pdl(scaled_tile_kernel<T>, grid, dim3(256), 0, s, a)));
  return ICX_OK;
}
