// Per-token quantisation: symmetric int8 with one scale per row.
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
