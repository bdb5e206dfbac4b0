// Per-token quantisation: symmetric int8 with one scale per row.
//
//   s = f32(max|x| / 127);  q = clamp(rte(x / s), -127, 127)
//
// the quotient exact before it is rounded.  Bound by HBM: the row is read
// once into registers (up to 64 values per thread, 16-byte loads all in
// flight), reduced, and written from there.  8192 rows of 8192 bf16: 40.5 us,
// 5.0 TB/s (floor 31.1 at 6.46 TB/s); one row of 768: 1.3 us.
//
// |x| is compared by its bits: a NaN's are above infinity's, whose are above
// every finite value's, so one integer maximum also finds rows that hold
// either.
//
// Rounding: u = x * f32(1/s) is off by less than 1.6e-5 (two roundings of
// 2^-24 at |u| <= 127), so rte(u) is the code unless u is within 1e-4 of a
// half; those (2e-4 of all values, and every exact tie) compare x with the
// midpoint (k + 1/2) s in 64 bits, where both are exact.
#include "capi.cuh"
#include "common.cuh"
#include "floats.cuh"

namespace icx {

constexpr uint32_t kInfBits = 0x7f800000u;
constexpr float kRound = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer (half to even)

__device__ __forceinline__ float token_scale(uint32_t peak_bits) {
  return peak_bits >= kInfBits ? __uint_as_float(0x7fc00000u)
                               : __fdiv_rn(__uint_as_float(peak_bits), 127.0f);
}

// The code of x for a scale whose reciprocal is finite, given u = x / s
// within 1e-4 of a half.
__device__ __noinline__ int code_near_half(float x, float s, float u) {
  const float k = floorf(u);
  const double d = (double)x - ((double)k + 0.5) * (double)s;
  return d > 0.0 ? (int)k + 1 : d < 0.0 ? (int)k : 2 * (int)rintf(0.5f * k + 0.25f);
}

// N codes as bytes.
template <int N>
__device__ __forceinline__ void token_codes(const float (&x)[N], float s, float inv, uint32_t (&out)[(N + 3) / 4]) {
  uint32_t c[N];
  if (s >= 1e-36f) {
    float worst = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float u = x[i] * inv, r = __fadd_rn(u, kRound);
      worst = fmaxf(worst, fabsf(u - __fsub_rn(r, kRound)));
      c[i] = __float_as_uint(r);
    }
    if (worst > 0.4999f) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float u = x[i] * inv;
        if (fabsf(u - rintf(u)) > 0.4999f) c[i] = (uint32_t)code_near_half(x[i], s, u);
      }
    }
  } else {   // 0, NaN, or too small for its reciprocal
#pragma unroll
    for (int i = 0; i < N; ++i)
      c[i] = s > 0.0f ? (uint32_t)max(-127, min(127, __double2int_rn((double)x[i] / (double)s))) : 0u;
  }
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    if (N >= 4)
      out[i / 4] = __byte_perm(__byte_perm(c[i], c[(i + 1) % N], 0x0040), __byte_perm(c[(i + 2) % N], c[(i + 3) % N], 0x0040), 0x5410);
    else
      out[0] = c[0];
  }
}

// Largest |x| by its bits: f32 bits, or for 16-bit types the larger of both
// half words, which peak_f32_bits turns into the f32 value's.
template <typename T, int E>
__device__ __forceinline__ uint32_t vec_peak(const Vec<T, E>& v) {
  uint32_t p = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < E; ++i) p = max(p, __float_as_uint(fabsf(v.v[i])));
  } else if constexpr (E == 1) {
    p = *reinterpret_cast<const uint16_t*>(&v.v[0]) & 0x7fffu;
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    p = max(m >> 16, m & 0xffffu);
  }
  return p;
}
template <typename T>
__device__ __forceinline__ uint32_t peak_f32_bits(uint32_t p) {
  if constexpr (sizeof(T) == 4) return p;
  const uint16_t h = (uint16_t)p;
  return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&h)));
}

// W warps per row; a thread holds V accesses of E values (E = 16 bytes' worth,
// or 1 where the row cannot be read in 16-byte pieces).
template <typename T, int W, int V, int E>
__global__ void __launch_bounds__(256)
    quantize_row_kernel(const T* __restrict__ x, int rows, int cols, size_t stride, int8_t* __restrict__ q,
                        float* __restrict__ scale) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t red[8];
  constexpr int kThreads = 32 * W;
  const int t = threadIdx.x % kThreads;
  const int row = blockIdx.x * (256 / kThreads) + threadIdx.x / kThreads;
  const bool here = row < rows;
  const T* src = x + (size_t)(here ? row : 0) * stride;
  Vec<T, E> v[V];   // as they are: half the registers of their f32 values
  uint32_t peak = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int at = (i * kThreads + t) * E;
    v[i] = Vec<T, E>{};
    if (here && at < cols) v[i] = *reinterpret_cast<const Vec<T, E>*>(src + at);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) peak = max(peak, vec_peak(v[i]));
  peak = peak_f32_bits<T>(peak);
  peak = __reduce_max_sync(0xffffffffu, peak);
  if (W > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = peak;
    __syncthreads();
    const int w0 = threadIdx.x / kThreads * W;
#pragma unroll
    for (int i = 0; i < W; ++i) peak = max(peak, red[w0 + i]);
  }
  if (!here) return;
  const float s = token_scale(peak), inv = __frcp_rn(s);
  if (t == 0) scale[row] = s;
  int8_t* out = q + (size_t)row * cols;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int at = (i * kThreads + t) * E;
    if (at >= cols) break;
    uint32_t c[(E + 3) / 4];
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = to_f32(v[i].v[e]);
    token_codes<E>(f, s, inv, c);
    if (E == 8) *reinterpret_cast<uint2*>(out + at) = make_uint2(c[0], c[(E + 3) / 4 - 1]);
    else if (E == 4) *reinterpret_cast<uint32_t*>(out + at) = c[0];
    else out[at] = (int8_t)c[0];
  }
}

// Rows wider than the registers of a CTA: two passes over the row, the second
// from L2.
template <typename T>
__global__ void __launch_bounds__(1024)
    quantize_wide_kernel(const T* __restrict__ x, int cols, size_t stride, int8_t* __restrict__ q,
                         float* __restrict__ scale, int vec) {
  pdl_wait();
  pdl_trigger();
  __shared__ uint32_t red[32];
  const T* src = x + (size_t)blockIdx.x * stride;
  int8_t* out = q + (size_t)blockIdx.x * cols;
  const int n4 = vec ? cols / 4 : 0;
  uint32_t peak = 0;
  float v[4];
  for (int i = threadIdx.x; i < n4; i += 1024) {
    load_f32<T, 4>(src + 4 * i, v, true);
#pragma unroll
    for (int e = 0; e < 4; ++e) peak = max(peak, __float_as_uint(fabsf(v[e])));
  }
  for (int i = 4 * n4 + threadIdx.x; i < cols; i += 1024) peak = max(peak, __float_as_uint(fabsf(to_f32(src[i]))));
  peak = __reduce_max_sync(0xffffffffu, peak);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = peak;
  __syncthreads();
  peak = __reduce_max_sync(0xffffffffu, red[threadIdx.x & 31]);
  const float s = token_scale(peak), inv = __frcp_rn(s);
  if (threadIdx.x == 0) scale[blockIdx.x] = s;
  uint32_t c[1];
  for (int i = threadIdx.x; i < n4; i += 1024) {
    load_f32<T, 4>(src + 4 * i, v, true);
    token_codes<4>(v, s, inv, c);
    *reinterpret_cast<uint32_t*>(out + 4 * i) = c[0];
  }
  for (int i = 4 * n4 + threadIdx.x; i < cols; i += 1024) {
    const float one[1] = {to_f32(src[i])};
    token_codes<1>(one, s, inv, c);
    out[i] = (int8_t)c[0];
  }
}

template <typename T, int W, int V, int E>
static cudaError_t launch_rows(cudaStream_t s, const T* x, int rows, int cols, size_t stride, int8_t* q, float* scale) {
  const int per = 8 / W;
  return launch_pdl(quantize_row_kernel<T, W, V, E>, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, x,
                    rows, cols, stride, q, scale);
}

// The fewest warps that hold a row at V accesses per thread: a row's loads are
// all in flight, and narrow rows share a CTA.
template <typename T, int E>
static cudaError_t launch_quantize(cudaStream_t s, const T* x, int rows, int cols, size_t stride, int8_t* q,
                                   float* scale, int vec) {
  constexpr int V = E == 1 ? 16 : 4;
  const int n = (cols + E - 1) / E;   // accesses per row
  if (n <= 32 * V / 4) return launch_rows<T, 1, V / 4, E>(s, x, rows, cols, stride, q, scale);
  if (n <= 32 * V) return launch_rows<T, 1, V, E>(s, x, rows, cols, stride, q, scale);
  if (n <= 64 * V) return launch_rows<T, 2, V, E>(s, x, rows, cols, stride, q, scale);
  if (n <= 128 * V) return launch_rows<T, 4, V, E>(s, x, rows, cols, stride, q, scale);
  if (n <= 256 * V) return launch_rows<T, 8, V, E>(s, x, rows, cols, stride, q, scale);
  if (n <= 512 * V) return launch_rows<T, 8, 2 * V, E>(s, x, rows, cols, stride, q, scale);
  return launch_pdl(quantize_wide_kernel<T>, dim3((unsigned)rows), dim3(1024), 0, s, x, cols, stride, q, scale, vec);
}

}  // namespace icx

using namespace icx;

extern "C" int icx_quantize_per_token(void* stream, const void* d_x, int x_type, size_t rows,
                                      size_t cols, size_t row_stride, int8_t* d_q, float* d_scale) {
  ICX_REQUIRE(is_float_type(x_type), "QuantizePerToken: input must be Float32, Float16 or BFloat16");
  ICX_REQUIRE(rows < (1ull << 31) && cols < (1ull << 30), "QuantizePerToken: shape too large");
  ICX_REQUIRE(rows <= 1 || row_stride >= cols, "QuantizePerToken: row stride %zu below the row length %zu",
              row_stride, cols);
  if (rows == 0) return ICX_OK;
  ICX_REQUIRE(d_scale && (cols == 0 || (d_x && d_q)), "QuantizePerToken: null pointer");
  cudaStream_t s = as_stream(stream);
  const size_t e = float_bytes(x_type), per16 = 16 / e;
  const bool vec = cols % per16 == 0 && (rows == 1 || row_stride % per16 == 0) &&
                   (reinterpret_cast<uintptr_t>(d_x) & 15) == 0 && (reinterpret_cast<uintptr_t>(d_q) & 7) == 0;
  ICX_FLOAT_DISPATCH(x_type, {
    const T* x = static_cast<const T*>(d_x);
    constexpr int E = 16 / sizeof(T);
    if (vec) ICX_CUDA((launch_quantize<T, E>(s, x, (int)rows, (int)cols, row_stride, d_q, d_scale, 1)));
    else ICX_CUDA((launch_quantize<T, 1>(s, x, (int)rows, (int)cols, row_stride, d_q, d_scale, 0)));
  });
  return ICX_OK;
}
