// f32 / f16 / bf16 element access and rounding for the decoder-layer kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/iconnx_b200.h"

namespace icx {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements in one vector access (p aligned to N * sizeof(T),
// at most 16 bytes).
template <typename T, int N>
struct alignas(N * sizeof(T)) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&x)[N], bool vec) {
  if (vec) {
    const Vec<T, N> u = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(u.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(p[i]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&x)[N]) {
  Vec<T, N> u;
#pragma unroll
  for (int i = 0; i < N; ++i) u.v[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Vec<T, N>*>(p) = u;
}

// Pairs of f32 in one instruction each.  A product and a following sum may be
// contracted to a fused multiply-add.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

inline bool is_float_type(int t) { return t == ICX_F32 || t == ICX_F16 || t == ICX_BF16; }
inline size_t float_bytes(int t) { return t == ICX_F32 ? 4 : 2; }

}  // namespace icx

// Runs the statement with T = the element type of code `type`.
#define ICX_FLOAT_DISPATCH(type, ...)            \
  do {                                           \
    if ((type) == ICX_F32) {                     \
      using T = float;                           \
      __VA_ARGS__;                               \
    } else if ((type) == ICX_F16) {              \
      using T = __half;                          \
      __VA_ARGS__;                               \
    } else {                                     \
      using T = __nv_bfloat16;                   \
      __VA_ARGS__;                               \
    }                                            \
  } while (0)
