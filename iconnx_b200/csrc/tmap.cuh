// Tensor maps of the GEMM kernels, and the device they are launched on.
#pragma once

#include <cuda.h>

#include <cstddef>

namespace icx {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t,
                                  void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled of the driver, or null.
EncodeTiledFn encode_fn();

// K-major byte matrix [rows, K] -> tensor map with a box of box_rows x 128
// bytes and the 128-byte swizzle.
int make_tmap(CUtensorMap* map, const void* base, size_t rows, size_t K, int box_rows);

// SMs of the current device (148 if it cannot be asked).
int sm_count();

}  // namespace icx
