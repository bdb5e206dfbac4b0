// Attention over the quantised K/V cache: kernels for f32 queries.
#include "kv_attention.cuh"

namespace icx {
ICX_ATTEND_INSTANCE(float)
}  // namespace icx
