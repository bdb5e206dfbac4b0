// Attention over the quantised K/V cache: kernels for bf16 queries.
#include "kv_attention.cuh"

namespace icx {
ICX_ATTEND_INSTANCE(__nv_bfloat16)
}  // namespace icx
