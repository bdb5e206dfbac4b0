// Attention over the quantised K/V cache: kernels for f16 queries.
#include "kv_attention.cuh"

namespace icx {
ICX_ATTEND_INSTANCE(__half)
}  // namespace icx
