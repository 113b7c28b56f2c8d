// Masked attention for many queries: bf16, head_dim 128.
#include "p3d_masked_fmha.cuh"

namespace p3d {
int masked_tiles_bf16_128(p3d_ctx *ctx, const MaskedParams &p, int dtype) { return masked_tiles<__nv_bfloat16, 128>(ctx, p, dtype); }
}  // namespace p3d
