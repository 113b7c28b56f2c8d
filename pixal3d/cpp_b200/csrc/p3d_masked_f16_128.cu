// Masked attention for many queries: f16, head_dim 128.
#include "p3d_masked_fmha.cuh"

namespace p3d {
int masked_tiles_f16_128(p3d_ctx *ctx, const MaskedParams &p, int dtype) { return masked_tiles<__half, 128>(ctx, p, dtype); }
}  // namespace p3d
