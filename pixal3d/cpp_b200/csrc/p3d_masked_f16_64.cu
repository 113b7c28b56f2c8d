// Masked attention for many queries: f16, head_dim 64.
#include "p3d_masked_fmha.cuh"

namespace p3d {
int masked_tiles_f16_64(p3d_ctx *ctx, const MaskedParams &p, int dtype) { return masked_tiles<__half, 64>(ctx, p, dtype); }
}  // namespace p3d
