// Matrix product of 8-bit integers with scales for each row and channel.
//
//   y[i, j] = act( (float(sum_k x[i, k] w[j, k]) xs[i]) ws[j] + bias[j] )
//
// The sum is exact in 32-bit integers (k <= 131071 keeps 128 * 128 * k below
// 2^31); it is rounded once to f32 (24 bits), then scaled in f32.
#include <algorithm>

#include "p3d_common.cuh"

namespace p3d {
namespace {

struct I8Params {
    const int8_t *x, *w;
    int64_t ldx, ldw;
    const float *xs, *ws, *bias;
    void *out;
    int64_t ldo;
    const float *gate;
    int64_t gate_ld;
    const int32_t *batch_offsets;
    int nbatch;
    int64_t M, N;
    int K;
    int out_dtype;
    int epi;
    int *fault;
};

// GELU, tanh form, to f32 accuracy: x * sigmoid(2 y).
__device__ __forceinline__ float gelu_exact_f(float x) {
    const float y = 0.7978845608028654f * fmaf(0.044715f * x, x * x, x);
    return x / (1.0f + __expf(-2.0f * y));
}

// Activation of one value: 16-bit outputs take the hardware tanh (relative
// error about 2^-11, half a step of f16), f32 outputs the exact forms.
__device__ __forceinline__ float act_f(float v, int epi, int out_dtype) {
    if (epi & P3D_EPI_GELU_TANH) return out_dtype == P3D_F32 ? gelu_exact_f(v) : gelu_tanh_f(v);
    if (epi & P3D_EPI_SILU) return v / (1.0f + __expf(-v));
    return v;
}

__device__ __forceinline__ void store_one(const I8Params &p, int64_t row, int64_t col, float v) {
    if (p.epi & P3D_EPI_RESIDUAL) {
        float g = 1.0f;
        if (p.gate) g = p.gate[static_cast<int64_t>(batch_of_row(p.batch_offsets, p.nbatch, row)) * p.gate_ld + col];
        static_cast<float *>(p.out)[row * p.ldo + col] += g * v;
        return;
    }
    if (p.out_dtype == P3D_F32)
        static_cast<float *>(p.out)[row * p.ldo + col] = v;
    else if (p.out_dtype == P3D_BF16)
        static_cast<__nv_bfloat16 *>(p.out)[row * p.ldo + col] = __float2bfloat16_rn(v);
    else
        static_cast<__half *>(p.out)[row * p.ldo + col] = __float2half_rn(v);
}

// 16 bytes of a row from byte k on; bytes at or past K are zero (and not read).
__device__ __forceinline__ int4 load16(const int8_t *row, int k, int K) {
    if (k + 16 <= K) return __ldg(reinterpret_cast<const int4 *>(row + k));
    uint32_t w[4] = {0, 0, 0, 0};
    for (int i = 0; i < 16 && k + i < K; ++i) w[i / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i % 4));
    return make_int4(w[0], w[1], w[2], w[3]);
}

// Few rows: a warp takes one channel and MR rows, its lanes stride over k.
// Bound by the weights' bytes, which are read once for MR rows.
constexpr int kRowThreads = 256;
template <int MR>
__global__ void __launch_bounds__(kRowThreads) linear_i8_rows_kernel(const I8Params p) {
    const int lane = threadIdx.x & 31;
    const int64_t col = static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
    const int64_t row0 = static_cast<int64_t>(blockIdx.y) * MR;
    if (col >= p.N) return;
    const int rows = static_cast<int>(min(static_cast<int64_t>(MR), p.M - row0));
    const int8_t *wr = p.w + col * p.ldw;
    int acc[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) acc[r] = 0;
    for (int k = lane * 16; k < p.K; k += 512) {
        const int4 b = load16(wr, k, p.K);
#pragma unroll
        for (int r = 0; r < MR; ++r) {
            if (r < rows) {
                const int4 a = load16(p.x + (row0 + r) * p.ldx, k, p.K);
                acc[r] = __dp4a(a.x, b.x, acc[r]);
                acc[r] = __dp4a(a.y, b.y, acc[r]);
                acc[r] = __dp4a(a.z, b.z, acc[r]);
                acc[r] = __dp4a(a.w, b.w, acc[r]);
            }
        }
    }
    const float ws = p.ws[col], bias = p.bias ? p.bias[col] : 0.0f;
#pragma unroll
    for (int r = 0; r < MR; ++r) {
        if (r < rows) {
            const int s = __reduce_add_sync(0xffffffffu, acc[r]);
            if (lane == r) {
                const int64_t row = row0 + r;
                store_one(p, row, col, act_f(fmaf(static_cast<float>(s) * p.xs[row], ws, bias), p.epi, p.out_dtype));
            }
        }
    }
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" int p3d_linear_i8(p3d_ctx *ctx, const int8_t *x, int64_t ldx, const float *x_scale, const int8_t *w,
                             int64_t ldw, const float *w_scale, const float *bias, int64_t m, int64_t n, int64_t k,
                             void *out, int64_t ldo, int out_dtype, int epilogue, const float *gate, int64_t gate_ld,
                             const int32_t *batch_offsets, int nbatch) {
    if (!ctx) return P3D_ERR_INVALID;
    P3D_REQUIRE(ctx, x && x_scale && w && w_scale && out, "p3d_linear_i8: null pointer");
    P3D_REQUIRE(ctx, m >= 0 && n > 0 && k > 0 && m < (int64_t(1) << 31) && n < (int64_t(1) << 31), "p3d_linear_i8: bad shape");
    if (k > 131071)
        return set_error(ctx, P3D_ERR_UNSUPPORTED, "p3d_linear_i8: k above 131071 could overflow the 32-bit sums");
    P3D_REQUIRE(ctx, ldx >= k && ldw >= k && ldx % 16 == 0 && ldw % 16 == 0,
                "p3d_linear_i8: ldx and ldw must be multiples of 16, at least k");
    P3D_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0,
                "p3d_linear_i8: x and w must be 16-byte aligned");
    P3D_REQUIRE(ctx, ldo >= n || m <= 1, "p3d_linear_i8: ldo < n");
    P3D_REQUIRE(ctx, out_dtype == P3D_F32 || is_16bit(out_dtype), "p3d_linear_i8: bad out_dtype");
    P3D_REQUIRE(ctx, reinterpret_cast<uintptr_t>(out) % dtype_size(out_dtype) == 0, "p3d_linear_i8: out not aligned to its elements");
    P3D_REQUIRE(ctx, (epilogue & ~(P3D_EPI_GELU_TANH | P3D_EPI_SILU | P3D_EPI_RESIDUAL)) == 0 &&
                         (epilogue & (P3D_EPI_GELU_TANH | P3D_EPI_SILU)) != (P3D_EPI_GELU_TANH | P3D_EPI_SILU),
                "p3d_linear_i8: at most one activation");
    P3D_REQUIRE(ctx, !(epilogue & P3D_EPI_RESIDUAL) || out_dtype == P3D_F32,
                "p3d_linear_i8: residual epilogue needs f32 out");
    P3D_REQUIRE(ctx, !gate || ((epilogue & P3D_EPI_RESIDUAL) && batch_offsets && nbatch > 0),
                "p3d_linear_i8: gate needs the residual epilogue and batch offsets");
    if (m == 0) return P3D_OK;
    DeviceGuard on(ctx->device);
    I8Params p{x, w, ldx, ldw, x_scale, w_scale, bias, out, ldo, gate, gate_ld, batch_offsets, nbatch,
               m, n, static_cast<int>(k), out_dtype, epilogue, ctx->fault};
    constexpr int MR = 4;
    dim3 grid(static_cast<unsigned>(ceil_div(n, kRowThreads / 32)), static_cast<unsigned>(ceil_div(m, MR)));
    linear_i8_rows_kernel<MR><<<grid, kRowThreads, 0, ctx->stream>>>(p);
    return check_launch(ctx, "linear_i8_rows");
}
