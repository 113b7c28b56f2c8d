// Quantisation of rows to 8-bit integers, one scale for each row.
//
//   s_i  = max(fl32(max_j |x_ij| / 127), 2^-126)
//   q_ij = rint(x_ij / s_i)          (ties to even, decided exactly)
//
// The result does not depend on how the quotient is rounded on its way: q is
// first rint(fl(x * fl(1/s))), which is off by at most one, and only where
// x / s lies within 2^-15 of a half.  The remainder r = x - q s is one FMA.
// It is a multiple of ulp(s) / 2 (q = 0 gives x itself, else |x| > s / 4), so
// it is exact while |r| < 2^e, s in [2^e, 2^(e+1)); beyond, 2|r| > s holds
// before and after its rounding.  Hence 2|r| >= s tells the elements that must
// move, or sit on a tie, from all others.  Halves are no rare event: half of
// the row's largest magnitude is 63.5 s.
// A row holding an infinity or a NaN gets the scale NaN and zeros, so that
// every product with it is NaN rather than a plausible number.
//
// Bound by HBM: each element is read once (2 or 4 bytes) and one byte is
// written; the row stays in registers between the two uses.
#include "p3d_common.cuh"

namespace p3d {
namespace {

constexpr int kQuantThreads = 256;

// Row maximum of |x| as the bits of an f32 (ordered like the values, with
// NaN above infinity above every finite value).
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct RowScale {
    float s, inv;
    bool bad;  // the row holds an infinity or a NaN
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    r.bad = amax_bits >= 0x7f800000u;
    r.s = fmaxf(__fdiv_rn(__uint_as_float(amax_bits), 127.0f), 1.17549435e-38f);
    r.inv = __frcp_rn(r.s);
    return r;
}

__device__ __forceinline__ int quant1(float x, const RowScale &rs) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
    const float qf = __fsub_rn(__fadd_rn(__fmul_rn(x, rs.inv), kMagic), kMagic);
    const float r = fmaf(-qf, rs.s, x);
    int q = static_cast<int>(qf);
    const float r2 = 2.0f * fabsf(r);
    if (r2 >= rs.s) {  // rare: the neighbour is nearer, or a tie
        const int other = q + (r > 0.0f ? 1 : -1);
        if (r2 > rs.s || (q & 1)) q = other;
    }
    return q;
}

// VEC elements of type T at p, as floats.
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[VEC]) {
    if constexpr (VEC * sizeof(T) == 16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
        if constexpr (sizeof(T) == 4) {
            v[0] = __uint_as_float(u.x);
            v[1] = __uint_as_float(u.y);
            v[2] = __uint_as_float(u.z);
            v[3] = __uint_as_float(u.w);
        } else {
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack2<T>(w[i]);
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = to_f32(p[i]);
    }
}

template <int VEC>
__device__ __forceinline__ void store_q(int8_t *p, const float (&v)[VEC], const RowScale &rs, int n, bool wide) {
    uint32_t w[(VEC + 3) / 4] = {};
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        w[i / 4] |= (static_cast<uint32_t>(rs.bad ? 0 : quant1(v[i], rs)) & 0xffu) << (8 * (i % 4));
    if (wide && n == VEC) {
        if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        if constexpr (VEC == 4) *reinterpret_cast<uint32_t *>(p) = w[0];
        if constexpr (VEC == 1) *p = static_cast<int8_t>(w[0]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < n) p[i] = static_cast<int8_t>(w[i / 4] >> (8 * (i % 4)));
    }
}

// TPR threads per row (32, or the whole block), each holding up to HOLD
// vectors of the row in registers; a longer row is read a second time.
template <typename T, int VEC, int TPR, int HOLD>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int64_t m, int k, int8_t *__restrict__ q, int64_t ldq,
                         float *__restrict__ scale, bool wide) {
    const int lane = threadIdx.x % TPR;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kQuantThreads / TPR) + threadIdx.x / TPR;
    if (TPR == 32 && row >= m) return;  // whole warps
    const T *xr = x + row * ldx;
    const int nv = (k + VEC - 1) / VEC;
    uint32_t amax = 0;
    float v[HOLD][VEC];
    auto load = [&](int i, float(&d)[VEC]) {
        if (VEC == 1 || (i + 1) * VEC <= k) {
            load_vec<T, VEC>(xr + static_cast<int64_t>(i) * VEC, d);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) d[e] = i * VEC + e < k ? to_f32(xr[static_cast<int64_t>(i) * VEC + e]) : 0.0f;
        }
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        const int i = lane + h * TPR;
        if (i < nv) load(i, v[h]);
    }
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        if (lane + h * TPR < nv) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) amax = max(amax, abs_bits(v[h][e]));
        }
    }
    for (int i = lane + HOLD * TPR; i < nv; i += TPR) {
        float d[VEC];
        load(i, d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) amax = max(amax, abs_bits(d[e]));
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if constexpr (TPR > 32) {
        __shared__ uint32_t part[TPR / 32];
        if (lane % 32 == 0) part[lane / 32] = amax;
        __syncthreads();
        amax = part[0];
#pragma unroll
        for (int w = 1; w < TPR / 32; ++w) amax = max(amax, part[w]);
    }
    const RowScale rs = row_scale(amax);
    if (lane == 0) scale[row] = rs.bad ? __int_as_float(0x7fc00000) : rs.s;
    int8_t *qr = q + row * ldq;
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        const int i = lane + h * TPR;
        if (i < nv) store_q<VEC>(qr + static_cast<int64_t>(i) * VEC, v[h], rs, min(VEC, k - i * VEC), wide);
    }
    for (int i = lane + HOLD * TPR; i < nv; i += TPR) {
        float d[VEC];
        load(i, d);
        store_q<VEC>(qr + static_cast<int64_t>(i) * VEC, d, rs, min(VEC, k - i * VEC), wide);
    }
}

template <typename T, int VEC>
int launch_quantize(p3d_ctx *ctx, const void *x, int64_t ldx, int64_t m, int64_t k, int8_t *q, int64_t ldq,
                    float *scale) {
    const T *xt = static_cast<const T *>(x);
    const bool wide = (reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(ldq)) % VEC == 0;
    const int64_t nv = ceil_div(k, VEC);
    const int kk = static_cast<int>(k);
    // A warp holds a row of 32 x 4 vectors; longer rows take a block.
    if (nv <= 32 * 4)
        quantize_rows_kernel<T, VEC, 32, 4><<<static_cast<unsigned>(ceil_div(m, kQuantThreads / 32)), kQuantThreads, 0, ctx->stream>>>(
            xt, ldx, m, kk, q, ldq, scale, wide);
    else
        quantize_rows_kernel<T, VEC, kQuantThreads, 4><<<static_cast<unsigned>(m), kQuantThreads, 0, ctx->stream>>>(
            xt, ldx, m, kk, q, ldq, scale, wide);
    return check_launch(ctx, "quantize_rows");
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" int p3d_quantize_rows(p3d_ctx *ctx, const void *x, int64_t ldx, int64_t m, int64_t k, int dtype, int8_t *q,
                                 int64_t ldq, float *scale) {
    if (!ctx) return P3D_ERR_INVALID;
    P3D_REQUIRE(ctx, x && q && scale, "p3d_quantize_rows: null pointer");
    P3D_REQUIRE(ctx, dtype == P3D_F32 || is_16bit(dtype), "p3d_quantize_rows: dtype must be f32, bf16 or f16");
    P3D_REQUIRE(ctx, m >= 0 && m < (int64_t(1) << 31) && k > 0 && k < (int64_t(1) << 30), "p3d_quantize_rows: bad shape");
    P3D_REQUIRE(ctx, (ldx >= k && ldq >= k) || m <= 1, "p3d_quantize_rows: leading dimension below k");
    P3D_REQUIRE(ctx,
                reinterpret_cast<uintptr_t>(x) % dtype_size(dtype) == 0 && reinterpret_cast<uintptr_t>(scale) % 4 == 0,
                "p3d_quantize_rows: x or scale not aligned to its elements");
    if (m == 0) return P3D_OK;
    DeviceGuard on(ctx->device);
    // 16-byte vectors where every row starts on a 16-byte boundary, single elements elsewhere
    const bool aligned = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (m == 1 || ldx * dtype_size(dtype) % 16 == 0);
    if (dtype == P3D_F32)
        return aligned ? launch_quantize<float, 4>(ctx, x, ldx, m, k, q, ldq, scale)
                       : launch_quantize<float, 1>(ctx, x, ldx, m, k, q, ldq, scale);
    if (dtype == P3D_BF16)
        return aligned ? launch_quantize<__nv_bfloat16, 8>(ctx, x, ldx, m, k, q, ldq, scale)
                       : launch_quantize<__nv_bfloat16, 1>(ctx, x, ldx, m, k, q, ldq, scale);
    return aligned ? launch_quantize<__half, 8>(ctx, x, ldx, m, k, q, ldq, scale)
                   : launch_quantize<__half, 1>(ctx, x, ldx, m, k, q, ldq, scale);
}
