// Rotary positions of packed heads.
//
// The pair (a, b) of a head at position p turns by the angle p f_i:
//   a' = A (a cos - b sin),  b' = A (a sin + b cos)
// with the pair's elements i and i + rot/2 (half layout) or 2i and 2i + 1
// (interleaved); elements from rot on are copied.  The angle is held in turns:
// t = p (f_i / 2 pi) in 64 bits, t - rint(t) rounded to f32 (at most 2^-25
// turns off, 2e-7 rad, whatever the position), then sincospif.
//
// Bound by HBM: the rows are read and written once, and the rot/2 angles of a
// token are computed once for all of its heads, into shared memory.
#include <algorithm>

#include "p3d_common.cuh"

namespace p3d {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxRotDim = 512;

struct RotaryParams {
    const void *x;
    int64_t ldx;
    void *out;
    int64_t ldo;
    int64_t n;
    const int32_t *positions;  // or null: offset + row
    int64_t offset;
    const double *freqs;  // [half]
    float amplitude;
    int heads, dim, half;
    int tokens;  // per block
};

template <typename T, int VEC>
struct Vec {
    float v[VEC];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC * sizeof(T) == 16) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    v[i] = __uint_as_float(w[i]);
                } else {
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
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (VEC * sizeof(T) == 16) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4)
                    w[i] = __float_as_uint(v[i]);
                else
                    w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
            }
            *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) p[i] = from_f32<T>(v[i]);
        }
    }
};

// An item is VEC pairs of one head: two vectors half apart (half layout) or
// 2 VEC consecutive elements (interleaved); then the copied elements, 2 VEC an
// item.  Every item reads all of its elements before it writes them, so out
// may be x itself.
template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryParams p) {
    extern __shared__ float2 table[];  // [tokens][half] (cos, sin) times the amplitude
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens;
    const int nt = static_cast<int>(min(static_cast<int64_t>(p.tokens), p.n - t0));
    for (int e = threadIdx.x; e < nt * p.half; e += kRotThreads) {
        const int64_t row = t0 + e / p.half;
        const double pos = static_cast<double>(p.positions ? p.positions[row] : p.offset + row);
        const double turns = pos * (__ldg(p.freqs + e % p.half) * 0.15915494309189533577);
        float s, c;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
        table[e] = make_float2(p.amplitude * c, p.amplitude * s);
    }
    __syncthreads();
    const int turned = p.half / VEC;                                    // items of turned pairs per head
    const int rest = p.dim - 2 * p.half;                                // copied elements per head
    const int iph = turned + (rest + 2 * VEC - 1) / (2 * VEC);          // items per head
    const int ipt = iph * p.heads;                                      // per token
    for (int e = threadIdx.x; e < nt * ipt; e += kRotThreads) {
        const int tok = e / ipt, in = e % ipt, head = in / iph, i = in % iph;
        const T *xr = static_cast<const T *>(p.x) + (t0 + tok) * p.ldx + static_cast<int64_t>(head) * p.dim;
        T *yr = static_cast<T *>(p.out) + (t0 + tok) * p.ldo + static_cast<int64_t>(head) * p.dim;
        if (i < turned) {
            const float2 *cs = table + tok * p.half + i * VEC;
            const int ia = HALF ? i * VEC : 2 * i * VEC, ib = HALF ? ia + p.half : ia + VEC;
            Vec<T, VEC> a, b;
            a.load(xr + ia);
            b.load(xr + ib);
            if constexpr (HALF) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float u = a.v[j], w = b.v[j];
                    a.v[j] = u * cs[j].x - w * cs[j].y;
                    b.v[j] = u * cs[j].y + w * cs[j].x;
                }
            } else if constexpr (VEC == 1) {
                const float u = a.v[0], w = b.v[0];
                a.v[0] = u * cs[0].x - w * cs[0].y;
                b.v[0] = u * cs[0].y + w * cs[0].x;
            } else {
#pragma unroll
                for (int j = 0; j < VEC / 2; ++j) {
                    const float u = a.v[2 * j], w = a.v[2 * j + 1];
                    a.v[2 * j] = u * cs[j].x - w * cs[j].y;
                    a.v[2 * j + 1] = u * cs[j].y + w * cs[j].x;
                    const float u2 = b.v[2 * j], w2 = b.v[2 * j + 1];
                    b.v[2 * j] = u2 * cs[VEC / 2 + j].x - w2 * cs[VEC / 2 + j].y;
                    b.v[2 * j + 1] = u2 * cs[VEC / 2 + j].y + w2 * cs[VEC / 2 + j].x;
                }
            }
            a.store(yr + ia);
            b.store(yr + ib);
        } else {
            const int c0 = 2 * p.half + (i - turned) * 2 * VEC;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = c0 + j * VEC;
                if (c >= p.dim) break;
                Vec<T, VEC> a;
                a.load(xr + c);
                a.store(yr + c);
            }
        }
    }
}

template <typename T, int VEC>
int launch_rotary(p3d_ctx *ctx, RotaryParams p, int layout) {
    // about 1024 items a block, so the angles are spread over few tokens
    const int ipt = p.heads * ((p.dim / 2 + VEC - 1) / VEC);
    p.tokens = std::max(1, std::min({1024 / std::max(ipt, 1), 4096 / p.half, 64}));
    const size_t smem = sizeof(float2) * p.tokens * p.half;
    const unsigned grid = static_cast<unsigned>(ceil_div(p.n, p.tokens));
    if (layout == P3D_ROTARY_HALF)
        rotary_kernel<T, VEC, true><<<grid, kRotThreads, smem, ctx->stream>>>(p);
    else
        rotary_kernel<T, VEC, false><<<grid, kRotThreads, smem, ctx->stream>>>(p);
    return check_launch(ctx, "rotary");
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" int p3d_rotary(p3d_ctx *ctx, const void *x, int64_t ldx, int64_t n, int heads, int head_dim, int rot_dim,
                          int layout, const int32_t *positions, int64_t position_offset, const double *freqs,
                          float amplitude, void *out, int64_t ldo, int dtype) {
    if (!ctx) return P3D_ERR_INVALID;
    P3D_REQUIRE(ctx, x && out && freqs, "p3d_rotary: null pointer");
    P3D_REQUIRE(ctx, dtype == P3D_F32 || is_16bit(dtype), "p3d_rotary: dtype must be f32, bf16 or f16");
    P3D_REQUIRE(ctx, layout == P3D_ROTARY_HALF || layout == P3D_ROTARY_INTERLEAVED, "p3d_rotary: unknown layout");
    P3D_REQUIRE(ctx, heads > 0 && heads < 65536 && head_dim > 0 && head_dim <= kMaxRotDim,
                "p3d_rotary: bad heads or head_dim (at most 512)");
    P3D_REQUIRE(ctx, rot_dim >= 2 && rot_dim % 2 == 0 && rot_dim <= head_dim,
                "p3d_rotary: rot_dim must be even, at least 2 and at most head_dim");
    const int64_t width = static_cast<int64_t>(heads) * head_dim;
    P3D_REQUIRE(ctx, n >= 0 && n < (int64_t(1) << 31), "p3d_rotary: bad row count");
    P3D_REQUIRE(ctx, n <= 1 || (ldx >= width && ldo >= width), "p3d_rotary: leading dimension below heads * head_dim");
    const size_t es = dtype_size(dtype);
    const uintptr_t xa = reinterpret_cast<uintptr_t>(x), oa = reinterpret_cast<uintptr_t>(out);
    P3D_REQUIRE(ctx, xa % es == 0 && oa % es == 0 && reinterpret_cast<uintptr_t>(freqs) % 8 == 0 &&
                         reinterpret_cast<uintptr_t>(positions) % 4 == 0,
                "p3d_rotary: a pointer is not aligned to its elements");
    if (n == 0) return P3D_OK;
    const uintptr_t xe = xa + ((n - 1) * ldx + width) * es, oe = oa + ((n - 1) * ldo + width) * es;
    P3D_REQUIRE(ctx, (xa == oa && (ldx == ldo || n == 1)) || xe <= oa || oe <= xa || (ldx == ldo && n > 1 &&
                         (xa > oa ? xa - oa : oa - xa) % (ldx * es) >= width * es &&
                         (xa > oa ? xa - oa : oa - xa) % (ldx * es) <= (ldx - width) * es),
                "p3d_rotary: out must be x itself or not overlap it");
    RotaryParams p{x, ldx, out, ldo, n, positions, position_offset, freqs, amplitude, heads, head_dim, rot_dim / 2, 1};
    DeviceGuard on(ctx->device);
    // 16-byte vectors where rows, heads and both elements of the pairs allow
    // them, single elements elsewhere
    const int vec = static_cast<int>(16 / es);
    const bool aligned = (xa | oa) % 16 == 0 && (n == 1 || (ldx % vec == 0 && ldo % vec == 0)) && head_dim % vec == 0 &&
                         p.half % vec == 0;
    if (dtype == P3D_F32) return aligned ? launch_rotary<float, 4>(ctx, p, layout) : launch_rotary<float, 1>(ctx, p, layout);
    if (dtype == P3D_BF16)
        return aligned ? launch_rotary<__nv_bfloat16, 8>(ctx, p, layout) : launch_rotary<__nv_bfloat16, 1>(ctx, p, layout);
    return aligned ? launch_rotary<__half, 8>(ctx, p, layout) : launch_rotary<__half, 1>(ctx, p, layout);
}
