// Rotary positions of packed heads.
//
// The pair (a, b) of a head at position p turns by the angle p f_i:
//   a' = A (a cos - b sin),  b' = A (a sin + b cos)
// with the pair's elements i and i + rot/2 (half layout) or 2i and 2i + 1
// (interleaved); elements from rot on are copied.  The angle is held in turns:
// t = p (f_i / 2 pi) in 64 bits, t - rint(t) rounded to f32, then sincospif: at
// most 2^-25 turns (2e-7 rad) off, and 2^-51 of |t| from the 64-bit roundings,
// which passes that where |t| > 2^26.
//
// Bound by HBM: the rows are read and written once, and the rot/2 angles of a
// token are computed once for all of its heads in a block, into shared memory,
// while the block's first rows are on their way.
//
// Where rows lie on 16-byte boundaries and no pair crosses its vectors (half:
// dim and rot/2 whole vectors; interleaved: dim even), a thread turns vectors
// in registers, four of them in flight.  Everything else goes through shared
// memory: the block's heads are copied there as they lie, turned there and
// copied out, by 16 bytes where rows lie on such boundaries, else by elements.
// 16368 x 32 x 64 f16, 48 of 64 turned: vectors 25.3 us, staged 28.5, staged off
// the boundaries 49.5 (in place 19.5, 26.2 and 40).
#include <algorithm>

#include "p3d_common.cuh"

namespace p3d {
namespace {

constexpr int kRotThreads = 256;
constexpr int kMaxRotDim = 512;

// n / d and n % d for n d < 2^32, d > 1 (a rounded-up reciprocal).
struct Divisor {
    uint32_t d, r;
    explicit Divisor(uint32_t v = 1) : d(v), r(v > 1 ? static_cast<uint32_t>(((uint64_t(1) << 32) + v - 1) / v) : 0) {}
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return d > 1 ? __umulhi(n, r) : n; }
};

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
    int tokens, group;  // tokens and heads of a block
    int items;          // vectors (items) of one token's heads in a block
    Divisor per_token, per_head, by_half;
    int vectors;  // staged kernel: rows and heads' groups lie on 16-byte boundaries
};

// Cosines and sines, times the amplitude, of the block's tokens: [tokens][half].
__device__ __forceinline__ void rotary_table(const RotaryParams &p, float2 *table, int64_t t0, int nt) {
    for (uint32_t e = threadIdx.x; e < static_cast<uint32_t>(nt * p.half); e += kRotThreads) {
        const uint32_t tok = p.by_half.div(e), i = e - tok * p.half;
        const int64_t row = t0 + tok;
        const double pos = static_cast<double>(p.positions ? p.positions[row] : p.offset + row);
        const double turns = pos * (__ldg(p.freqs + i) * 0.15915494309189533577);
        float s, c;
        sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
        table[e] = make_float2(p.amplitude * c, p.amplitude * s);
    }
}

// 16 bytes as elements.
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    float v[N];
    __device__ __forceinline__ explicit Vec(const uint4 &u) {
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
    }
    __device__ __forceinline__ uint4 bits() const {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4)
                w[i] = __float_as_uint(v[i]);
            else
                w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ void turn(float &a, float &b, const float2 &cs) {
    const float u = a, w = b;
    a = u * cs.x - w * cs.y;
    b = u * cs.y + w * cs.x;
}

// Half: an item is the vectors i and i + half of a head, then the copied
// vectors one by one.  Interleaved: an item is one vector of a head.  Every
// item is read before it is written and no other reads it, so out may be x.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryParams p) {
    constexpr int N = Vec<T>::N;
    constexpr int FLY = HALF ? 2 : 4;  // items in flight
    extern __shared__ float2 table[];
    pdl_wait();
    pdl_trigger();
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens;
    const int nt = static_cast<int>(min(static_cast<int64_t>(p.tokens), p.n - t0));
    const int pairs = p.half / N;  // half: items that turn, of a head
    const uint32_t total = static_cast<uint32_t>(nt * p.items);
    for (uint32_t e0 = threadIdx.x; e0 - threadIdx.x < total; e0 += FLY * kRotThreads) {
        uint4 a[FLY], b[HALF ? FLY : 1];
        int64_t at[FLY];
        int tok[FLY], i[FLY];
#pragma unroll
        for (int f = 0; f < FLY; ++f) {
            const uint32_t e = e0 + f * kRotThreads;
            tok[f] = p.tokens > 1 ? p.per_token.div(e) : 0;
            const uint32_t in = e - tok[f] * p.items, head = p.per_head.div(in);
            i[f] = in - head * p.per_head.d;
            const int elem = HALF ? (i[f] < pairs ? i[f] : i[f] + pairs) * N : i[f] * N;
            at[f] = static_cast<int64_t>(head) * p.dim + elem;
            if (e < total) {
                const T *x = static_cast<const T *>(p.x) + (t0 + tok[f]) * p.ldx + at[f];
                a[f] = *reinterpret_cast<const uint4 *>(x);
                if (HALF && i[f] < pairs) b[HALF ? f : 0] = *reinterpret_cast<const uint4 *>(x + p.half);
            }
        }
        if (e0 == threadIdx.x) {
            rotary_table(p, table, t0, nt);
            __syncthreads();
        }
#pragma unroll
        for (int f = 0; f < FLY; ++f) {
            if (e0 + f * kRotThreads >= total) break;
            T *y = static_cast<T *>(p.out) + (t0 + tok[f]) * p.ldo + at[f];
            const float2 *cs = table + tok[f] * p.half;
            if constexpr (HALF) {
                if (i[f] < pairs) {
                    Vec<T> u(a[f]), w(b[f]);
#pragma unroll
                    for (int j = 0; j < N; ++j) turn(u.v[j], w.v[j], cs[i[f] * N + j]);
                    *reinterpret_cast<uint4 *>(y) = u.bits();
                    *reinterpret_cast<uint4 *>(y + p.half) = w.bits();
                } else {
                    *reinterpret_cast<uint4 *>(y) = a[f];
                }
            } else {
                Vec<T> u(a[f]);
                const int first = i[f] * (N / 2);  // pair
#pragma unroll
                for (int j = 0; j < N / 2; ++j)
                    if (first + j < p.half) turn(u.v[2 * j], u.v[2 * j + 1], cs[first + j]);
                *reinterpret_cast<uint4 *>(y) = u.bits();
            }
        }
    }
}

// Any layout: `group` heads of `tokens` tokens through shared memory.
template <typename T, bool HALF>
__global__ void __launch_bounds__(kRotThreads) rotary_staged_kernel(const RotaryParams p) {
    constexpr int N = Vec<T>::N;
    extern __shared__ float2 table[];
    T *rows = reinterpret_cast<T *>(table + ((p.tokens * p.half + 1) & ~1));  // [tokens][group * dim], 16-byte aligned
    pdl_wait();
    pdl_trigger();
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tokens;
    const int nt = static_cast<int>(min(static_cast<int64_t>(p.tokens), p.n - t0));
    const int head0 = blockIdx.y * p.group;
    const int wide = p.group * p.dim;                            // staged elements of a token
    const int width = min(p.group, p.heads - head0) * p.dim;     // of them present
    const int64_t col = static_cast<int64_t>(head0) * p.dim;
    if (p.vectors) {
        for (int tok = 0; tok < nt; ++tok) {
            const T *x = static_cast<const T *>(p.x) + (t0 + tok) * p.ldx + col;
            for (int c = threadIdx.x * N; c < width; c += kRotThreads * N) cp_async16(rows + tok * wide + c, x + c, 16);
        }
        cp_async_commit();
    } else {
        for (int tok = 0; tok < nt; ++tok) {
            const T *x = static_cast<const T *>(p.x) + (t0 + tok) * p.ldx + col;
#pragma unroll 4
            for (int c = threadIdx.x; c < width; c += kRotThreads) rows[tok * wide + c] = x[c];
        }
    }
    rotary_table(p, table, t0, nt);
    cp_async_wait<0>();
    __syncthreads();
    // the pairs are turned where they lie
    const uint32_t pairs = static_cast<uint32_t>(width / p.dim * p.half);
    for (int tok = 0; tok < nt; ++tok) {
        T *from = rows + tok * wide;
        const float2 *cs = table + tok * p.half;
#pragma unroll 4
        for (uint32_t e = threadIdx.x; e < pairs; e += kRotThreads) {
            const uint32_t head = p.by_half.div(e), i = e - head * p.half;
            T *h = from + head * p.dim;
            T &a = HALF ? h[i] : h[2 * i], &b = HALF ? h[i + p.half] : h[2 * i + 1];
            float u = to_f32(a), w = to_f32(b);
            turn(u, w, cs[i]);
            a = from_f32<T>(u);
            b = from_f32<T>(w);
        }
    }
    __syncthreads();
    for (int tok = 0; tok < nt; ++tok) {
        T *y = static_cast<T *>(p.out) + (t0 + tok) * p.ldo + col;
        const T *from = rows + tok * wide;
        if (p.vectors) {
            for (int c = threadIdx.x * N; c < width; c += kRotThreads * N)
                *reinterpret_cast<uint4 *>(y + c) = *reinterpret_cast<const uint4 *>(from + c);
        } else {
#pragma unroll 4
            for (int c = threadIdx.x; c < width; c += kRotThreads) y[c] = from[c];
        }
    }
}

template <typename T, bool HALF>
int launch_rotary(p3d_ctx *ctx, RotaryParams p) {
    constexpr int N = Vec<T>::N, es = sizeof(T);
    const uintptr_t xa = reinterpret_cast<uintptr_t>(p.x), oa = reinterpret_cast<uintptr_t>(p.out);
    const bool rows16 = (xa | oa) % 16 == 0 && (p.n == 1 || (p.ldx % N == 0 && p.ldo % N == 0));
    p.by_half = Divisor(p.half);
    const int iph = HALF ? (p.dim - p.half) / N : p.dim / N;  // items of a head
    if (rows16 && p.dim % N == 0 && (!HALF || p.half % N == 0) && static_cast<int64_t>(p.heads) * iph < (1 << 24)) {
        p.per_head = Divisor(iph);
        p.items = p.heads * iph;
        // 1024 items a block, so the angles are spread over few tokens, and a
        // few tokens' rows keep every thread's vectors in flight
        p.tokens = std::max(1, std::min({1024 / p.items, 4096 / p.half, 64}));
        p.per_token = Divisor(p.items);
        P3D_CUDA(ctx, launch_pdl(rotary_kernel<T, HALF>, dim3(static_cast<unsigned>(ceil_div(p.n, p.tokens))), dim3(kRotThreads),
                                 sizeof(float2) * p.tokens * p.half, ctx->stream, p));
        return check_launch(ctx, "rotary");
    }
    // whole groups of N heads start on 16-byte boundaries of aligned rows, whatever dim is
    p.group = std::min(p.heads, std::max(N, 16384 / es / p.dim / N * N));
    p.vectors = rows16 && static_cast<int64_t>(p.heads) * p.dim % N == 0;
    p.tokens = std::max(1, std::min({16384 / (p.group * p.dim * es), 1024 / p.half, 16}));
    const size_t smem = sizeof(float2) * ((p.tokens * p.half + 1) & ~1) + static_cast<size_t>(p.tokens) * p.group * p.dim * es;
    P3D_CUDA(ctx, launch_pdl(rotary_staged_kernel<T, HALF>,
                             dim3(static_cast<unsigned>(ceil_div(p.n, p.tokens)), static_cast<unsigned>(ceil_div(p.heads, p.group))),
                             dim3(kRotThreads), smem, ctx->stream, p));
    return check_launch(ctx, "rotary_staged");
}

template <typename T>
int launch_layout(p3d_ctx *ctx, const RotaryParams &p, int layout) {
    return layout == P3D_ROTARY_HALF ? launch_rotary<T, true>(ctx, p) : launch_rotary<T, false>(ctx, p);
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
    RotaryParams p{};
    p.x = x;
    p.ldx = ldx;
    p.out = out;
    p.ldo = ldo;
    p.n = n;
    p.positions = positions;
    p.offset = position_offset;
    p.freqs = freqs;
    p.amplitude = amplitude;
    p.heads = heads;
    p.dim = head_dim;
    p.half = rot_dim / 2;
    DeviceGuard on(ctx->device);
    if (dtype == P3D_F32) return launch_layout<float>(ctx, p, layout);
    if (dtype == P3D_BF16) return launch_layout<__nv_bfloat16>(ctx, p, layout);
    return launch_layout<__half>(ctx, p, layout);
}
