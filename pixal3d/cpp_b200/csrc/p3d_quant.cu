// Quantisation of rows to 8-bit integers, one scale for each row.
//
//   s_i  = max(fl32(max_j |x_ij| / 127), 2^-126)
//   q_ij = rint(x_ij / s_i)          (ties to even, decided exactly)
//
// The result does not depend on how the quotient is rounded on its way: q is
// first x * fl(1/s) rounded to an integer, which is off by at most one, and only where
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
// written; the row stays in registers between the two uses.  Elements go in
// pairs and the integer is the low byte of x / s + 1.5 * 2^23, so one element
// takes about five instructions.  A row is read in the 16-byte words it
// touches, wherever it starts: a word never crosses an allocation, and what
// lies beside the row is masked.  8184 x 4096 f16 takes
// 18.2 us (5.5 TB/s), f32 27.2 (6.2 TB/s).
#include "p3d_common.cuh"

namespace p3d {
namespace {

struct RowScale {
    float s, inv;
    bool bad;  // the row holds an infinity or a NaN
};
// From the row's largest |x| as the bits of an f32 (ordered like the values,
// with NaN above infinity above every finite value).
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    r.bad = amax_bits >= 0x7f800000u;
    r.s = fmaxf(__fdiv_rn(__uint_as_float(amax_bits), 127.0f), 1.17549435e-38f);
    r.inv = __frcp_rn(r.s);
    return r;
}

constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, which is then the low byte

// The neighbour of t's integer where that is nearer to x, or x lies halfway
// and the neighbour is even.
__device__ __forceinline__ uint32_t settle(uint32_t t, float x, float s) {
    const float r = fmaf(kMagic - __uint_as_float(t), s, x);
    const float r2 = 2.0f * fabsf(r);
    if (r2 > s || (r2 == s && (t & 1))) t += r > 0.0f ? 1u : 0xffffffffu;
    return t;
}

// Four elements to four bytes.
__device__ __forceinline__ uint32_t quant4(float a, float b, float c, float d, const RowScale &rs) {
    const F2 inv(rs.inv, rs.inv), magic(kMagic, kMagic), less(-kMagic, -kMagic), s(-rs.s, -rs.s);
    const F2 ab(a, b), cd(c, d);
    const F2 t0 = fma2(ab, inv, magic), t1 = fma2(cd, inv, magic);
    float r[4], t[4];
    fma2(add2(t0, less), s, ab).get(r[0], r[1]);
    fma2(add2(t1, less), s, cd).get(r[2], r[3]);
    t0.get(t[0], t[1]);
    t1.get(t[2], t[3]);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(t[i]);
    if (2.0f * fmaxf(fmaxf(fabsf(r[0]), fabsf(r[1])), fmaxf(fabsf(r[2]), fabsf(r[3]))) >= rs.s) {  // rare
        w[0] = settle(w[0], a, rs.s);
        w[1] = settle(w[1], b, rs.s);
        w[2] = settle(w[2], c, rs.s);
        w[3] = settle(w[3], d, rs.s);
    }
    return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
}

// A 16-byte word of a row.
template <typename T>
struct Word {
    static constexpr int N = 16 / sizeof(T);
    uint32_t w[4];
    __device__ __forceinline__ void load(const void *p) {
        const uint4 u = __ldg(static_cast<const uint4 *>(p));
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    }
    // elements outside [lo, hi) to zero
    __device__ __forceinline__ void keep(int lo, int hi) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < lo || e >= hi) w[e * sizeof(T) / 4] &= sizeof(T) == 4 ? 0u : (e & 1) ? 0x0000ffffu : 0xffff0000u;
    }
    // running maximum of |x|: f32 bits, or two 16-bit patterns
    __device__ __forceinline__ void top(uint32_t &m) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) m = sizeof(T) == 4 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
    }
    __device__ __forceinline__ void quantise(const RowScale &rs, uint32_t (&q)[N / 4]) const {
        if constexpr (sizeof(T) == 4) {
            q[0] = quant4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]), rs);
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float2 a = unpack2<T>(w[2 * h]), b = unpack2<T>(w[2 * h + 1]);
                q[h] = quant4(a.x, a.y, b.x, b.y, rs);
            }
        }
        if (rs.bad) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) q[i] = 0;
        }
    }
};

// Running maxima of a row's threads (o < their number apart) to f32 bits.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t m, int width) {
    if (sizeof(T) == 2) {
        m = max(m & 0xffffu, m >> 16);
        m = __float_as_uint(unpack2<T>(m).x);
    }
    for (int o = 1; o < width; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
template <>
__device__ __forceinline__ uint32_t top_bits<float>(uint32_t m, int width) {
    for (int o = 1; o < width; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// TPR threads a row (8, 32, or a whole block of more), each holding up to HOLD words
// of it in registers; a longer row is read a second time.
template <int TPR>
constexpr int quant_block() {
    return TPR > 32 ? TPR : 256;
}
template <typename T, int TPR, int HOLD>
__global__ void __launch_bounds__(quant_block<TPR>())
    quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int64_t m, int k, int8_t *__restrict__ q, int64_t ldq,
                         float *__restrict__ scale) {
    constexpr int N = Word<T>::N;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x % TPR;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * (quant_block<TPR>() / TPR) + threadIdx.x / TPR;
    const bool live = at < m;  // every thread stays for the shuffles
    const int64_t row = live ? at : m - 1;
    const uintptr_t p0 = reinterpret_cast<uintptr_t>(x + row * ldx);
    const int off = static_cast<int>(p0 & 15) / static_cast<int>(sizeof(T));  // elements of the first word before the row
    const char *base = reinterpret_cast<const char *>(p0 & ~uintptr_t(15));
    const int nw = (off + k + N - 1) / N;
    auto trim = [&](int i, Word<T> &u) {
        if (i == 0 || i == nw - 1) u.keep(i == 0 ? off : 0, min(N, off + k - i * N));
    };
    Word<T> v[HOLD];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (lane + h * TPR < nw) v[h].load(base + static_cast<int64_t>(lane + h * TPR) * 16);  // all on their way first
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (lane + h * TPR < nw) {
            trim(lane + h * TPR, v[h]);
            v[h].top(top);
        }
#pragma unroll 4
    for (int i = lane + HOLD * TPR; i < nw; i += TPR) {
        Word<T> u;
        u.load(base + static_cast<int64_t>(i) * 16);
        trim(i, u);
        u.top(top);
    }
    top = top_bits<T>(top, TPR < 32 ? TPR : 32);
    if constexpr (TPR > 32) {
        __shared__ uint32_t part[TPR / 32];
        if (lane % 32 == 0) part[lane / 32] = top;
        __syncthreads();
        top = part[0];
#pragma unroll
        for (int w = 1; w < TPR / 32; ++w) top = max(top, part[w]);
    }
    if (!live) return;
    const RowScale rs = row_scale(top);
    if (lane == 0) scale[row] = rs.bad ? __int_as_float(0x7fc00000) : rs.s;
    int8_t *qr = q + row * ldq - off;  // word i's bytes go to qr + N i
    const bool wide = reinterpret_cast<uintptr_t>(qr) % N == 0;
    auto store = [&](int i, const Word<T> &u) {
        uint32_t w[N / 4];
        u.quantise(rs, w);
        int8_t *d = qr + static_cast<int64_t>(i) * N;
        const int lo = i == 0 ? off : 0, hi = min(N, off + k - i * N);
        if (wide && lo == 0 && hi == N) {
            if constexpr (N == 8)
                *reinterpret_cast<uint2 *>(d) = make_uint2(w[0], w[1]);
            else
                *reinterpret_cast<uint32_t *>(d) = w[0];
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (e >= lo && e < hi) d[e] = static_cast<int8_t>(w[e / 4] >> (8 * (e % 4)));
        }
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if (lane + h * TPR < nw) store(lane + h * TPR, v[h]);
    for (int i = lane + HOLD * TPR; i < nw; i += TPR) {
        Word<T> u;
        u.load(base + static_cast<int64_t>(i) * 16);
        store(i, u);  // writes the row's own elements only
    }
}

template <typename T, int TPR, int HOLD>
int launch_width(p3d_ctx *ctx, const T *x, int64_t ldx, int64_t m, int k, int8_t *q, int64_t ldq, float *scale) {
    P3D_CUDA(ctx, launch_pdl(quantize_rows_kernel<T, TPR, HOLD>, dim3(static_cast<unsigned>(ceil_div(m, quant_block<TPR>() / TPR))),
                             dim3(quant_block<TPR>()), 0, ctx->stream, x, ldx, m, k, q, ldq, scale));
    return check_launch(ctx, "quantize_rows");
}

template <typename T>
int launch_quantize(p3d_ctx *ctx, const void *x, int64_t ldx, int64_t m, int64_t k, int8_t *q, int64_t ldq, float *scale) {
    const T *xt = static_cast<const T *>(x);
    const int kk = static_cast<int>(k);
    // one word more where rows start inside one
    const bool whole = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (m == 1 || ldx * sizeof(T) % 16 == 0);
    const int64_t words = ceil_div(k, Word<T>::N) + (whole ? 0 : 1);
    // Words held a thread against rows in flight an SM; us with the choice and
    // its best neighbours: 64 f16 columns (8 words) 5.1, 32 threads 15.5;
    // 1024 bf16 (128) 6.8, 64 threads 9.2; 773 f32 (194) 16.0, 4 words 18.0;
    // 4096 f16 (512) 18.4, 32 x 16 29.3, 128 x 4 19.7; 4096 f32 (1024) 27.4,
    // 64 x 8 35.9; 33000 f16 (4126) 23.6, 128 x 8 28.7 (43532, 8184, 21766,
    // 8184, 8184 and 1000 rows).  Fewer rows than SMs take a whole block each:
    // one row of 4096 f16 1.9 against 2.8 us.
    if (m < ctx->num_sms && words > 32) return launch_width<T, 256, 2>(ctx, xt, ldx, m, kk, q, ldq, scale);
    if (words <= 32) return launch_width<T, 8, 4>(ctx, xt, ldx, m, kk, q, ldq, scale);
    if (words <= 128) return launch_width<T, 32, 4>(ctx, xt, ldx, m, kk, q, ldq, scale);
    if (words <= 256) return launch_width<T, 32, 8>(ctx, xt, ldx, m, kk, q, ldq, scale);
    if (words <= 512) return launch_width<T, 64, 8>(ctx, xt, ldx, m, kk, q, ldq, scale);
    if (words <= 1024) return launch_width<T, 128, 8>(ctx, xt, ldx, m, kk, q, ldq, scale);
    return launch_width<T, 256, 8>(ctx, xt, ldx, m, kk, q, ldq, scale);
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
    if (dtype == P3D_F32) return launch_quantize<float>(ctx, x, ldx, m, k, q, ldq, scale);
    if (dtype == P3D_BF16) return launch_quantize<__nv_bfloat16>(ctx, x, ldx, m, k, q, ldq, scale);
    return launch_quantize<__half>(ctx, x, ldx, m, k, q, ldq, scale);
}
