// Masked attention for few query rows: one query of each sequence at a time,
// its keys split over warps and blocks and joined.
//
// With one new token a sequence the work is reading K and V once: 2 d bytes a
// key and shared head, at 4 d operations for each of its heads.  A block takes
// one query, one K/V head with the (up to 16) query heads that share it, and
// one range of keys; its 4 warps take 16-key tiles in turn, each with its own
// running maximum and sum, and are joined in shared memory; the blocks of a
// query are joined by a second kernel.
//
// The 16 rows of m16n8k16 are heads, so all rows of a tile see the same keys:
// a hidden key's V is never read (zeros stand in), whatever it holds.  K and V
// go from memory to the operand registers without shared memory, because a
// contraction may take its index in any order and a column any name: lane
// (g, j) = (lane / 4, lane % 4) loads 16 bytes, dims 32 c + 8 j .. + 7 of key
// g, and uses them as the k indices of two products, Q's rows being loaded the
// same way; for V it loads dims 64 s + 8 g .. + 7 of the keys 2j, 2j + 1,
// 2j + 8, 2j + 9, and product i takes the i-th dim of every lane.
#include <algorithm>

#include "p3d_masked.cuh"

namespace p3d {
namespace {

constexpr int kWarps = 4;
constexpr int kThreadsR = 32 * kWarps;

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t word(const uint4 &u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

template <typename T, int D>
__global__ void __launch_bounds__(kThreadsR) masked_rows_kernel(const MaskedParams p) {
    constexpr int KC = D / 32;  // 16-byte chunks of a K row per lane
    constexpr int VS = D / 64;  // 64-dim slabs of V
    __shared__ float sm_o[kWarps][16][D];
    __shared__ float sm_m[kWarps][16], sm_l[kWarps][16];

    const int htiles = (p.group + 15) / 16;
    int64_t b = blockIdx.x;
    const int split = static_cast<int>(b % p.nsplit);
    b /= p.nsplit;
    const int ht = static_cast<int>(b % htiles);
    b /= htiles;
    const int hk = static_cast<int>(b % p.kv_heads);
    const int qi = static_cast<int>(b / p.kv_heads);
    const int seq = blockIdx.y;
    const SeqRange sr = seq_range(p, seq);
    if (qi >= sr.lq) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    const int64_t qrow = sr.q0 + qi;
    const int pos = qi + sr.lk - sr.lq;
    const int pre = p.prefix ? min(max(p.prefix[seq], 0), sr.lk) : 0;
    const int end = p.causal ? max(pre, min(sr.lk, pos + 1)) : sr.lk;  // keys from here on are hidden
    const int docq = p.doc_q ? p.doc_q[qrow] : 0;
    const int head0 = hk * p.group + ht * 16;
    const int nrows = min(16, p.group - ht * 16);
    // this block's keys, in whole 16-key tiles
    const int tiles = (max(end, 0) + 15) / 16;
    const int per = (tiles + p.nsplit - 1) / p.nsplit;
    const int tile0 = split * per, tile1 = min(tiles, tile0 + per);

    const T *kb = static_cast<const T *>(p.k) + sr.k0 * p.ldk + hk * D;
    const T *vb = static_cast<const T *>(p.v) + sr.k0 * p.ldv + hk * D;

    uint32_t qf[KC][2][4];  // [chunk][product][operand word]
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        const T *q0 = static_cast<const T *>(p.q) + qrow * p.ldq + static_cast<int64_t>(head0) * D + c * 32 + j * 8;
        const uint4 lo = g < nrows ? *reinterpret_cast<const uint4 *>(q0 + g * D) : make_uint4(0, 0, 0, 0);
        const uint4 hi = g + 8 < nrows ? *reinterpret_cast<const uint4 *>(q0 + (g + 8) * D) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            qf[c][h][0] = word(lo, 2 * h);
            qf[c][h][1] = word(hi, 2 * h);
            qf[c][h][2] = word(lo, 2 * h + 1);
            qf[c][h][3] = word(hi, 2 * h + 1);
        }
    }
    float slope[2] = {0.0f, 0.0f};
    if (p.slopes) {
        if (g < nrows) slope[0] = p.slopes[head0 + g] * 1.4426950408889634f;
        if (g + 8 < nrows) slope[1] = p.slopes[head0 + g + 8] * 1.4426950408889634f;
    }

    float o[VS][8][4];
#pragma unroll
    for (int s = 0; s < VS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[s][i][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    uint4 kf[2][KC];
    auto load_k = [&](int tile) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = min(tile * 16 + t * 8 + g, sr.lk - 1);  // a row past the end is read as the last, then hidden
#pragma unroll
            for (int c = 0; c < KC; ++c)
                kf[t][c] = __ldg(reinterpret_cast<const uint4 *>(kb + key * p.ldk + c * 32 + j * 8));
        }
    };
    if (tile0 + warp < tile1) load_k(tile0 + warp);
    for (int tile = tile0 + warp; tile < tile1; tile += kWarps) {
        bool vis[4];
        uint4 vf[4][VS];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int key = tile * 16 + 2 * j + (e & 1) + (e >> 1) * 8;
            vis[e] = key < end && (key < pre || ((!p.causal || key <= pos) && (!p.doc_k || p.doc_k[sr.k0 + key] == docq)));
#pragma unroll
            for (int s = 0; s < VS; ++s)
                vf[e][s] = vis[e] ? __ldg(reinterpret_cast<const uint4 *>(vb + key * p.ldv + s * 64 + g * 8)) : make_uint4(0, 0, 0, 0);
        }
        float sc[2][4];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[t][e] = 0.0f;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                mma16816<T>(sc[t], qf[c][0], kf[t][c].x, kf[t][c].y);
                mma16816<T>(sc[t], qf[c][1], kf[t][c].z, kf[t][c].w);
            }
        }
        if (tile + kWarps < tile1) load_k(tile + kWarps);
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = tile * 16 + t * 8 + 2 * j + (e & 1), r = e >> 1;
                float x = p.c1 > 0.0f ? capped(sc[t][e], p.c0, p.c1) : sc[t][e] * p.c0;
                if (p.slopes) x = fmaf(-slope[r], static_cast<float>(abs(pos - key)), x);
                x = vis[2 * t + (e & 1)] ? x : -INFINITY;
                sc[t][e] = x;
                mx[r] = fmaxf(mx[r], x);
            }
        bool raised = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            raised |= mx[r] > m[r];
        }
        if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float mn = fmaxf(m[r], mx[r]);
                const float a = m[r] == mn ? 1.0f : ex2f(m[r] - mn);  // m = -inf: 0
                m[r] = mn;
                l[r] *= a;
#pragma unroll
                for (int s = 0; s < VS; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        o[s][i][2 * r] *= a;
                        o[s][i][2 * r + 1] *= a;
                    }
            }
        }
        uint32_t pf[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float base = m[r] == -INFINITY ? 0.0f : m[r];
                const uint32_t w = pack2<T>(ex2f(sc[t][2 * r] - base), ex2f(sc[t][2 * r + 1] - base));
                const float2 f = unpack2<T>(w);  // the sum takes the weights as the product sees them
                l[r] += f.x + f.y;
                pf[2 * t + r] = w;
            }
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
                const uint32_t b0 = __byte_perm(word(vf[0][s], i / 2), word(vf[1][s], i / 2), sel);
                const uint32_t b1 = __byte_perm(word(vf[2][s], i / 2), word(vf[3][s], i / 2), sel);
                mma16816<T>(o[s][i], pf, b0, b1);
            }
    }
    // join the warps
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (j == 0) {
            sm_m[warp][g + 8 * r] = m[r];
            sm_l[warp][g + 8 * r] = l[r];
        }
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sm_o[warp][g + 8 * r][s * 64 + 16 * j + i] = o[s][i][2 * r];
                sm_o[warp][g + 8 * r][s * 64 + 16 * j + 8 + i] = o[s][i][2 * r + 1];
            }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nrows * D; e += kThreadsR) {
        const int r = e / D, d = e % D;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w][r]);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float a = ex2f(sm_m[w][r] - base);
            ll = fmaf(sm_l[w][r], a, ll);
            oo = fmaf(sm_o[w][r][d], a, oo);
        }
        const int head = head0 + r;
        if (p.nsplit == 1) {
            static_cast<T *>(p.out)[qrow * p.ldo + static_cast<int64_t>(head) * D + d] =
                from_f32<T>(ll == 0.0f ? 0.0f : oo / ll);
        } else {
            const int64_t at = (qrow * p.heads + head) * p.nsplit + split;
            p.part_o[at * D + d] = oo;
            if (d == 0) p.part_ml[at] = make_float2(mm, ll);
        }
    }
}

// A warp joins the splits of one row and head.
template <typename T, int D>
__global__ void __launch_bounds__(256) masked_join_kernel(const MaskedParams p) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int head = static_cast<int>(item % p.heads);
    const int64_t qi = item / p.heads;
    const SeqRange sr = seq_range(p, blockIdx.y);
    if (qi >= sr.lq || qi >= p.max_q) return;
    const int64_t at = ((sr.q0 + qi) * p.heads + head) * p.nsplit;
    float mm = -INFINITY;
    for (int s = lane; s < p.nsplit; s += 32) mm = fmaxf(mm, p.part_ml[at + s].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    const float base = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, oo[E] = {};
    for (int s = 0; s < p.nsplit; ++s) {
        const float2 ml = p.part_ml[at + s];
        const float a = ex2f(ml.x - base);
        ll = fmaf(ml.y, a, ll);
        const float *src = p.part_o + (at + s) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) oo[e] = fmaf(src[e], a, oo[e]);
    }
    T *dst = static_cast<T *>(p.out) + (sr.q0 + qi) * p.ldo + static_cast<int64_t>(head) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) dst[e] = from_f32<T>(ll == 0.0f ? 0.0f : oo[e] / ll);
}

template <typename T, int D>
int launch_rows(p3d_ctx *ctx, const MaskedParams &p) {
    const int64_t blocks = static_cast<int64_t>(p.nsplit) * ((p.group + 15) / 16) * p.kv_heads * p.max_q;
    if (blocks >= (int64_t(1) << 31)) return set_error(ctx, P3D_ERR_UNSUPPORTED, "p3d_masked_attention: too many query rows");
    masked_rows_kernel<T, D><<<dim3(static_cast<unsigned>(blocks), p.nseq), kThreadsR, 0, ctx->stream>>>(p);
    int rc = check_launch(ctx, "masked_rows");
    if (rc || p.nsplit == 1) return rc;
    masked_join_kernel<T, D><<<dim3(static_cast<unsigned>(ceil_div(p.max_q * p.heads, 8)), p.nseq), 256, 0, ctx->stream>>>(p);
    return check_launch(ctx, "masked_join");
}

}  // namespace

int masked_attention_rows(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype) {
    if (dtype == P3D_BF16)
        return head_dim == 64 ? launch_rows<__nv_bfloat16, 64>(ctx, p) : launch_rows<__nv_bfloat16, 128>(ctx, p);
    return head_dim == 64 ? launch_rows<__half, 64>(ctx, p) : launch_rows<__half, 128>(ctx, p);
}

}  // namespace p3d
