// Masked attention for few query rows over few keys: a block takes one query
// and one K/V head with the (up to 16) query heads that share it; its warps
// take 16-key tiles in turn, each with its own running maximum and sum, and
// are joined in shared memory.  (Long keys: p3d_masked_pieces.cu.)
//
// A call is a chain of memory latencies rather than bytes: 300 keys, 16 heads
// of 64 take 5.8 us, 8 sequences of 500 keys 7.1; with 4 warps instead of 8
// they took 6.6 and 9.4.
//
// All heads of a block see the same keys, so a hidden key's V is never read
// (zeros stand in), whatever it holds.
//
// Scores are S[head][key] = Q K^T (m16n8k16, the heads as its 16 rows), the
// output O^T[dim][head] += V^T P^T with 8 heads as columns: S's accumulator
// layout, row lane / 4 and columns 2 (lane % 4) + {0, 1}, is the layout of the
// second product's B operand, so the weights go from one to the other inside a
// lane, and up to 8 heads take half the accumulators that O[head][dim] would.
// K and V go from memory to the operand registers without shared memory,
// because a contraction may take its index in any order and a row any name:
// lane (g, j) = (lane / 4, lane % 4) loads 16 bytes, dims 32 c + 8 j .. + 7 of
// key g, and uses them as the k indices of two products, Q's rows being loaded
// the same way; for V it loads dims 64 s + 8 g .. + 7 of the keys 2j, 2j + 1,
// 2j + 8, 2j + 9, and product i has dims 64 s + 8 g + 2 i and + 1 as its rows g
// and g + 8.
#include <algorithm>

#include "p3d_masked_small.cuh"

namespace p3d {
namespace {

template <int D, int HT, int W>
struct RowsShared {
    float o[W][8 * HT][D + 4];  // + 4: the 8 dims a lane stores start in different banks for different heads
    float m[W][8 * HT], l[W][8 * HT];
};

// Item `local` (query, K/V head, group of 8 HT of its heads) of sequence seq.
template <typename T, int D, int HT, int W>
__device__ __forceinline__ void rows_item(const MaskedParams &p, RowsShared<D, HT, W> &sm, const SeqRange &sr, int seq, int local) {
    constexpr int KC = D / 32;  // 16-byte chunks of a K row per lane
    constexpr int VS = D / 64;  // 64-dim slabs of V
    constexpr int H = 8 * HT;
    const int ht = local % p.head_tiles, hk = local / p.head_tiles % p.kv_heads, qi = local / p.head_tiles / p.kv_heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3;
    const int64_t qrow = sr.q0 + qi;
    const int pos = qi + sr.lk - sr.lq;
    const int pre = p.prefix ? min(max(p.prefix[seq], 0), sr.lk) : 0;
    const int end = p.causal ? max(pre, min(sr.lk, pos + 1)) : sr.lk;  // keys from here on are hidden
    const int docq = p.doc_q ? p.doc_q[qrow] : 0;
    const int head0 = hk * p.group + ht * H;
    const int nrows = min(H, p.group - ht * H);
    const int tiles = (max(end, 0) + 15) / 16;

    const T *kb = static_cast<const T *>(p.k) + sr.k0 * p.ldk + hk * D;
    const T *vb = static_cast<const T *>(p.v) + sr.k0 * p.ldv + hk * D;

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
    if (warp < tiles) load_k(warp);

    uint4 qf[HT][KC];
#pragma unroll
    for (int r = 0; r < HT; ++r)
#pragma unroll
        for (int c = 0; c < KC; ++c)
            qf[r][c] = g + 8 * r < nrows ? *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + qrow * p.ldq +
                                                                            static_cast<int64_t>(head0 + g + 8 * r) * D + c * 32 + j * 8)
                                         : make_uint4(0, 0, 0, 0);
    float slope[HT];
#pragma unroll
    for (int r = 0; r < HT; ++r)
        slope[r] = p.slopes && g + 8 * r < nrows ? p.slopes[head0 + g + 8 * r] * 1.4426950408889634f : 0.0f;

    float o[VS][4][HT][4];  // [slab][product][8 heads]: (dim, head 2j), (dim, 2j + 1), (dim + 1, 2j), (dim + 1, 2j + 1)
#pragma unroll
    for (int s = 0; s < VS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < HT; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[s][i][r][e] = 0.0f;
    float m[HT], l[HT];  // of head g + 8 r
#pragma unroll
    for (int r = 0; r < HT; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
    }

    for (int tile = warp; tile < tiles; tile += W) {
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
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a[4] = {word(qf[0][c], 2 * h), HT > 1 ? word(qf[HT - 1][c], 2 * h) : 0u,
                                           word(qf[0][c], 2 * h + 1), HT > 1 ? word(qf[HT - 1][c], 2 * h + 1) : 0u};
                    mma16816<T>(sc[t], a, word(kf[t][c], 2 * h), word(kf[t][c], 2 * h + 1));
                }
        }
        if (tile + W < tiles) load_k(tile + W);
        float mx[HT];
        bool raised = false;
#pragma unroll
        for (int r = 0; r < HT; ++r) {
            mx[r] = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = tile * 16 + t * 8 + 2 * j + e;
                    float x = sc[t][2 * r + e];
                    x = p.c1 > 0.0f ? capped(x, p.c0, p.c1) : x * p.c0;
                    if (p.slopes) x = fmaf(-slope[r], static_cast<float>(abs(pos - key)), x);
                    x = vis[2 * t + e] ? x : -INFINITY;
                    sc[t][2 * r + e] = x;
                    mx[r] = fmaxf(mx[r], x);
                }
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2)) - kLift<T>;
            raised |= mx[r] > m[r];
        }
        if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
            for (int r = 0; r < HT; ++r) {
                const float mn = fmaxf(m[r], mx[r]);
                const float a = m[r] == mn ? 1.0f : ex2f(m[r] - mn);  // m = -inf: 0
                m[r] = mn;
                l[r] *= a;
                const float a0 = __shfl_sync(0xffffffffu, a, 8 * j), a1 = __shfl_sync(0xffffffffu, a, 8 * j + 4);  // heads 2j, 2j + 1
#pragma unroll
                for (int s = 0; s < VS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[s][i][r][0] *= a0;
                        o[s][i][r][1] *= a1;
                        o[s][i][r][2] *= a0;
                        o[s][i][r][3] *= a1;
                    }
            }
        }
        uint32_t pf[HT][2];
#pragma unroll
        for (int r = 0; r < HT; ++r) {
            const float base = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                pf[r][t] = pack2<T>(ex2f(sc[t][2 * r] - base), ex2f(sc[t][2 * r + 1] - base));
                const float2 f = unpack2<T>(pf[r][t]);  // the sum takes the weights as the product sees them
                l[r] += f.x + f.y;
            }
        }
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a[4] = {__byte_perm(word(vf[0][s], i), word(vf[1][s], i), 0x5410u),
                                       __byte_perm(word(vf[0][s], i), word(vf[1][s], i), 0x7632u),
                                       __byte_perm(word(vf[2][s], i), word(vf[3][s], i), 0x5410u),
                                       __byte_perm(word(vf[2][s], i), word(vf[3][s], i), 0x7632u)};
#pragma unroll
                for (int r = 0; r < HT; ++r) mma16816<T>(o[s][i][r], a, pf[r][0], pf[r][1]);
            }
    }
    // join the warps
#pragma unroll
    for (int r = 0; r < HT; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (j == 0) {
            sm.m[warp][g + 8 * r] = m[r];
            sm.l[warp][g + 8 * r] = l[r];
        }
#pragma unroll
        for (int s = 0; s < VS; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<float4 *>(&sm.o[warp][8 * r + 2 * j + e][s * 64 + g * 8 + 4 * h]) =
                        make_float4(o[s][2 * h][r][e], o[s][2 * h][r][2 + e], o[s][2 * h + 1][r][e], o[s][2 * h + 1][r][2 + e]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < nrows * (D / 4); e += 32 * W) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) mm = fmaxf(mm, sm.m[w][r]);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f;
        float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float a = ex2f(sm.m[w][r] - base);
            const float4 x = *reinterpret_cast<const float4 *>(&sm.o[w][r][d]);
            ll = fmaf(sm.l[w][r], a, ll);
            oo.x = fmaf(x.x, a, oo.x);
            oo.y = fmaf(x.y, a, oo.y);
            oo.z = fmaf(x.z, a, oo.z);
            oo.w = fmaf(x.w, a, oo.w);
        }
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
        *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + qrow * p.ldo + static_cast<int64_t>(head0 + r) * D + d) =
            make_uint2(pack2<T>(oo.x * inv, oo.y * inv), pack2<T>(oo.z * inv, oo.w * inv));
    }
}

template <int D, int HT>
constexpr int item_warps() {
    return D * HT > 128 ? 4 : 8;  // 16 heads of 128 would need 68 KB for the join
}
template <typename T, int D, int HT>
__global__ void __launch_bounds__(32 * item_warps<D, HT>()) masked_items_kernel(const MaskedParams p) {
    constexpr int W = item_warps<D, HT>();
    __shared__ RowsShared<D, HT, W> sm;
    pdl_wait();
    pdl_trigger();
    const SeqRange sr = seq_range(p, blockIdx.y);
    if (blockIdx.x < min(static_cast<int64_t>(sr.lq), p.max_q) * p.kv_heads * p.head_tiles)
        rows_item<T, D, HT, W>(p, sm, sr, blockIdx.y, blockIdx.x);
}

template <typename T, int D, int HT>
int launch_rows(p3d_ctx *ctx, const MaskedParams &p) {
    const int64_t items = p.max_q * p.kv_heads * p.head_tiles;  // of the longest sequence
    if (items >= (int64_t(1) << 31)) return set_error(ctx, P3D_ERR_UNSUPPORTED, "p3d_masked_attention: too many query rows");
    P3D_CUDA(ctx, launch_pdl(masked_items_kernel<T, D, HT>, dim3(static_cast<unsigned>(items), p.nseq),
                             dim3(32 * item_warps<D, HT>()), 0, ctx->stream, p));
    return check_launch(ctx, "masked_items");
}

template <typename T, int D>
int launch_heads(p3d_ctx *ctx, MaskedParams p) {
    p.head_tiles = static_cast<int>(ceil_div(p.group, p.group > 8 ? 16 : 8));
    return p.group > 8 ? launch_rows<T, D, 2>(ctx, p) : launch_rows<T, D, 1>(ctx, p);
}

}  // namespace

int masked_attention_rows(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype) {
    if (dtype == P3D_BF16)
        return head_dim == 64 ? launch_heads<__nv_bfloat16, 64>(ctx, p) : launch_heads<__nv_bfloat16, 128>(ctx, p);
    return head_dim == 64 ? launch_heads<__half, 64>(ctx, p) : launch_heads<__half, 128>(ctx, p);
}

}  // namespace p3d
