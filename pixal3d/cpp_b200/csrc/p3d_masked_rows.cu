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

#include "p3d_masked.cuh"

namespace p3d {
namespace {

constexpr int kWarps = 4;  // of a block that walks a range, and of the join
constexpr int kThreadsR = 32 * kWarps;
// A block that takes a whole item of few keys has 8 warps: half as many tiles
// one after the other.

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

__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

__device__ __forceinline__ uint32_t word(const uint4 &u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// Key tiles of one item of a sequence (at least one, so that every item has a
// block) and the sequence's items: query, K/V head, 8 * HT of its heads.
__device__ __forceinline__ int item_tiles(const SeqRange &sr) { return max(1, (sr.lk + 15) / 16); }
__device__ __forceinline__ int seq_items(const MaskedParams &p, const SeqRange &sr) {
    return static_cast<int>(min(static_cast<int64_t>(sr.lq), p.max_q)) * p.kv_heads * p.head_tiles;
}

// The tiles of all items (a whole warp calls it).
__device__ __forceinline__ int64_t all_tiles(const MaskedParams &p, int lane) {
    int64_t t = 0;
    for (int s = lane; s < p.nseq; s += 32) {
        const SeqRange sr = seq_range(p, s);
        t += static_cast<int64_t>(item_tiles(sr)) * seq_items(p, sr);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    return t;
}

// Tiles and items of the sequences before `seq`, or, with seq < 0, of those
// before the one that holds tile x, whose number is returned.
__device__ __forceinline__ int find_seq(const MaskedParams &p, int lane, int seq, int64_t x, int64_t &tiles, int64_t &items) {
    tiles = items = 0;
    for (int c = 0; c < p.nseq; c += 32) {
        int64_t w = 0, n = 0;
        if (c + lane < p.nseq) {
            const SeqRange sr = seq_range(p, c + lane);
            n = seq_items(p, sr);
            w = n * item_tiles(sr);
        }
        int64_t wi = w, ni = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t a = __shfl_up_sync(0xffffffffu, wi, o), b = __shfl_up_sync(0xffffffffu, ni, o);
            if (lane >= o) {
                wi += a;
                ni += b;
            }
        }
        const unsigned hit = __ballot_sync(0xffffffffu, seq >= 0 ? c + lane == seq : tiles + wi > x);
        if (hit) {
            const int l = __ffs(hit) - 1;
            tiles += __shfl_sync(0xffffffffu, wi - w, l);
            items += __shfl_sync(0xffffffffu, ni - n, l);
            return c + l;
        }
        tiles += __shfl_sync(0xffffffffu, wi, 31);
        items += __shfl_sync(0xffffffffu, ni, 31);
    }
    return p.nseq;
}

template <int D, int HT, int W>
struct RowsShared {
    float o[W][8 * HT][D + 4];  // + 4: the 8 dims a lane stores start in different banks for different heads
    float m[W][8 * HT], l[W][8 * HT];
};

// One item's key tiles [t0, t1): item `local` of sequence seq.  Writes the
// output when `whole`, else the part `slot` (sums against its own maximum).
// HT: 8 heads a block, or 16.
template <typename T, int D, int HT, int W>
__device__ __forceinline__ void rows_item(const MaskedParams &p, RowsShared<D, HT, W> &sm, const SeqRange &sr, int seq, int local, int t0,
                                          int t1, bool whole, int64_t slot) {
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
    const int tile0 = t0, tile1 = min(t1, (max(end, 0) + 15) / 16);

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
    if (tile0 + warp < tile1) load_k(tile0 + warp);

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

    // With 128-byte rows the tile after the next is fetched into L2, a line a
    // lane (16 sequences of up to 8192 keys, 16 heads: 98 -> 82 us); with
    // 256-byte rows the registers' own loads keep enough in flight and the same
    // made it slower (99 -> 106 us).
    auto prefetch = [&](int tile) {
        constexpr int LINES = D / 64;  // of a row
        const int key = min(tile * 16 + lane / LINES % 16, sr.lk - 1);
        if (LINES == 2 || lane < 16) prefetch_l2(kb + key * p.ldk + lane % LINES * 64);
        if (LINES == 2 || lane >= 16) prefetch_l2(vb + key * p.ldv + lane % LINES * 64);
    };
    constexpr int kAhead = D == 64 ? 2 : 0;
    for (int a = 1; a < kAhead; ++a)
        if (tile0 + warp + a * W < tile1) prefetch(tile0 + warp + a * W);
    for (int tile = tile0 + warp; tile < tile1; tile += W) {
        if (kAhead > 0 && tile + kAhead * W < tile1) prefetch(tile + kAhead * W);
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
        if (tile + W < tile1) load_k(tile + W);
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
            mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
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
    __syncthreads();  // the last item's parts have been read
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
        if (whole) {
            const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
            *reinterpret_cast<uint2 *>(static_cast<T *>(p.out) + qrow * p.ldo + static_cast<int64_t>(head0 + r) * D + d) =
                make_uint2(pack2<T>(oo.x * inv, oo.y * inv), pack2<T>(oo.z * inv, oo.w * inv));
        } else {
            *reinterpret_cast<float4 *>(p.part_o + (slot * H + r) * D + d) = oo;
            if (d == 0) p.part_ml[slot * H + r] = make_float2(mm, ll);
        }
    }
}

// Blocks an SM holds at once (registers).
template <int D, int HT>
constexpr int rows_per_sm() {
    return (D == 64 ? 4 : 3) - (HT - 1);
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
    if (static_cast<int>(blockIdx.x) < seq_items(p, sr))
        rows_item<T, D, HT, W>(p, sm, sr, blockIdx.y, blockIdx.x, 0, item_tiles(sr), true, 0);
}

template <typename T, int D, int HT>
__global__ void __launch_bounds__(kThreadsR, rows_per_sm<D, HT>()) masked_ranges_kernel(const MaskedParams p) {
    __shared__ RowsShared<D, HT, kWarps> sm;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t total = all_tiles(p, lane);  // every warp finds the same
    int64_t x = total * blockIdx.x / p.ranges;
    const int64_t x1 = total * (blockIdx.x + 1) / p.ranges;
    if (x >= x1) return;
    int64_t before, item;
    int seq = find_seq(p, lane, -1, x, before, item);
    if (seq >= p.nseq) return;
    SeqRange sr = seq_range(p, seq);
    int w = item_tiles(sr);
    int local = static_cast<int>((x - before) / w), t = static_cast<int>((x - before) % w);
    item += local;
    while (x < x1) {
        const int take = static_cast<int>(min(static_cast<int64_t>(w - t), x1 - x));
        rows_item<T, D, HT, kWarps>(p, sm, sr, seq, local, t, t + take, take == w, blockIdx.x + item);
        x += take;
        t = 0;
        ++local;
        ++item;
        while (x < x1 && local >= seq_items(p, sr) && seq + 1 < p.nseq) {
            sr = seq_range(p, ++seq);
            w = item_tiles(sr);
            local = 0;
        }
    }
}

// A block joins the parts of one query row and head.  Part number: block +
// item, which no other (block, item) pair has, as the items a block meets
// begin where the last block's end.
template <typename T, int D>
__global__ void __launch_bounds__(kThreadsR) masked_join_kernel(const MaskedParams p) {
    constexpr int E = D / 32;
    __shared__ float so[kWarps][D];
    __shared__ float2 sml[kWarps];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x % p.heads, qi = blockIdx.x / p.heads, seq = blockIdx.y;
    const SeqRange sr = seq_range(p, seq);
    if (qi >= sr.lq) return;
    const int H = p.group > 8 ? 16 : 8;
    const int in = head % p.group, local = (qi * p.kv_heads + head / p.group) * p.head_tiles + in / H, r = in % H;
    const int64_t total = all_tiles(p, lane);
    int64_t first, item;
    find_seq(p, lane, seq, 0, first, item);
    const int w = item_tiles(sr);
    first += static_cast<int64_t>(local) * w;
    item += local;
    // tile x lies in range ((x + 1) ranges - 1) / total
    const int64_t b0 = ((first + 1) * p.ranges - 1) / total, b1 = ((first + w) * p.ranges - 1) / total;
    if (b0 == b1) return;  // one block had all of it
    const int64_t s0 = b0 + item, s1 = b1 + item;
    float mm = -INFINITY;
    for (int64_t s = s0 + threadIdx.x % 32 * kWarps + warp; s <= s1; s += 32 * kWarps) mm = fmaxf(mm, p.part_ml[s * H + r].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    const float base = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, oo[E] = {};
#pragma unroll 8
    for (int64_t s = s0 + warp; s <= s1; s += kWarps) {
        const float2 ml = p.part_ml[s * H + r];
        const float a = ex2f(ml.x - base);
        ll = fmaf(ml.y, a, ll);
        const float *src = p.part_o + (s * H + r) * D + lane * E;
        float v[E];
        if constexpr (E == 4) {
            const float4 f = *reinterpret_cast<const float4 *>(src);
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
            const float2 f = *reinterpret_cast<const float2 *>(src);
            v[0] = f.x, v[1] = f.y;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) oo[e] = fmaf(v[e], a, oo[e]);
    }
    if (lane == 0) sml[warp] = make_float2(mm, ll);
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = oo[e];
    __syncthreads();
    if (threadIdx.x * 2 < D) {
        const int d = threadIdx.x * 2;
        float top = -INFINITY, sum = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) top = fmaxf(top, sml[k].x);
        const float b = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
            const float a = ex2f(sml[k].x - b);
            sum = fmaf(sml[k].y, a, sum);
            y0 = fmaf(so[k][d], a, y0);
            y1 = fmaf(so[k][d + 1], a, y1);
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        *reinterpret_cast<uint32_t *>(static_cast<T *>(p.out) + (sr.q0 + static_cast<int64_t>(qi)) * p.ldo +
                                      static_cast<int64_t>(head) * D + d) = pack2<T>(y0 * inv, y1 * inv);
    }
}

template <typename T, int D, int HT>
int launch_rows(p3d_ctx *ctx, MaskedParams p) {
    const int64_t items = p.max_q * p.kv_heads * p.head_tiles;  // of the longest sequence
    if (p.ranges > 0) {
        P3D_CUDA(ctx, launch_pdl(masked_ranges_kernel<T, D, HT>, dim3(p.ranges), dim3(kThreadsR), 0, ctx->stream, p));
        const int rc = check_launch(ctx, "masked_ranges");
        if (rc) return rc;
        P3D_CUDA(ctx, launch_pdl(masked_join_kernel<T, D>, dim3(static_cast<unsigned>(p.max_q * p.heads), p.nseq), dim3(kThreadsR), 0,
                                 ctx->stream, p));
        return check_launch(ctx, "masked_join");
    }
    if (items >= (int64_t(1) << 31)) return set_error(ctx, P3D_ERR_UNSUPPORTED, "p3d_masked_attention: too many query rows");
    P3D_CUDA(ctx, launch_pdl(masked_items_kernel<T, D, HT>, dim3(static_cast<unsigned>(items), p.nseq),
                             dim3(32 * item_warps<D, HT>()), 0, ctx->stream, p));
    return check_launch(ctx, "masked_items");
}

template <typename T, int D>
int launch_heads(p3d_ctx *ctx, const MaskedParams &p) {
    return p.group > 8 ? launch_rows<T, D, 2>(ctx, p) : launch_rows<T, D, 1>(ctx, p);
}

}  // namespace

// Up to 512 keys an item is one block's (a cut and its join cost 2.4 us: 300
// keys, 16 heads 5.8 against 8.7 us; at 1000 keys both take 11), and so it is where there are items for
// four rounds of the GPU.  Otherwise as many ranges as blocks fit, each of at
// least 12 tiles: one sequence of 16384 keys, 4 K/V heads 14.4 us with 16 and
// 15.9 with 8; 2000 keys, 12 heads 10.2 us with 4, 10.7 with 8, 14.4 with 32.
int masked_rows_ranges(int64_t items, int64_t max_k, int group, int head_dim) {
    const int64_t tiles = ceil_div(max_k, 16);
    const int64_t capacity = 148 * ((head_dim == 64 ? 4 : 3) - (group > 8 ? 1 : 0));
    if (tiles <= 32 || items >= 4 * capacity) return 0;
    return static_cast<int>(std::max<int64_t>(1, std::min(capacity, items * tiles / 12)));
}

int masked_attention_rows(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype) {
    if (dtype == P3D_BF16)
        return head_dim == 64 ? launch_heads<__nv_bfloat16, 64>(ctx, p) : launch_heads<__nv_bfloat16, 128>(ctx, p);
    return head_dim == 64 ? launch_heads<__half, 64>(ctx, p) : launch_heads<__half, 128>(ctx, p);
}

}  // namespace p3d
