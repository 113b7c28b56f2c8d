// Masked attention for few query rows over long keys.
//
// The work is reading K and V once: 4 d bytes a key and K/V head at 4 d
// operations for each row, a row being a query and one of the heads that share
// the K/V head.  An item is one sequence's K/V head with up to 8 HT of its
// rows, and is cut into pieces of equal length.  Block b of G takes the pieces
// b, b + G, b + 2 G, ... in the order sequence, piece, item: blocks that run
// side by side then read the same keys of neighbouring heads, which lie side
// by side in memory (pieces in item order, every block at its own place, read
// 16 sequences of up to 8192 keys, 16 heads of 64, at 4.0 instead of 5.0 TB/s),
// and the sequences' lengths do not matter.  A second kernel joins the pieces.
// A block is a TMA producer, which keeps whole stages of 128 or 256 keys of K
// and V in flight across its pieces, and 8 warps that take 16 or 32 keys of a
// stage each, with their own running maxima and sums, joined when the piece
// ends.
//
// Scores are S[row][key] = Q K^T (m16n8k16), the output O^T[dim][row] += V^T
// P^T with 8 rows as columns: S's accumulator layout, row lane / 4 and columns
// 2 (lane % 4) + {0, 1}, is the layout of the second product's B operand, so
// the weights go from one to the other inside a lane.  A contraction may take
// its index in any order and a row any name: lane (g, j) = (lane / 4, lane % 4)
// reads 16 bytes, dims 32 c + 8 j .. + 7 of key g, and uses them as the k
// indices of two products; for V it reads dims 64 s + 8 g .. + 7 of the keys
// 2j, 2j + 1, 2j + 8, 2j + 9, and product i has dims 64 s + 8 g + 2 i and + 1
// as its rows g and g + 8.
//
// Hidden places: a tile that every row sees needs no mask; in others a hidden
// score is -inf whatever it was, and since 0 * NaN is NaN, infinities and NaN
// of the tile's V leave the product and are then added to the rows that see
// them.  Every wait is bounded.
#include <algorithm>
#include <type_traits>

#include "p3d_masked_small.cuh"

namespace p3d {
namespace {

constexpr int kWarps = 8;                       // consumers
constexpr int kThreads = 32 * (kWarps + 1);     // and the producer

template <int D, int HT>
struct Cfg {
    static constexpr int TPW = D == 64 ? 2 : 1;        // 16-key tiles of a warp and stage
    static constexpr int TILES = TPW * kWarps;         // of a stage
    static constexpr int KEYS = 16 * TILES;
    static constexpr int SUB = KEYS * 128;             // KEYS x 64 dims, 128-byte rows in the 128-byte swizzle
    static constexpr int KC = D / 32, VS = D / 64, SUBS = D / 64;
    static constexpr int ROWS = 8 * HT;
    static constexpr int NF = VS * 4 * HT;       // accumulator quadruples of a lane
    static constexpr int STAGE = 2 * SUBS * SUB;
    static constexpr int Q_BYTES = HT * KC * 512;
    static constexpr int JOIN = (kWarps / 2) * (NF * 512 + HT * 256);
    static constexpr int FIT = (232448 - Q_BYTES - JOIN - 1024 - 256) / STAGE;
    static constexpr int STAGES = FIT > 6 ? 6 : FIT;
    static constexpr int SMEM = STAGES * STAGE + Q_BYTES + JOIN + 1024 + 256;
    static_assert(STAGES >= 2 && SMEM <= 232448, "shared memory");
};

// Key tiles of an item (at least one, so that every item has a piece), a
// sequence's rows of one K/V head, its items and all their pieces.
__device__ __forceinline__ int item_tiles(const SeqRange &sr) { return max(1, (sr.lk + 15) / 16); }
__device__ __forceinline__ int seq_rows(const MaskedParams &p, const SeqRange &sr) {
    return static_cast<int>(min(static_cast<int64_t>(sr.lq), p.max_q)) * p.group;
}
__device__ __forceinline__ int seq_items(const MaskedParams &p, const SeqRange &sr) {
    return (seq_rows(p, sr) + p.item_rows - 1) / p.item_rows * p.kv_heads;
}
// Pieces of an item, and their tiles: p.piece, or, in a sequence longer than
// max_k, as many as leave it no more pieces than one of max_k keys has (the
// results' space is of that many; the last ones may be empty).
__device__ __forceinline__ int item_pieces(const MaskedParams &p, const SeqRange &sr) {
    return min((item_tiles(sr) + p.piece - 1) / p.piece, p.most_pieces);
}
__device__ __forceinline__ int piece_tiles(const MaskedParams &p, const SeqRange &sr) {
    return max(p.piece, (item_tiles(sr) + p.most_pieces - 1) / p.most_pieces);
}

// Places in the order of all pieces (whole warps call these).
struct Walk {
    int64_t u = 0, before = 0;  // the piece, and the pieces before its sequence
    SeqRange sr;
    int seq = 0, items = 0, pieces = 0, length = 0;
    int item, t, take;  // of the piece: its item, first key tile, tiles
    bool whole;         // the item's only piece

    // From sequence `seq` on: the one that holds piece u, or the sequence
    // `want`; false past the last.
    __device__ __forceinline__ bool find(const MaskedParams &p, int lane, int want = -1) {
        for (; seq < p.nseq; seq += 32) {
            int64_t n = 0;
            if (seq + lane < p.nseq) {
                const SeqRange s = seq_range(p, seq + lane);
                n = static_cast<int64_t>(seq_items(p, s)) * item_pieces(p, s);
            }
            int64_t upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t a = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += a;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, want >= 0 ? seq + lane == want : before + upto > u);
            if (hit) {
                const int l = __ffs(hit) - 1;
                before += __shfl_sync(0xffffffffu, upto - n, l);
                seq += l;
                sr = seq_range(p, seq);
                items = seq_items(p, sr);
                pieces = item_pieces(p, sr);
                length = piece_tiles(p, sr);
                return true;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        return false;
    }
    // To piece u (not before the present one); false past the last.
    __device__ __forceinline__ bool go(const MaskedParams &p, int lane, int64_t to) {
        u = to;
        if (u >= before + static_cast<int64_t>(items) * pieces && !find(p, lane)) return false;
        const int in = static_cast<int>(u - before);
        item = in % items;
        t = in / items * length;
        take = max(min(length, item_tiles(sr) - t), 0);
        whole = pieces == 1;
        return true;
    }
};

// Infinity or NaN in the low half.
template <typename T>
__device__ __forceinline__ bool odd16(uint32_t h) {
    constexpr uint32_t e = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
    return (h & e) == e;
}

template <typename T, int D, int HT>
__global__ void __launch_bounds__(kThreads, 1)
    masked_pieces_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const MaskedParams p) {
    using C = Cfg<D, HT>;
    constexpr int KC = C::KC, VS = C::VS, ST = C::STAGES, MT = (HT + 1) / 2, TPW = C::TPW, NT = 2 * TPW;  // NT: 8-key columns
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *stages = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint4 *sq = reinterpret_cast<uint4 *>(stages + ST * C::STAGE);                // [HT][KC][lane]
    float4 *so = reinterpret_cast<float4 *>(stages + ST * C::STAGE + C::Q_BYTES);  // [kWarps / 2][NF][lane]
    float2 *sml = reinterpret_cast<float2 *>(so + (kWarps / 2) * C::NF * 32);      // [kWarps / 2][HT][lane]
    uint64_t *full = reinterpret_cast<uint64_t *>(sml + (kWarps / 2) * HT * 32), *empty = full + ST;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kWarps);
        }
        fence_barrier_init();
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    Walk at;
    const bool any = at.go(p, lane, blockIdx.x);  // every warp finds the same
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;

    if (warp == kWarps) {
        // ---------------------------------------------------------- producer
        for (bool more = any; more && ok; more = at.go(p, lane, at.u + gridDim.x)) {
            const int hk = at.item % p.kv_heads;
            for (int t = at.t; t < at.t + at.take && ok; t += C::TILES) {
                if (lane == 0) {
                    ok = mbar_wait(&empty[stage], phase ^ 1, p.fault);
                    if (ok) {
                        uint8_t *b = stages + stage * C::STAGE;
                        mbar_arrive_expect_tx(&full[stage], C::STAGE);
#pragma unroll
                        for (int s = 0; s < C::SUBS; ++s)
                            tma_load_2d(b + s * C::SUB, &tk, &full[stage], hk * D + s * 64, at.sr.k0 + t * 16);
#pragma unroll
                        for (int s = 0; s < C::SUBS; ++s)
                            tma_load_2d(b + (C::SUBS + s) * C::SUB, &tv, &full[stage], hk * D + s * 64, at.sr.k0 + t * 16);
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                if (++stage == ST) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        return;
    }

    // --------------------------------------------------------------- consumers
    // A warp whose wait ran out computes no further but keeps every barrier.
    const int g = lane >> 2, j = lane & 3;
    auto barrier = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    for (bool more = any; more; more = at.go(p, lane, at.u + gridDim.x)) {
        const SeqRange sr = at.sr;
        const int hk = at.item % p.kv_heads, row0 = at.item / p.kv_heads * p.item_rows;
        const int rows = min(C::ROWS, seq_rows(p, sr) - row0);
        const int shift = sr.lk - sr.lq;
        const int pre = p.prefix ? min(max(p.prefix[at.seq], 0), sr.lk) : 0;
        auto edge_of = [&](int pos) { return p.causal ? min(sr.lk, max(pre, pos + 1)) : sr.lk; };
        const int edge_lo = edge_of(row0 / p.group + shift), edge_hi = edge_of((row0 + rows - 1) / p.group + shift);
        // rows g + 8 r of this lane
        int pos[HT], edge[HT], docq[HT];
        float slope[HT];
#pragma unroll
        for (int r = 0; r < HT; ++r) {
            const int row = row0 + min(g + 8 * r, rows - 1);
            const int qi = row / p.group;
            pos[r] = qi + shift;
            edge[r] = edge_of(pos[r]);
            docq[r] = p.doc_q ? p.doc_q[sr.q0 + qi] : 0;
            slope[r] = p.slopes ? p.slopes[hk * p.group + row % p.group] * 1.4426950408889634f : 0.0f;
        }
        auto sees = [&](int key, int r) {
            return key < edge[r] && (key < pre || !p.doc_k || ((!p.causal || key <= pos[r]) && p.doc_k[sr.k0 + key] == docq[r]));
        };
        // Q as the first product's operand
        for (int e = threadIdx.x; e < HT * KC * 32; e += 32 * kWarps) {
            const int l = e & 31, c = e / 32 % KC, r = e / (32 * KC), in = (l >> 2) + 8 * r, row = row0 + in;
            sq[e] = in < rows ? *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.q) + (sr.q0 + static_cast<int64_t>(row / p.group)) * p.ldq +
                                                                  static_cast<int64_t>(hk * p.group + row % p.group) * D + c * 32 + (l & 3) * 8)
                              : make_uint4(0, 0, 0, 0);
        }
        barrier();

        float o[VS][4][HT][4];  // [slab][product][8 rows]: (dim, row 2j), (dim, 2j + 1), (dim + 1, 2j), (dim + 1, 2j + 1)
        float m[HT], l[HT];
#pragma unroll
        for (int r = 0; r < HT; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
#pragma unroll
            for (int s = 0; s < VS; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[s][i][r][e] = 0.0f;
        }
        const int key_end = (at.t + at.take) * 16;  // keys from here on are another piece's
        for (int t0 = at.t; t0 < at.t + at.take; t0 += C::TILES) {
            const int k0 = (t0 + warp * TPW) * 16;
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, p.fault));
            const bool mine = ok && k0 < min(key_end, edge_hi);
            // every row sees every key
            const bool all = k0 + 16 * TPW <= min(key_end, edge_lo) && (!p.doc_k || k0 + 16 * TPW <= pre);
            if (mine) {
                const uint8_t *kb = stages + stage * C::STAGE + warp * TPW * 16 * 128;
                const uint8_t *vb = kb + C::SUBS * C::SUB;
                float sc[MT][NT][4];
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[a][t][e] = 0.0f;
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    uint4 kf[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        kf[t] = *reinterpret_cast<const uint4 *>(kb + (c >> 1) * C::SUB + (t * 8 + g) * 128 + ((((c & 1) * 4 + j) ^ g) << 4));
#pragma unroll
                    for (int a = 0; a < MT; ++a) {
                        const uint4 lo = sq[(2 * a * KC + c) * 32 + lane];
                        const uint4 hi = 2 * a + 1 < HT ? sq[((2 * a + 1) * KC + c) * 32 + lane] : make_uint4(0, 0, 0, 0);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t q[4] = {word(lo, 2 * h), word(hi, 2 * h), word(lo, 2 * h + 1), word(hi, 2 * h + 1)};
#pragma unroll
                            for (int t = 0; t < NT; ++t) mma16816<T>(sc[a][t], q, word(kf[t], 2 * h), word(kf[t], 2 * h + 1));
                        }
                    }
                }
                bool raised = false;
                float mx[HT];
#pragma unroll
                for (int r = 0; r < HT; ++r) {
                    mx[r] = -INFINITY;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int key = k0 + t * 8 + 2 * j + e;
                            float x = sc[r / 2][t][2 * (r & 1) + e];
                            x = p.c1 > 0.0f ? capped(x, p.c0, p.c1) : x * p.c0;
                            if (p.slopes) x = fmaf(-slope[r], static_cast<float>(abs(pos[r] - key)), x);
                            if (!all) x = key < key_end && sees(key, r) ? x : -INFINITY;
                            sc[r / 2][t][2 * (r & 1) + e] = x;
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
                        const float a0 = __shfl_sync(0xffffffffu, a, 8 * j), a1 = __shfl_sync(0xffffffffu, a, 8 * j + 4);  // rows 2j, 2j + 1
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
                uint32_t pf[HT][NT];
#pragma unroll
                for (int r = 0; r < HT; ++r) {
                    const float base = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        pf[r][t] = pack2<T>(ex2f(sc[r / 2][t][2 * (r & 1)] - base), ex2f(sc[r / 2][t][2 * (r & 1) + 1] - base));
                        const float2 f = unpack2<T>(pf[r][t]);  // the sum takes the weights as the product sees them
                        l[r] += f.x + f.y;
                    }
                }
#pragma unroll
                for (int us = 0; us < TPW * VS; ++us) {
                    const int u = us / VS, s = us % VS;  // tile, slab
                    uint4 vf[4];
                    bool odd = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = 2 * j + (e & 1) + (e >> 1) * 8;
                        vf[e] = *reinterpret_cast<const uint4 *>(vb + s * C::SUB + (u * 16 + key) * 128 + ((g ^ (key & 7)) << 4));
                    }
                    if (!all) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int i = 0; i < 4; ++i) odd |= odd16<T>(word(vf[e], i)) || odd16<T>(word(vf[e], i) >> 16);
                        odd = __any_sync(0xffffffffu, odd);
                    }
                    uint32_t w[4][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[e][i] = word(vf[e], i);
                    if (odd) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll 1
                            for (int jj = 0; jj < 4; ++jj) {
                                const int key = k0 + u * 16 + 2 * jj + (e & 1) + (e >> 1) * 8;
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const uint32_t v = __shfl_sync(0xffffffffu, word(vf[e], i), (lane & ~3) | jj);
                                    const float2 f = unpack2<T>(v);
#pragma unroll
                                    for (int r = 0; r < HT; ++r)
#pragma unroll
                                        for (int h = 0; h < 2; ++h) {
                                            const int row = row0 + min(8 * r + 2 * j + h, rows - 1), qi = row / p.group, at_q = qi + shift;
                                            const bool seen = key < key_end && key < edge_of(at_q) &&
                                                              (key < pre || !p.doc_k || ((!p.causal || key <= at_q) &&
                                                                                         p.doc_k[sr.k0 + key] == p.doc_q[sr.q0 + qi]));
                                            if (seen && !isfinite(f.x)) o[s][i][r][h] += f.x;
                                            if (seen && !isfinite(f.y)) o[s][i][r][2 + h] += f.y;
                                        }
                                }
                            }
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (odd16<T>(w[e][i])) w[e][i] &= 0xffff0000u;
                                if (odd16<T>(w[e][i] >> 16)) w[e][i] &= 0x0000ffffu;
                            }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t a[4] = {__byte_perm(w[0][i], w[1][i], 0x5410u), __byte_perm(w[0][i], w[1][i], 0x7632u),
                                               __byte_perm(w[2][i], w[3][i], 0x5410u), __byte_perm(w[2][i], w[3][i], 0x7632u)};
#pragma unroll
                        for (int r = 0; r < HT; ++r) mma16816<T>(o[s][i][r], a, pf[r][2 * u], pf[r][2 * u + 1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
            if (++stage == ST) {
                stage = 0;
                phase ^= 1;
            }
        }
        // join the warps: the upper half of those left hands over to the lower
#pragma unroll
        for (int r = 0; r < HT; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
#pragma unroll 1
        for (int n = kWarps / 2; n > 0; n >>= 1) {
            if (warp >= n && warp < 2 * n) {
#pragma unroll
                for (int s = 0; s < VS; ++s)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < HT; ++r)
                            so[((warp - n) * C::NF + (s * 4 + i) * HT + r) * 32 + lane] =
                                make_float4(o[s][i][r][0], o[s][i][r][1], o[s][i][r][2], o[s][i][r][3]);
#pragma unroll
                for (int r = 0; r < HT; ++r) sml[((warp - n) * HT + r) * 32 + lane] = make_float2(m[r], l[r]);
            }
            barrier();
            if (warp < n) {
#pragma unroll
                for (int r = 0; r < HT; ++r) {
                    const float2 ml = sml[(warp * HT + r) * 32 + lane];
                    const float mn = fmaxf(m[r], ml.x), base = mn == -INFINITY ? 0.0f : mn;
                    const float a = ex2f(m[r] - base), b = ex2f(ml.x - base);
                    m[r] = mn;
                    l[r] = l[r] * a + ml.y * b;
                    const float a0 = __shfl_sync(0xffffffffu, a, 8 * j), a1 = __shfl_sync(0xffffffffu, a, 8 * j + 4);
                    const float b0 = __shfl_sync(0xffffffffu, b, 8 * j), b1 = __shfl_sync(0xffffffffu, b, 8 * j + 4);
#pragma unroll
                    for (int s = 0; s < VS; ++s)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 f = so[(warp * C::NF + (s * 4 + i) * HT + r) * 32 + lane];
                            o[s][i][r][0] = o[s][i][r][0] * a0 + f.x * b0;
                            o[s][i][r][1] = o[s][i][r][1] * a1 + f.y * b1;
                            o[s][i][r][2] = o[s][i][r][2] * a0 + f.z * b0;
                            o[s][i][r][3] = o[s][i][r][3] * a1 + f.w * b1;
                        }
                }
            }
            barrier();
        }
        if (warp == 0) {
            const bool whole = at.whole;
            const int64_t part = at.u;
#pragma unroll
            for (int r = 0; r < HT; ++r) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int in = 8 * r + 2 * j + h;
                    const float sum = __shfl_sync(0xffffffffu, l[r], 8 * j + 4 * h);
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    if (in >= rows || !ok || (!whole && part >= p.parts)) continue;
                    const int row = row0 + in;
#pragma unroll
                    for (int s = 0; s < VS; ++s) {
                        float y[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            y[2 * i] = o[s][i][r][h];
                            y[2 * i + 1] = o[s][i][r][2 + h];
                        }
                        if (whole) {
                            T *dst = static_cast<T *>(p.out) + (sr.q0 + static_cast<int64_t>(row / p.group)) * p.ldo +
                                     static_cast<int64_t>(hk * p.group + row % p.group) * D + s * 64 + g * 8;
                            *reinterpret_cast<uint4 *>(dst) =
                                make_uint4(pack2<T>(y[0] * inv, y[1] * inv), pack2<T>(y[2] * inv, y[3] * inv),
                                           pack2<T>(y[4] * inv, y[5] * inv), pack2<T>(y[6] * inv, y[7] * inv));
                        } else {
                            float4 *dst = reinterpret_cast<float4 *>(p.part_o + (part * p.item_rows + in) * D + s * 64 + g * 8);
                            dst[0] = make_float4(y[0], y[1], y[2], y[3]);
                            dst[1] = make_float4(y[4], y[5], y[6], y[7]);
                        }
                    }
                }
                if (!whole && j == 0 && part < p.parts) p.part_ml[part * p.item_rows + 8 * r + g] = make_float2(m[r], l[r]);
            }
            __syncwarp();
        }
    }
}

constexpr int kJoinWarps = 4;
// A block joins the parts of one query and head.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) masked_join_kernel(const MaskedParams p) {
    constexpr int E = D / 32;
    __shared__ float so[kJoinWarps][D];
    __shared__ float2 sml[kJoinWarps];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x % p.heads, qi = blockIdx.x / p.heads, seq = blockIdx.y;
    const SeqRange sr = seq_range(p, seq);
    if (qi >= sr.lq) return;
    const int row = qi * p.group + head % p.group, r = row % p.item_rows;
    Walk at;
    at.find(p, lane, seq);
    const int n = at.pieces;
    if (n == 1) return;  // written by the block that had it
    const int64_t first = at.before + row / p.item_rows * p.kv_heads + head / p.group;
    if (first + static_cast<int64_t>(n - 1) * at.items >= p.parts) return;  // offsets that overlap: more pieces than rows_k holds
    auto part = [&](int piece) { return (first + static_cast<int64_t>(piece) * at.items) * p.item_rows + r; };
    float mm = -INFINITY;
    for (int b = lane * kJoinWarps + warp; b < n; b += 32 * kJoinWarps) mm = fmaxf(mm, p.part_ml[part(b)].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    const float base = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, oo[E] = {};
#pragma unroll 8
    for (int b = warp; b < n; b += kJoinWarps) {
        const float2 ml = p.part_ml[part(b)];
        const float a = ex2f(ml.x - base);
        ll = fmaf(ml.y, a, ll);
        const float *src = p.part_o + part(b) * D + lane * E;
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
        for (int k = 0; k < kJoinWarps; ++k) top = fmaxf(top, sml[k].x);
        const float b = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int k = 0; k < kJoinWarps; ++k) {
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
int launch_pieces(p3d_ctx *ctx, const MaskedParams &p, int dtype) {
    using C = Cfg<D, HT>;
    CUtensorMap tk, tv;
    int rc = make_tmap_16bit_2d(ctx, &tk, p.k, dtype, p.rows_k, static_cast<uint64_t>(p.kv_heads) * D, p.ldk, C::KEYS);
    if (rc || (rc = make_tmap_16bit_2d(ctx, &tv, p.v, dtype, p.rows_k, static_cast<uint64_t>(p.kv_heads) * D, p.ldv, C::KEYS))) return rc;
    auto kernel = masked_pieces_kernel<T, D, HT>;
    P3D_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    P3D_CUDA(ctx, launch_pdl(kernel, dim3(p.blocks), dim3(kThreads), C::SMEM, ctx->stream, tk, tv, p));
    if ((rc = check_launch(ctx, "masked_pieces"))) return rc;
    P3D_CUDA(ctx, launch_pdl(masked_join_kernel<T, D>, dim3(static_cast<unsigned>(p.max_q * p.heads), p.nseq), dim3(32 * kJoinWarps), 0,
                             ctx->stream, p));
    return check_launch(ctx, "masked_join");
}

template <typename T, int D>
int launch_rows(p3d_ctx *ctx, const MaskedParams &p, int dtype) {
    if (p.item_rows == 8) return launch_pieces<T, D, 1>(ctx, p, dtype);
    if constexpr (D == 64) {
        if (p.item_rows == 24) return launch_pieces<T, D, 3>(ctx, p, dtype);
    }
    return launch_pieces<T, D, 2>(ctx, p, dtype);
}

}  // namespace

int masked_attention_pieces(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype) {
    if (dtype == P3D_BF16) return head_dim == 64 ? launch_rows<__nv_bfloat16, 64>(ctx, p, dtype) : launch_rows<__nv_bfloat16, 128>(ctx, p, dtype);
    return head_dim == 64 ? launch_rows<__half, 64>(ctx, p, dtype) : launch_rows<__half, 128>(ctx, p, dtype);
}

}  // namespace p3d
