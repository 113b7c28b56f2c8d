#pragma once

// Masked attention on tcgen05 tensor cores, for many query rows.
//
// A CTA takes 128 queries of one head and the key blocks (64 keys) that any of
// them sees; two CTAs share an SM (256 TMEM columns each), so one's softmax
// runs beside the other's products.  6 warps:
//   warp 0     finds the blocks to visit and loads them (TMA): 32 blocks are
//              classified at a time as hidden, seen by every query, or mixed,
//              from the positions and the documents' smallest and largest
//              number in the block; hidden blocks are neither read nor computed
//   warp 1     TMEM allocator, one thread issues the MMAs
//   warps 2-5  softmax: thread = query = TMEM lane
// Per visited block i (buffer b = i & 1): S_b = Q K^T; the softmax threads read
// their row, apply the score rules (and, in mixed blocks only, the mask), and
// write P_b over S_b as 16-bit; O += P_b V with P from TMEM.  The running
// maximum is raised lazily: O and the sum are rescaled when a block's maximum
// exceeds it by more than 8 (2^8 in P; f16: 2^15, as the maximum is held lower),
// which keeps P within 16-bit range and the result exact, as both are taken
// against the same maximum.  The sum takes the weights as the product does,
// rounded: at 64 dims it is a column of that product (V beside a tile of ones,
// N = 80), at 128, where no TMEM is left for it, 16-bit numbers added to f32 ones
// (2 x 4092, 16 heads of 64, causal behind a prefix: error against 64 bits 1.26
// times one rounding of the result's, 1.37 with the sum of the unrounded weights;
// 141 -> 137 us; 16384 in 5 documents, 16 of 128: 1.11 and 1.18 times, 587 -> 596).
//
// Hidden places: a hidden score is replaced by -inf whatever it was, but a
// hidden key's V still meets P = 0 in the product, and 0 * NaN is NaN.  So the
// V tile of a mixed block is searched for infinities and NaN before its
// product; what is found is set to zero in shared memory and the block noted,
// and at the end each query adds the noted blocks' non-finite values that it
// does see.  Blocks that every query sees need none of this.
//
// Documents: the CTAs take the tiles with the most visits first, from an order
// that a kernel before this one found, with the tiles' documents.
//
// Few CTAs over long keys: the visits are cut into splits, whose sums against
// their own maxima a second kernel joins (one sequence of 64 queries, 16 heads
// of 64, 8192 keys: 106 us without, 21.7 with).
//
// Rows past the sequence's end compute on whatever the tile holds and are not
// stored.  Every wait is bounded.
#include <type_traits>

#include "p3d_fmha.cuh"
#include "p3d_masked.cuh"

namespace p3d {
namespace {

constexpr int kM = 128;
constexpr int kN = 64;
constexpr int kThreadsF = 192;
constexpr float kRescaleLog2 = 8.0f;
constexpr int kSub = kN * 128;    // one 64-key x 64-dim operand tile, 128-byte rows
constexpr int kTags = 8;          // unread tags: at most stages + 2
constexpr uint32_t kTmemCols = 256;
constexpr uint32_t kOCol = 128;   // S/P 0 (64) | S/P 1 (64) | O (up to 128; 64 dims: and the sum of weights)
constexpr int kSmem = 100 * 1024;  // more than a third of an SM's: never a third CTA waiting for TMEM

template <int D>
struct Cfg {
    static constexpr int SUBS = D / 64;
    static constexpr int Q_BYTES = SUBS * kM * 128;
    static constexpr int KV_BYTES = SUBS * kSub;
    static constexpr int STAGES = D == 64 ? 4 : 2;  // of K, and of V
    // The sum of weights: 64 dims leave TMEM columns for a product with ones (the
    // 16 columns behind O); 128 dims fill them, and the softmax threads add up.
    static constexpr bool ONES = D == 64;
    static constexpr int ONES_BYTES = ONES ? kSub : 0;
    static constexpr uint32_t L_COL = kOCol + D;
    static_assert(Q_BYTES + 2 * STAGES * KV_BYTES + ONES_BYTES + 1024 + 512 + 4 * kN * 4 <= kSmem, "shared memory");
    static_assert(!ONES || L_COL + 16 <= kTmemCols, "TMEM");
    static_assert(STAGES + 2 <= kTags, "tag ring");
};

__device__ __forceinline__ float min3f(float a, float b, float c) {
    float r;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float row_min64(const float (&s)[64]) {
    float m[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        m[c] = s[c];
#pragma unroll
        for (int e = 4 + c; e < 60; e += 8) m[c] = min3f(m[c], s[e], s[e + 4]);
        m[c] = fminf(m[c], s[60 + c]);
    }
    return fminf(min3f(m[0], m[1], m[2]), m[3]);
}

// a += the low, b += the high half of a packed pair.
template <typename T>
__device__ __forceinline__ void add_pair(float &a, float &b, uint32_t w) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tadd.rn.f32.bf16 %0, lo, %0;\n\tadd.rn.f32.bf16 %1, hi, %1;\n\t}"
            : "+f"(a), "+f"(b)
            : "r"(w));
    else
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tadd.rn.f32.f16 %0, lo, %0;\n\tadd.rn.f32.f16 %1, hi, %1;\n\t}"
            : "+f"(a), "+f"(b)
            : "r"(w));
}

// Infinities and NaN of a packed pair set to zero.
template <typename T>
__device__ __forceinline__ void clean_pair(uint32_t &w) {
    constexpr uint32_t e = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
    const bool lo = (w & e) == e, hi = ((w >> 16) & e) == e;
    if (lo) w &= 0xffff0000u;
    if (hi) w &= 0x0000ffffu;
}

// Whether a vector holds any infinity or NaN: an exponent of ones leaves a zero
// half, and a borrow out of one marks the vector whichever half it was.
template <typename T>
__device__ __forceinline__ bool any_nonfinite(const uint4 &u) {
    constexpr uint32_t e = std::is_same<T, __nv_bfloat16>::value ? 0x7f807f80u : 0x7c007c00u;
    auto zero_half = [](uint32_t w) {
        const uint32_t t = (w & e) ^ e;
        return (t - 0x00010001u) & ~t;
    };
    return ((zero_half(u.x) | zero_half(u.y) | zero_half(u.z) | zero_half(u.w)) & 0x80008000u) != 0;
}

// Scores to capped scores, as capped(): each by its polynomial or, beyond half
// the cap, by the exponential and a reciprocal, which with the weights' own
// exponential are three operations of the XU pipe for each score instead of one
// (8192 x 8192, 16 heads of 128: 584 us, 1145 with far scores in every block;
// that form for all scores of such a block 1074).  Where no score of the
// warp's rows is far the second form is left out; where one is, the others still
// take the polynomial, whose error goes with the score and not with the cap
// (the far one may be another row's, or a hidden key's).
__device__ __forceinline__ void cap_row(float (&s)[64], float c0, float c1) {
    const float ct = c0 * kCapT;
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < 64; e += 4) {
        mul2(F2(s[e], s[e + 1]), F2(ct, ct)).get(s[e], s[e + 1]);
        mul2(F2(s[e + 2], s[e + 3]), F2(ct, ct)).get(s[e + 2], s[e + 3]);
        top = max3f(max3f(top, fabsf(s[e]), fabsf(s[e + 1])), fabsf(s[e + 2]), fabsf(s[e + 3]));
    }
    const float k0 = kCap0 * c1, k1 = kCap1 * c1, k2 = kCap2 * c1, k3 = kCap3 * c1;
    if (__all_sync(0xffffffffu, top <= 0.5f)) {
#pragma unroll
        for (int e = 0; e < 64; e += 2) {
            const F2 t(s[e], s[e + 1]);
            const F2 u = mul2(t, t);
            const F2 q = fma2(fma2(fma2(u, F2(k3, k3), F2(k2, k2)), u, F2(k1, k1)), u, F2(k0, k0));
            mul2(t, q).get(s[e], s[e + 1]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 64; ++e) {
            float t = s[e];
            asm volatile("" : "+f"(t));  // in order: no more registers than the near form
            const float u = t * t, f = capped_far(t, c1);
            const float x = t * fmaf(fmaf(fmaf(u, k3, k2), u, k1), u, k0);
            s[e] = fabsf(t) <= 0.5f ? x : f;
        }
    }
}

// The polynomial of near capped scores with its factors folded in: the capped
// score in units of log2 is s (f0 + u (f1 + u (f2 + u f3))), u = s^2, for
// |s| <= top; top < 0 where a factor would leave 32 bits' range.
struct NearCap {
    float f0, f1, f2, f3, top;
    __device__ __forceinline__ NearCap(float c0, float c1) {
        const float ct = c0 * kCapT, cc = ct * ct;
        f0 = kCap0 * c1 * ct;
        f1 = kCap1 * c1 * ct * cc;
        f2 = kCap2 * c1 * ct * cc * cc;
        f3 = kCap3 * c1 * ct * cc * cc * cc;
        const bool fits = fabsf(f0) > 1e-30f && fabsf(f0) < 1e30f && fabsf(f3) > 1e-30f && fabsf(f3) < 1e30f;
        top = fits ? 0.5f / ct : -1.0f;
    }
};

// s scale - slope |d - e| for the 64 keys e of a block, d the query's position
// relative to the block's first key.  A block that lies on one side of all of
// the warp's queries needs no absolute value.
__device__ __forceinline__ void bias_row(float (&s)[64], float scale, float slope, int d) {
    const float df = static_cast<float>(d);
    const bool left = __all_sync(0xffffffffu, d >= 63), right = __all_sync(0xffffffffu, d <= 0);
    if (left || right) {
        const float step = left ? slope : -slope, base = -step * df;  // its rounding, 2^-24 of slope d, is the one that the other form lacks
#pragma unroll
        for (int e = 0; e < 64; e += 2)
            fma2(F2(s[e], s[e + 1]), F2(scale, scale),
                 F2(fmaf(step, static_cast<float>(e), base), fmaf(step, static_cast<float>(e + 1), base)))
                .get(s[e], s[e + 1]);
    } else {
#pragma unroll
        for (int e = 0; e < 64; ++e) s[e] = fmaf(s[e], scale, -slope * fabsf(df - static_cast<float>(e)));
    }
}

// First of the splits' results of query qi (below max_q) of a sequence: by the
// sequence's place, not by the row, since q may hold many more rows.
__device__ __forceinline__ int64_t split_part(const MaskedParams &p, int seq, int64_t qi, int head) {
    return ((seq * p.max_q + qi) * p.heads + head) * p.splits;
}

template <typename T, int D, bool CAP, bool BIAS, bool DOCS>
__global__ void __launch_bounds__(kThreadsF, 2)
    masked_fmha_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const MaskedParams p) {
    using C = Cfg<D>;
    constexpr int ST = C::STAGES;
    pdl_wait();
    const int head = blockIdx.x;
    int seq = blockIdx.y;
    const int split = blockIdx.z % p.splits, z = blockIdx.z / p.splits, tiles = gridDim.z / p.splits;
    int tile = p.causal ? tiles - 1 - z : z;  // the longest rows first
    int qdoc_lo = 0, qdoc_hi = 0;  // documents of the tile's queries
    const bool ordered = DOCS && p.tile_order;
    if (ordered) {
        const int4 item = p.tile_order[z * p.nseq + seq];
        seq = item.w / tiles;
        tile = item.w % tiles;
        qdoc_lo = item.y;
        qdoc_hi = item.z;
    }
    const SeqRange sr = seq_range(p, seq);
    const int row0 = tile * kM;                       // first query of the tile, within the sequence
    const int nrows = min(min(sr.lq, static_cast<int>(p.max_q)) - row0, kM);
    if (nrows <= 0) return;
    const int hk = head / p.group;
    const int shift = sr.lk - sr.lq;                  // position of query i: i + shift
    const int pre = p.prefix ? min(max(p.prefix[seq], 0), sr.lk) : 0;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *sQ = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t *sK = sQ + C::Q_BYTES;
    uint8_t *sV = sK + ST * C::KV_BYTES;
    uint8_t *sOnes = sV + ST * C::KV_BYTES;
    uint64_t *q_full = reinterpret_cast<uint64_t *>(sOnes + C::ONES_BYTES);
    uint64_t *k_full = q_full + 1, *k_empty = k_full + ST, *v_full = k_empty + ST, *v_empty = v_full + ST;
    uint64_t *s_full = v_empty + ST, *p_full = s_full + 2, *pv_done = p_full + 2, *done_bar = pv_done + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done_bar + 1);
    volatile int *tags = reinterpret_cast<int *>(tmem_slot + 1);  // block << 2 | mixed << 1 | last
    volatile int *tag_lo = tags + kTags, *tag_hi = tag_lo + kTags;  // the block's documents
    int *any_seen = const_cast<int *>(tag_hi) + kTags;
    int *bad = any_seen + 1;  // first and last block with non-finite values taken out
    int *sdoc = reinterpret_cast<int *>((reinterpret_cast<uintptr_t>(bad + 2) + 15) & ~uintptr_t(15));  // [4 warps][64] document numbers

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < ST; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&s_full[b], 1);
            mbar_init(&p_full[b], 4);
            mbar_init(&pv_done[b], 1);
        }
        mbar_init(done_bar, 1);
        fence_barrier_init();
        bad[0] = 0x7fffffff;
        bad[1] = -1;
        prefetch_tmap(&tq);
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }

    // Blocks to visit (warp 0, all lanes alike): bit l of `seen` / `mixed` is
    // block chunk + l.
    const int pos_lo = row0 + shift, pos_hi = row0 + nrows - 1 + shift;
    const int limit = p.causal ? min(sr.lk, max(pre, pos_hi + 1)) : sr.lk;  // no query of the tile sees a key from here on
    const int blocks = max(0, (limit + kN - 1) / kN);
    // this split's share of the visits
    int chunk = static_cast<int>(static_cast<int64_t>(blocks) * split / p.splits);
    const int visits = static_cast<int>(static_cast<int64_t>(blocks) * (split + 1) / p.splits);
    uint32_t seen = 0, mixed = 0;
    int block_lo = 0, block_hi = 0;  // the smallest and largest document of the lane's block
    // The order of the visits.  Under a distance bias the scores of most rows
    // fall away from their own position, so the tile's own block comes first,
    // then those to its left, going away, then those to its right: the running
    // maximum is then raised a few times and not at every block.
    const int own_block = BIAS ? min(blocks - 1, max(0, pos_hi / kN)) : -1;
    auto block_at = [&](int visit) { return visit <= own_block ? own_block - visit : visit; };
    auto classify = [&]() {
        const bool in = chunk + lane < visits;
        const int blk = block_at(chunk + lane), kb = blk * kN;
        if (DOCS && in) {
            const int2 r = p.doc_range[doc_block(sr, seq) + blk];
            block_lo = r.x;
            block_hi = r.y;
        }
        const bool doc_meets = !DOCS || (block_lo <= qdoc_hi && qdoc_lo <= block_hi);
        const bool doc_all = !DOCS || (block_lo == block_hi && qdoc_lo == qdoc_hi && block_lo == qdoc_lo);
        const bool some = in && (kb < pre || doc_meets);
        const bool all = kb + kN <= sr.lk && (kb + kN <= pre || ((!p.causal || kb + kN - 1 <= pos_lo) && doc_all));
        seen = __ballot_sync(0xffffffffu, some);
        mixed = __ballot_sync(0xffffffffu, some && !all);
    };
    auto next_block = [&](bool &is_mixed, int &lo, int &hi) -> int {  // the next block to visit, or -1
        while (seen == 0) {
            chunk += 32;
            if (chunk >= visits) return -1;
            classify();
        }
        const int l = __ffs(seen) - 1;
        is_mixed = (mixed >> l) & 1;
        if constexpr (DOCS) {
            lo = __shfl_sync(0xffffffffu, block_lo, l);
            hi = __shfl_sync(0xffffffffu, block_hi, l);
        }
        seen &= seen - 1;
        return block_at(chunk + l);
    };
    bool cur_mixed = false;
    int cur = -1, cur_lo = 0, cur_hi = 0;
    if (warp == 0) {
        if (DOCS && !ordered) {
            int lo = 0x7fffffff, hi = -0x7fffffff - 1;
            for (int r = lane; r < nrows; r += 32) {
                const int d = p.doc_q[sr.q0 + row0 + r];
                lo = min(lo, d);
                hi = max(hi, d);
            }
            qdoc_lo = __reduce_min_sync(0xffffffffu, lo);
            qdoc_hi = __reduce_max_sync(0xffffffffu, hi);
        }
        if (chunk < visits) {
            classify();
            cur = next_block(cur_mixed, cur_lo, cur_hi);
        }
        if (lane == 0) *any_seen = cur >= 0;
    }
    if constexpr (C::ONES) {
        const uint32_t one2 = std::is_same<T, __nv_bfloat16>::value ? 0x3F803F80u : 0x3C003C00u;
        for (int e = threadIdx.x; e < C::ONES_BYTES / 16; e += kThreadsF)
            reinterpret_cast<uint4 *>(sOnes)[e] = make_uint4(one2, one2, one2, one2);
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();  // after the allocation: a dependent grid's CTA must not take this one's TMEM
    const uint32_t tmem = *tmem_slot;
    const bool nothing = *any_seen == 0;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;

    if (nothing && p.splits > 1) {
        for (int e = threadIdx.x; e < nrows; e += kThreadsF)
            p.part_ml[split_part(p, seq, row0 + e, head) + split] = make_float2(-INFINITY, 0.0f);
    } else if (nothing) {
        T *o = static_cast<T *>(p.out) + (sr.q0 + static_cast<int64_t>(row0)) * p.ldo + static_cast<int64_t>(head) * D;
        for (int e = threadIdx.x; e < nrows * (D / 8); e += kThreadsF)
            *reinterpret_cast<uint4 *>(o + (e / (D / 8)) * p.ldo + e % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
    } else if (warp == 0) {
        // ---------------------------------------------------------- producer
        if (lane == 0) {
            mbar_arrive_expect_tx(q_full, C::Q_BYTES);
#pragma unroll
            for (int s = 0; s < C::SUBS; ++s) tma_load_2d(sQ + s * kM * 128, &tq, q_full, head * D + s * 64, sr.q0 + row0);
        }
        int stage = 0;
        uint32_t phase = 0;
        for (int i = 0; cur >= 0; ++i) {
            bool nxt_mixed = false;
            int nxt_lo = 0, nxt_hi = 0;
            const int nxt = next_block(nxt_mixed, nxt_lo, nxt_hi);
            int ok = 1;
            if (lane == 0) {
                ok = mbar_wait(&k_empty[stage], phase ^ 1, p.fault);
                if (ok) {
                    tags[i % kTags] = cur << 2 | (cur_mixed ? 2 : 0) | (nxt < 0 ? 1 : 0);
                    if (DOCS && cur_mixed) {
                        tag_lo[i % kTags] = cur_lo;
                        tag_hi[i % kTags] = cur_hi;
                    }
                    mbar_arrive_expect_tx(&k_full[stage], C::KV_BYTES);
#pragma unroll
                    for (int s = 0; s < C::SUBS; ++s)
                        tma_load_2d(sK + stage * C::KV_BYTES + s * kSub, &tk, &k_full[stage], hk * D + s * 64, sr.k0 + cur * kN);
                    ok = mbar_wait(&v_empty[stage], phase ^ 1, p.fault);
                }
                if (ok) {
                    mbar_arrive_expect_tx(&v_full[stage], C::KV_BYTES);
#pragma unroll
                    for (int s = 0; s < C::SUBS; ++s)
                        tma_load_2d(sV + stage * C::KV_BYTES + s * kSub, &tv, &v_full[stage], hk * D + s * 64, sr.k0 + cur * kN);
                }
            }
            if (!__shfl_sync(0xffffffffu, ok, 0)) break;
            cur = nxt;
            cur_mixed = nxt_mixed;
            cur_lo = nxt_lo;
            cur_hi = nxt_hi;
            if (++stage == ST) {
                stage = 0;
                phase ^= 1;
            }
        }
    } else if (warp == 1) {
        // --------------------------------------------------------------- MMA
        if (lane == 0) {
            constexpr uint32_t idesc_s = idesc_f32acc(kM, kN, kBf16);
            constexpr uint32_t idesc_o = idesc_f32acc(kM, C::ONES ? D + 16 : D, kBf16, true);
            const uint32_t q_addr = smem_u32(sQ);
            bool ok = mbar_wait(q_full, 0, p.fault);
            auto issue_pv = [&](int i) -> bool {
                const int b = i & 1, st = i % ST;
                if (!mbar_wait(&v_full[st], (i / ST) & 1, p.fault) || !mbar_wait(&p_full[b], (i >> 1) & 1, p.fault)) return false;
                tc_fence_after();
                const uint32_t v_addr = smem_u32(sV + st * C::KV_BYTES);
                // columns 64 on of the V operand: the second half of its dims, or the ones
                const uint32_t next = C::ONES ? smem_u32(sOnes) - v_addr : kSub;
#pragma unroll
                for (int kk = 0; kk < kN / 16; ++kk)  // 16 keys: 8 packed TMEM columns of P, 2048 bytes of V
                    umma_f16_ts(tmem + kOCol, tmem + b * kN + kk * 8, sw128_desc_mn(v_addr + kk * 2048, next), idesc_o,
                                (i > 0 || kk > 0) ? 1u : 0u);
                umma_commit(&pv_done[b]);
                umma_commit(&v_empty[st]);
                return true;
            };
            for (int i = 0; ok; ++i) {
                const int b = i & 1, st = i % ST;
                if (!(ok = mbar_wait(&k_full[st], (i / ST) & 1, p.fault))) break;
                const bool last = tags[i % kTags] & 1;
                // S/P buffer b was last read by block i - 2's product
                if (i >= 2 && !(ok = mbar_wait(&pv_done[b], ((i - 2) >> 1) & 1, p.fault))) break;
                tc_fence_after();
                const uint32_t k_addr = smem_u32(sK + st * C::KV_BYTES);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_f16(tmem + b * kN, sw128_desc(q_addr + (kk / 4) * kM * 128 + (kk % 4) * 32),
                             sw128_desc(k_addr + (kk / 4) * kSub + (kk % 4) * 32), idesc_s, kk > 0 ? 1u : 0u);
                umma_commit(&s_full[b]);
                umma_commit(&k_empty[st]);
                if (i > 0 && !(ok = issue_pv(i - 1))) break;
                if (last) {
                    ok = issue_pv(i);
                    break;
                }
            }
            umma_commit(done_bar);
            mbar_wait(done_bar, 0, p.fault);
        }
        __syncwarp();
    } else {
        // ----------------------------------------------------------- softmax
        const int row = (warp & 3) * 32 + lane;  // TMEM lane quarter of the warp
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const int pos = row0 + row + shift;
        const bool valid = row < nrows;
        const int docq = DOCS && valid ? p.doc_q[sr.q0 + row0 + row] : 0;
        const float slope = BIAS ? p.slopes[head] * 1.4426950408889634f : 0.0f;
        const int edge = p.causal ? min(sr.lk, max(pre, pos + 1)) : sr.lk;  // keys seen where documents do not decide
        auto visible = [&](int j) -> bool {
            return j < edge && (j < pre || !DOCS || ((!p.causal || j <= pos) && p.doc_k[sr.k0 + j] == docq));
        };
        NearCap near(p.c0, p.c1);
        if (!valid) near.top = INFINITY;  // a row past the end has no say: what it holds changes no output's rounding
        float m_run = -INFINITY;
        float l0 = 0.0f, l1 = 0.0f;  // 128 dims: the sum of weights, even and odd keys
        bool ok = true;
        auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {  // warp-uniform: tcgen05.ld/st follow
            int r = 1;
            if (lane == 0) r = mbar_wait(bar, parity, p.fault) ? 1 : 0;
            return __shfl_sync(0xffffffffu, r, 0) != 0;
        };
        // documents of this warp's queries
        const int wdoc_lo = __reduce_min_sync(0xffffffffu, valid ? docq : 0x7fffffff);
        const int wdoc_hi = __reduce_max_sync(0xffffffffu, valid ? docq : -0x7fffffff - 1);
        int i = 0;
        for (;; ++i) {
            const int b = i & 1, st = i % ST;
            int tag = 0, lo = 0, hi = 0, n0 = 0, n1 = 0;
            // Not k_full for the tag: its next phase does not wait for these warps, and a
            // late one would miss its own.
            if (!(ok = wait(&s_full[b], (i >> 1) & 1))) break;
            tag = __shfl_sync(0xffffffffu, lane == 0 ? tags[i % kTags] : 0, 0);  // lane 0 has waited
            if (DOCS && (tag & 2)) {
                // The documents of a mixed block: most are of one, which came with the
                // tag (all loaded: 628 against 585 us for 16384 queries in 5 documents).
                lo = __shfl_sync(0xffffffffu, lane == 0 ? tag_lo[i % kTags] : 0, 0);
                hi = __shfl_sync(0xffffffffu, lane == 0 ? tag_hi[i % kTags] : 0, 0);
                if (lo != hi) {
                    const int j = (tag >> 2) * kN + lane;
                    n0 = p.doc_k[sr.k0 + min(j, sr.lk - 1)];
                    n1 = p.doc_k[sr.k0 + min(j + 32, sr.lk - 1)];
                }
            }
            const int j0 = (tag >> 2) * kN;
            bool some = true, all = !(tag & 2);  // whether this warp's queries see any key, every key of the block
            if (DOCS && !all) {
                some = j0 < pre || (lo <= wdoc_hi && wdoc_lo <= hi);
                all = j0 + kN <= sr.lk && (j0 + kN <= pre || ((!p.causal || j0 + kN - 1 <= pos - lane) && lo == hi &&
                                                               wdoc_lo == wdoc_hi && lo == wdoc_lo));
            }
            tc_fence_after();
            uint32_t pk[32];
            if (some) {
                float s[kN];
                {
                    float v0[32], v1[32];
                    tmem_ld32(tmem + lane_base + b * kN, v0);
                    tmem_ld32(tmem + lane_base + b * kN + 32, v1);
                    tmem_ld_wait_regs(v0);
                    tmem_ld_wait_regs(v1);
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        s[e] = v0[e];
                        s[32 + e] = v1[e];
                    }
                }
                // Near capped scores of a block that the mask leaves whole: the cap
                // rises with the score, so the maximum comes before it, and its last
                // product takes the subtraction in (5 operations a pair, not 7; 2 x 4092
                // queries, 16 heads of 64: 312 against 278 us; 8192, 16 of 128: 640
                // against 618; 8192 in 3 documents, 16 of 128: 302 against 290; where
                // documents are short and causal the spills of the two forms cost
                // more than it gives: 8000 in 7, 32 of 128, 210 against 221).
                bool folded = false;
                float mx = 0.0f;
                if constexpr (CAP && !BIAS) {
                    if (all) {
                        mx = row_max64(s);
                        folded = __all_sync(0xffffffffu, !(fmaxf(mx, -row_min64(s)) > near.top));
                        const float u = mx * mx;
                        mx *= fmaf(fmaf(fmaf(u, near.f3, near.f2), u, near.f1), u, near.f0);
                    }
                }
                if constexpr (CAP) {
                    if (!folded) cap_row(s, p.c0, p.c1);
                }
                if constexpr (BIAS) bias_row(s, CAP ? 1.0f : p.c0, slope, pos - j0);
                if (!all) {
                    const int shared = pre - j0, own = (p.causal ? min(sr.lk, pos + 1) : sr.lk) - j0;
                    if (!DOCS || lo == hi) {  // without documents lo, hi and docq are 0
                        const int end = docq == lo ? max(own, shared) : shared;
#pragma unroll
                        for (int e = 0; e < kN; ++e) s[e] = e < end ? s[e] : -INFINITY;
                    } else {
                        int *d = sdoc + (warp - 2) * kN;
                        __syncwarp();
                        d[lane] = n0;
                        d[lane + 32] = n1;
                        __syncwarp();
                        // (bitwise: short-circuit forms became 64 divergent branches, 4.4 us a block)
#pragma unroll
                        for (int e = 0; e < kN; e += 4) {
                            const int4 n = *reinterpret_cast<const int4 *>(d + e);
                            s[e] = ((e < shared) | ((e < own) & (n.x == docq))) ? s[e] : -INFINITY;
                            s[e + 1] = ((e + 1 < shared) | ((e + 1 < own) & (n.y == docq))) ? s[e + 1] : -INFINITY;
                            s[e + 2] = ((e + 2 < shared) | ((e + 2 < own) & (n.z == docq))) ? s[e + 2] : -INFINITY;
                            s[e + 3] = ((e + 3 < shared) | ((e + 3 < own) & (n.w == docq))) ? s[e + 3] : -INFINITY;
                        }
                    }
                }
                const float unit = (CAP || BIAS) ? 1.0f : p.c0;
                if (!folded) mx = row_max64(s) * unit;
                if constexpr (kLift<T> > 0.0f) mx -= kLift<T> - kRescaleLog2;
                const bool need = i > 0 && mx > m_run + kRescaleLog2;
                if (i == 0) m_run = mx;
                if (__any_sync(0xffffffffu, need)) {
                    if (!(ok = wait(&pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1))) break;
                    tc_fence_after();
                    const float alpha = need ? ex2f(m_run - mx) : 1.0f;
                    if (need) m_run = mx;
#pragma unroll
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        tmem_ld32(tmem + lane_base + kOCol + c, o);
                        tmem_ld_wait_regs(o);
                        uint32_t r[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(o[e] * alpha);
                        tmem_st32(tmem + lane_base + kOCol + c, r);
                    }
                    if constexpr (C::ONES) {
                        float l = tmem_ld1(tmem + lane_base + C::L_COL);
                        tmem_ld_wait_reg(l);
                        tmem_st1(tmem + lane_base + C::L_COL, l * alpha);
                    }
                    tmem_st_wait();
                    l0 *= alpha;
                    l1 *= alpha;
                }
                // a row that has seen no key yet has nothing to subtract: its weights are 2^-inf
                const float nm = m_run == -INFINITY ? 0.0f : -m_run;
                auto weights = [&](int e, F2 x) {
                    float x0, x1;
                    x.get(x0, x1);
                    x0 = ex2f(x0);
                    x1 = ex2f(x1);
                    pk[e] = pack2<T>(x0, x1);
                    if constexpr (!C::ONES) add_pair<T>(l0, l1, pk[e]);
                };
                if (CAP && !BIAS && folded) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const F2 x(s[2 * e], s[2 * e + 1]), u = mul2(x, x);
                        const F2 q = fma2(fma2(fma2(u, F2(near.f3, near.f3), F2(near.f2, near.f2)), u, F2(near.f1, near.f1)), u,
                                          F2(near.f0, near.f0));
                        weights(e, fma2(x, q, F2(nm, nm)));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) weights(e, fma2(F2(s[2 * e], s[2 * e + 1]), F2(unit, unit), F2(nm, nm)));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) pk[e] = 0;
            }
            if (tag & 2) {
                // non-finite values leave the V tile before the product; every
                // lane waits, as each reads what TMA wrote
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(&v_full[st], (i / ST) & 1, p.fault)))) break;
                uint4 *v = reinterpret_cast<uint4 *>(sV + st * C::KV_BYTES);
                bool found = false;
                for (int e = (warp - 2) * 32 + lane; e < C::KV_BYTES / 16; e += 128) {
                    uint4 u = v[e];
                    if (!any_nonfinite<T>(u)) continue;
                    clean_pair<T>(u.x);
                    clean_pair<T>(u.y);
                    clean_pair<T>(u.z);
                    clean_pair<T>(u.w);
                    v[e] = u;
                    found = true;
                }
                if (found) {
                    fence_proxy_async_smem();
                    atomicMin(&bad[0], tag >> 2);
                    atomicMax(&bad[1], tag >> 2);
                }
                __syncwarp();
            }
            tmem_st32(tmem + lane_base + b * kN, pk);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[b]);
            if (tag & 1) break;
        }
        if (ok) ok = wait(&pv_done[i & 1], (i >> 1) & 1);
        tc_fence_after();
        asm volatile("bar.sync 1, 128;" ::: "memory");  // every softmax warp has noted its blocks
        float l = l0 + l1;
        if constexpr (C::ONES) {
            l = tmem_ld1(tmem + lane_base + C::L_COL);
            tmem_ld_wait_reg(l);
        }
        const float inv = p.splits > 1 ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
        const int64_t part = split_part(p, seq, row0 + row, head) + split;
        if (p.splits > 1 && ok && valid) p.part_ml[part] = make_float2(m_run, l);
        const int bad0 = bad[0], bad1 = bad[1];
        T *dst = static_cast<T *>(p.out) + (sr.q0 + static_cast<int64_t>(row0) + row) * p.ldo + static_cast<int64_t>(head) * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
            float o[32];
            __syncwarp();
            tmem_ld32(tmem + lane_base + kOCol + c, o);
            tmem_ld_wait_regs(o);
            if (!ok || !valid) continue;
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= inv;
            for (int j = bad0 * kN; bad1 >= 0 && j < min((bad1 + 1) * kN, sr.lk); ++j) {
                if (!visible(j)) continue;
                const T *v = static_cast<const T *>(p.v) + (sr.k0 + static_cast<int64_t>(j)) * p.ldv + static_cast<int64_t>(hk) * D + c;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float x = to_f32(v[e]);
                    if (!isfinite(x)) o[e] += x;
                }
            }
            if (p.splits > 1) {
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    *reinterpret_cast<float4 *>(p.part_o + part * D + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
                uint4 u;
                u.x = pack2<T>(o[e], o[e + 1]);
                u.y = pack2<T>(o[e + 2], o[e + 3]);
                u.z = pack2<T>(o[e + 4], o[e + 5]);
                u.w = pack2<T>(o[e + 6], o[e + 7]);
                *reinterpret_cast<uint4 *>(dst + c + e) = u;
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// A warp joins the splits of one query and head.
template <typename T, int D>
__global__ void __launch_bounds__(256) masked_splits_kernel(const MaskedParams p) {
    constexpr int E = D / 32;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int head = static_cast<int>(item % p.heads);
    const int64_t qi = item / p.heads;
    const SeqRange sr = seq_range(p, blockIdx.y);
    if (qi >= sr.lq || qi >= p.max_q) return;
    const int64_t at = split_part(p, blockIdx.y, qi, head);
    const float mine = lane < p.splits ? p.part_ml[at + lane].x : -INFINITY;
    float mm = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    float ll = 0.0f, oo[E] = {};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float2 ml = p.part_ml[at + s];
        if (ml.x == -INFINITY) continue;  // saw nothing and wrote no sums
        const float a = ex2f(ml.x - mm);
        ll = fmaf(ml.y, a, ll);
        const float *src = p.part_o + (at + s) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) oo[e] = fmaf(src[e], a, oo[e]);
    }
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    T *dst = static_cast<T *>(p.out) + (sr.q0 + qi) * p.ldo + static_cast<int64_t>(head) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t *>(dst + e) = pack2<T>(oo[e] * inv, oo[e + 1] * inv);
}

template <typename T, int D, bool CAP, bool BIAS, bool DOCS>
int launch_fmha(p3d_ctx *ctx, const MaskedParams &p, int dtype) {
    CUtensorMap tq, tk, tv;
    int rc = make_tmap_16bit_2d(ctx, &tq, p.q, dtype, p.rows_q, static_cast<uint64_t>(p.heads) * D, p.ldq, kM);
    if (rc || (rc = make_tmap_16bit_2d(ctx, &tk, p.k, dtype, p.rows_k, static_cast<uint64_t>(p.kv_heads) * D, p.ldk, kN)) ||
        (rc = make_tmap_16bit_2d(ctx, &tv, p.v, dtype, p.rows_k, static_cast<uint64_t>(p.kv_heads) * D, p.ldv, kN)))
        return rc;
    const int64_t tiles = ceil_div(p.max_q, kM);
    if (tiles * p.splits > 65535) return set_error(ctx, P3D_ERR_UNSUPPORTED, "p3d_masked_attention: max_q above 8388480");
    auto kernel = masked_fmha_kernel<T, D, CAP, BIAS, DOCS>;
    P3D_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    P3D_CUDA(ctx, launch_pdl(kernel, dim3(p.heads, p.nseq, static_cast<unsigned>(tiles * p.splits)), dim3(kThreadsF), kSmem, ctx->stream,
                             tq, tk, tv, p));
    rc = check_launch(ctx, "masked_fmha");
    if (rc || p.splits == 1) return rc;
    P3D_CUDA(ctx, launch_pdl(masked_splits_kernel<T, D>, dim3(static_cast<unsigned>(ceil_div(p.max_q * p.heads, 8)), p.nseq), dim3(256),
                             0, ctx->stream, p));
    return check_launch(ctx, "masked_splits");
}

template <typename T, int D, bool DOCS>
int launch_rules(p3d_ctx *ctx, const MaskedParams &p, int dtype) {
    if (p.c1 > 0.0f)
        return p.slopes ? launch_fmha<T, D, true, true, DOCS>(ctx, p, dtype) : launch_fmha<T, D, true, false, DOCS>(ctx, p, dtype);
    return p.slopes ? launch_fmha<T, D, false, true, DOCS>(ctx, p, dtype) : launch_fmha<T, D, false, false, DOCS>(ctx, p, dtype);
}

// The kernel of a type, head_dim and rules (one translation unit a type and head_dim).
template <typename T, int D>
int masked_tiles(p3d_ctx *ctx, const MaskedParams &p, int dtype) {
    return p.doc_k ? launch_rules<T, D, true>(ctx, p, dtype) : launch_rules<T, D, false>(ctx, p, dtype);
}

}  // namespace
}  // namespace p3d
