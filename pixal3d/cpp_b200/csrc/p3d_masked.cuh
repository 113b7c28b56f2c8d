// What the masked-attention kernels share: the rules of visibility and of the
// scores, and the sequence geometry.
#pragma once

#include "p3d_common.cuh"

namespace p3d {

struct MaskedParams {
    const void *q, *k, *v;
    void *out;
    int64_t ldq, ldk, ldv, ldo;
    const int32_t *cu_q, *cu_k;
    int nseq, heads, kv_heads, group;
    int64_t rows_q, rows_k, max_q, max_k;
    // scores in units of log2: x = s c0, or with a cap (c1 > 0) c1 tanh(s c0 / (2 log2 e))
    float c0, c1;
    int causal;
    const int32_t *prefix, *doc_q, *doc_k;
    const float *slopes;
    int head_tiles;  // few keys: groups of 8 or 16 heads of a K/V head
    // few queries, long keys: rows (query, head) of an item, key tiles of a
    // piece, pieces of an item at most, blocks, and the pieces' results:
    // [parts][item_rows][D] sums against their own maxima, and (maximum, sum)
    int item_rows, piece, most_pieces, blocks;
    int64_t parts;
    int splits;  // many queries: of the key blocks; results [(sequence, query), head][split]
    float *part_o;
    float2 *part_ml;
    int2 *doc_range; // (smallest, largest) document number of every 64-key block
    // many queries of documents: (key blocks, smallest and largest document
    // number, sequence * tiles + tile) of the query tiles as they lie, and by
    // their blocks, largest first (null: not ordered); a counter
    int4 *tile_found, *tile_order;
    int *tile_count;
    int *fault;
};

// Rows of sequence s.  Offsets that point outside the buffers are clamped, so
// that a wrong offset can give a wrong result but no access out of bounds.
struct SeqRange {
    int q0, lq, k0, lk;
};
__device__ __forceinline__ SeqRange seq_range(const MaskedParams &p, int s) {
    SeqRange r;
    const int nq = static_cast<int>(p.rows_q), nk = static_cast<int>(p.rows_k);
    r.q0 = min(max(p.cu_q[s], 0), nq);
    r.lq = max(min(p.cu_q[s + 1], nq) - r.q0, 0);
    r.k0 = min(max(p.cu_k[s], 0), nk);
    r.lk = max(min(p.cu_k[s + 1], nk) - r.k0, 0);
    return r;
}

// Where the sequence's key blocks begin in doc_range: sequences that follow
// one another never share an entry, and the last lies below
// rows_k / 64 + nseq + 1.
__device__ __forceinline__ int doc_block(const SeqRange &sr, int seq) { return sr.k0 / 64 + seq; }

__device__ __forceinline__ float ex2f(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcpf(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Weights are rounded to the operand type, since they are the second product's
// operand: half a step (2^-8 of a bf16 weight, 2^-11 of an f16 one) of each
// weight by itself.  f16 has few exponents, so there the running maximum is
// held this many powers of two below the scores' own: weights down to 2^-29 of the
// largest keep all their bits (2^-14 without) and those down to 2^-40 count
// (2^-25).  Where the maximum may lag 8 behind, it is held 7 below instead of 15:
// 2^-21 and 2^-32.  No weight passes 2^15.
template <typename T>
constexpr float kLift = 0.0f;
template <>
inline constexpr float kLift<__half> = 15.0f;

// The capped score in units of log2, c1 tanh(t) with t = s c0 / (2 log2 e).
// Scores within half the cap: t q(t^2), q of degree 3 fitted to an absolute
// error of 1.3e-7 (least maximum over [0, 1/2]), 2.4e-6 of the score itself.
constexpr float kCapT = 0.34657359027997264f;  // ln(2) / 2: t = s c0 kCapT
constexpr float kCap0 = 0.999997676f, kCap1 = -0.333206552f, kCap2 = 0.131451456f, kCap3 = -0.043372481f;
// Any t: tanh(t) = 1 - 2 / (1 + e^2t), some 2^-22 of the cap off.  (The hardware
// tanh's 2^-11 of the score is not enough: a score of 20 would be 0.01 off, 1 %
// of its weight.)
__device__ __forceinline__ float capped_far(float t, float c1) {
    return fmaf(-2.0f * c1, rcpf(1.0f + ex2f(t * 2.885390081777927f)), c1);
}
__device__ __forceinline__ float capped(float s, float c0, float c1) {
    const float t = s * c0 * kCapT, u = t * t;
    if (fabsf(t) <= 0.5f) return c1 * t * fmaf(fmaf(fmaf(u, kCap3, kCap2), u, kCap1), u, kCap0);
    return capped_far(t, c1);
}

}  // namespace p3d
