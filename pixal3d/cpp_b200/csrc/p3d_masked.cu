// C ABI entry of the masked attention (kernels in p3d_masked_rows.cu,
// p3d_masked_pieces.cu and p3d_masked_fmha.cuh).
#include <algorithm>
#include <cmath>

#include "p3d_masked.cuh"

namespace p3d {
int masked_attention_rows(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype);
int masked_attention_pieces(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype);
int masked_tiles_bf16_64(p3d_ctx *ctx, const MaskedParams &p, int dtype);
int masked_tiles_bf16_128(p3d_ctx *ctx, const MaskedParams &p, int dtype);
int masked_tiles_f16_64(p3d_ctx *ctx, const MaskedParams &p, int dtype);
int masked_tiles_f16_128(p3d_ctx *ctx, const MaskedParams &p, int dtype);

namespace {

// Up to this many queries a sequence go to the kernels for few rows; up to
// this many keys, to the one that takes each query alone.
constexpr int64_t kFewRows = 8, kFewKeys = 512;

// Query tiles that are ordered at most: more of them leave a last wave too
// short to matter.
constexpr int kOrderTiles = 1024;

// The SMs that work is cut for, B200's.  The plans below give the workspace's size
// too, which is asked for without a context, so the size and the call must agree:
// a context whose device has other SMs runs the same plan.
constexpr int64_t kPlanSms = 148;
constexpr int64_t kPlaces = 2 * kPlanSms;  // CTAs of masked_fmha_kernel at once

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

// Smallest and largest document number of every key block, a warp a block.
__global__ void __launch_bounds__(256) doc_range_kernel(const MaskedParams p) {
    pdl_wait();
    pdl_trigger();
    if (p.tile_count && threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) *p.tile_count = 0;
    const SeqRange sr = seq_range(p, blockIdx.y);
    const int lane = threadIdx.x & 31, step = gridDim.x * 8;
    for (int b = blockIdx.x * 8 + (threadIdx.x >> 5); b * 64 < sr.lk; b += step) {
        const int j = b * 64 + lane;
        const int a = p.doc_k[sr.k0 + min(j, sr.lk - 1)], c = p.doc_k[sr.k0 + min(j + 32, sr.lk - 1)];
        const int lo = __reduce_min_sync(0xffffffffu, min(a, c)), hi = __reduce_max_sync(0xffffffffu, max(a, c));
        if (lane == 0) p.doc_range[doc_block(sr, blockIdx.y) + b] = make_int2(lo, hi);
    }
}

// The order of the query tiles: those with the most key blocks first.  A tile
// that holds the end of one document and the start of the next reads both, so
// where it came late its CTA ran on alone (16384 queries in 5 documents, 16
// heads: 660 us as they lie, 628 with this kernel's own time).  A warp
// counts a tile's blocks as the attention kernel will visit them; the last
// block ranks the counts.  Every tile comes once whatever the counts are, and
// none depends on another: the order changes no result.
__global__ void __launch_bounds__(256) doc_order_kernel(const MaskedParams p, int tiles) {
    __shared__ int counts[kOrderTiles];
    __shared__ int last;
    pdl_wait();
    pdl_trigger();
    const int n = tiles * p.nseq, lane = threadIdx.x & 31, item = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item < n) {
        const int seq = item / tiles, row0 = item % tiles * 128;
        const SeqRange sr = seq_range(p, seq);
        const int nrows = min(min(sr.lq, static_cast<int>(p.max_q)) - row0, 128);
        int count = -1, lo = 0x7fffffff, hi = -0x7fffffff - 1;
        if (nrows > 0) {
#pragma unroll
            for (int r = 0; r < 128; r += 32) {
                const int d = p.doc_q[sr.q0 + row0 + min(r + lane, nrows - 1)];
                lo = min(lo, d);
                hi = max(hi, d);
            }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
            const int pre = p.prefix ? min(max(p.prefix[seq], 0), sr.lk) : 0;
            const int limit = p.causal ? min(sr.lk, max(pre, row0 + nrows + sr.lk - sr.lq)) : sr.lk;
            const int2 *range = p.doc_range + doc_block(sr, seq);
            count = 0;
#pragma unroll 4
            for (int b = lane; b * 64 < limit; b += 32) {
                const int2 r = range[b];
                count += b * 64 < pre || (r.x <= hi && lo <= r.y);
            }
            count = __reduce_add_sync(0xffffffffu, count);
        }
        if (lane == 0) __stcg(p.tile_found + item, make_int4(count, lo, hi, item));
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(p.tile_count, 1) == static_cast<int>(gridDim.x) - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (int i = threadIdx.x; i < n; i += 256) counts[i] = __ldcg(&p.tile_found[i].x);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
        const int mine = counts[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += counts[j] > mine || (counts[j] == mine && j < i);
        p.tile_order[rank] = __ldcg(p.tile_found + i);
    }
}

// Many queries: the documents' block ranges and the tiles' order, then the
// tensor-core kernel.
int masked_attention_tiles(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype) {
    if (p.doc_k) {
        const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(ceil_div(std::max<int64_t>(p.max_k, 1), 8 * 64), 1024));
        P3D_CUDA(ctx, launch_pdl(doc_range_kernel, dim3(blocks, p.nseq), dim3(256), 0, ctx->stream, p));
        int rc = check_launch(ctx, "doc_range");
        if (rc) return rc;
        if (p.tile_order) {
            const int tiles = static_cast<int>(ceil_div(p.max_q, 128));
            P3D_CUDA(ctx, launch_pdl(doc_order_kernel, dim3(static_cast<unsigned>(ceil_div(tiles * p.nseq, 8))), dim3(256), 0, ctx->stream,
                                     p, tiles));
            if ((rc = check_launch(ctx, "doc_order"))) return rc;
        }
    }
    if (dtype == P3D_BF16) return head_dim == 64 ? masked_tiles_bf16_64(ctx, p, dtype) : masked_tiles_bf16_128(ctx, p, dtype);
    return head_dim == 64 ? masked_tiles_f16_64(ctx, p, dtype) : masked_tiles_f16_128(ctx, p, dtype);
}

// Few queries over long keys: rows of an item (8, 16 or 24 of the K/V head's
// queries and heads), 16-key tiles of a piece, blocks, pieces at most,
// and the bytes of their results.
struct PiecePlan {
    int item_rows, piece, most_pieces, blocks;
    int64_t parts;
    size_t o, ml;
    PiecePlan(int nseq, int64_t max_q, int64_t max_k, int64_t rows_k, int heads, int kv_heads, int head_dim) {
        const int64_t rows = std::max<int64_t>(max_q * (heads / kv_heads), 1);
        const int64_t tiles = std::max<int64_t>(1, ceil_div(std::min(rows_k, nseq * max_k) / nseq, 16));  // of a mean item
        // Passes of 8 rows for up to 8, else of 16, but of 24 for 17 to 24 rows of 64
        // dims (192 bytes of spills) over many keys, which then come once, not twice.
        // us by passes of at most 16 / 24 (queries x heads of each K/V head x K/V
        // heads, sequences x keys): 1 x 24 x 1, 16 x 9000 26.8 / 24.0; 5 x 4 x 4, 4 x
        // 16000 36.0 / 31.2; 3 x 8 x 4, 2 x 16000 21.8 / 23.8; 6 x 4 x 4, 1 x 4000 11.0 /
        // 13.5; 40 and 48 rows 20.0 / 23.4 and 29.2 / 39.8.  Of 8 / 16: 32 rows 26.9 / 21.9
        // and 79.4 / 66.6, 128 dims 121.6 / 105.5 and 38.2 / 31.8 (20 rows 51.9 / 56.0).
        // Passes of 32 rows (516 bytes) 28.9 and 73.6 instead of 21.9 and 66.6.
        const bool once = head_dim == 64 && rows > 16 && rows <= 24 && nseq * kv_heads * tiles >= 8500;
        item_rows = once ? 24 : rows > 8 ? 16 : 8;
        const int64_t items = kv_heads * ceil_div(rows, item_rows);  // of a sequence
        // The fewest rounds of the blocks, one an SM, times a piece's length and its own
        // cost, over pieces of whole stages and no longer than a block's even
        // share, so that uneven sequences end together (4 sequences of up to
        // 16000 keys, 5 queries 89 against 122 us without that bound; the own
        // cost taken as 8 tiles, not 32: 5 sequences of up to 16381 keys, 32
        // heads over 8 55.3 against 52.4 us).
        const int64_t share = std::max<int64_t>(nseq * items * tiles / kPlanSms, 16);
        int64_t best = 0;
        piece = 16;
        for (int64_t l = 16; l < std::min(tiles, share) + 16; l += std::max<int64_t>(16, l / 8 / 16 * 16)) {
            const int64_t cost = ceil_div(nseq * items * ceil_div(tiles, l), kPlanSms) * (l + 32);
            if (best == 0 || cost < best) {
                best = cost;
                piece = static_cast<int>(l);
            }
        }
        most_pieces = static_cast<int>(ceil_div(std::max<int64_t>(max_k, 1), 16 * static_cast<int64_t>(piece)));
        blocks = static_cast<int>(std::min<int64_t>(kPlanSms, nseq * items * most_pieces));
        // of all sequences: by their number, or by the rows that they share
        parts = items * std::min(static_cast<int64_t>(nseq) * most_pieces, (rows_k / 16 + nseq) / piece + nseq);
        o = align256(static_cast<size_t>(parts) * item_rows * head_dim * sizeof(float));
        ml = align256(static_cast<size_t>(parts) * item_rows * sizeof(float2));
    }
};

// Many queries: splits of the key blocks (where the CTAs would fill less than
// half of the GPU's places, pieces of at least 8 blocks), whether the tiles
// are ordered (documents, more CTAs than places), and the bytes of the
// documents' ranges, of the order and of the splits' results.
struct TilePlan {
    int splits;
    int64_t tiles;
    bool ordered;
    size_t docs, order, o, ml;
    TilePlan(int nseq, int64_t max_q, int64_t max_k, int64_t rows_k, int heads, int head_dim, bool documents) {
        const int64_t ctas = static_cast<int64_t>(heads) * nseq * ceil_div(max_q, 128);
        splits = ctas > kPlanSms ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({kPlaces / std::max<int64_t>(ctas, 1), max_k / 512, 16})));
        tiles = nseq * ceil_div(max_q, 128);
        ordered = documents && ctas > kPlaces && tiles <= kOrderTiles;
        order = ordered ? align256(static_cast<size_t>(2 * tiles + 1) * sizeof(int4)) : 0;
        docs = documents ? align256(static_cast<size_t>(rows_k / 64 + nseq + 1) * sizeof(int2)) : 0;
        // at most kPlaces x 128 rows, whatever rows q has beside the sequences'
        const size_t parts = splits > 1 ? static_cast<size_t>(nseq) * max_q * heads * splits : 0;
        o = align256(parts * head_dim * sizeof(float));
        ml = align256(parts * sizeof(float2));
    }
};

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" size_t p3d_masked_attention_workspace(int nseq, int64_t max_q, int64_t max_k, int64_t rows_q, int64_t rows_k,
                                                 int heads, int kv_heads, int head_dim, int documents) {
    if (nseq <= 0 || max_q <= 0 || max_k < 0 || rows_q <= 0 || rows_k < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
    if (max_q > kFewRows) {
        const TilePlan plan(nseq, max_q, max_k, rows_k, heads, head_dim, documents != 0);
        return plan.docs + plan.order + plan.o + plan.ml;
    }
    if (max_k <= kFewKeys) return 0;
    const PiecePlan plan(nseq, max_q, max_k, rows_k, heads, kv_heads, head_dim);
    return plan.o + plan.ml;
}

extern "C" int p3d_masked_attention(p3d_ctx *ctx, const void *q, int64_t ldq, const void *k, int64_t ldk, const void *v,
                                    int64_t ldv, void *out, int64_t ldo, const int32_t *cu_q, const int32_t *cu_k, int nseq,
                                    int64_t max_q, int64_t max_k, int64_t rows_q, int64_t rows_k, int heads, int kv_heads,
                                    int head_dim, float scale, const p3d_attention_rules *rules, void *ws, size_t ws_bytes,
                                    int dtype) {
    if (!ctx) return P3D_ERR_INVALID;
    P3D_REQUIRE(ctx, rows_q >= 0 && rows_k >= 0 && rows_q < (int64_t(1) << 31) && rows_k < (int64_t(1) << 31) && max_q >= 0 &&
                         max_k >= 0 && max_q <= rows_q && max_k <= rows_k,
                "p3d_masked_attention: bad row counts (max_q <= rows_q, max_k <= rows_k)");
    P3D_REQUIRE(ctx, nseq > 0 && nseq < 65536, "p3d_masked_attention: bad nseq");
    if (max_q == 0) return P3D_OK;
    P3D_REQUIRE(ctx, q && out && cu_q && cu_k && ((k && v) || rows_k == 0), "p3d_masked_attention: null pointer");
    if (head_dim != 64 && head_dim != 128)
        return set_error(ctx, P3D_ERR_UNSUPPORTED, "p3d_masked_attention: head_dim must be 64 or 128");
    P3D_REQUIRE(ctx, is_16bit(dtype), "p3d_masked_attention: dtype must be bf16 or f16");
    P3D_REQUIRE(ctx, heads > 0 && heads < 65536 && kv_heads > 0 && heads % kv_heads == 0,
                "p3d_masked_attention: heads must be a multiple of kv_heads");
    P3D_REQUIRE(ctx, scale > 0.0f && std::isfinite(scale), "p3d_masked_attention: scale must be finite and positive");
    P3D_REQUIRE(ctx, ldq % 8 == 0 && ldk % 8 == 0 && ldv % 8 == 0 && ldo % 8 == 0,
                "p3d_masked_attention: leading dimensions must keep 16-byte rows");
    P3D_REQUIRE(ctx, (ldq >= static_cast<int64_t>(heads) * head_dim && ldo >= static_cast<int64_t>(heads) * head_dim) || rows_q == 1,
                "p3d_masked_attention: ldq / ldo below heads * head_dim");
    P3D_REQUIRE(ctx, (ldk >= static_cast<int64_t>(kv_heads) * head_dim && ldv >= static_cast<int64_t>(kv_heads) * head_dim) || rows_k <= 1,
                "p3d_masked_attention: ldk / ldv below kv_heads * head_dim");
    P3D_REQUIRE(ctx,
                ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                  reinterpret_cast<uintptr_t>(out)) & 15) == 0,
                "p3d_masked_attention: q/k/v/out must be 16-byte aligned");
    p3d_attention_rules r{};
    if (rules) r = *rules;
    P3D_REQUIRE(ctx, r.softcap == 0.0f || (r.softcap >= 1e-6f && r.softcap <= 1e6f),
                "p3d_masked_attention: softcap must be 0 (none) or between 1e-6 and 1e6");
    P3D_REQUIRE(ctx, (r.doc_q == nullptr) == (r.doc_k == nullptr) || rows_k == 0,
                "p3d_masked_attention: doc_q and doc_k go together");
    const size_t need = p3d_masked_attention_workspace(nseq, max_q, max_k, rows_q, rows_k, heads, kv_heads, head_dim,
                                                       r.doc_k != nullptr);
    P3D_REQUIRE(ctx, need == 0 || (ws && ws_bytes >= need && reinterpret_cast<uintptr_t>(ws) % 256 == 0),
                "p3d_masked_attention: workspace too small or not 256-byte aligned");
    MaskedParams p{};
    p.q = q;
    p.k = k;
    p.v = v;
    p.out = out;
    p.ldq = ldq;
    p.ldk = ldk;
    p.ldv = ldv;
    p.ldo = ldo;
    p.cu_q = cu_q;
    p.cu_k = cu_k;
    p.nseq = nseq;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.group = heads / kv_heads;
    p.rows_q = rows_q;
    p.rows_k = rows_k;
    p.max_q = max_q;
    p.max_k = max_k;
    constexpr float kLog2e = 1.4426950408889634f;
    p.c0 = r.softcap > 0.0f ? scale / r.softcap * 2.0f * kLog2e : scale * kLog2e;
    p.c1 = r.softcap > 0.0f ? r.softcap * kLog2e : 0.0f;
    p.causal = r.causal != 0;
    p.prefix = r.prefix;
    p.doc_q = r.doc_q;
    p.doc_k = r.doc_k;
    p.slopes = r.slopes;
    p.fault = ctx->fault;
    DeviceGuard on(ctx->device);
    if (max_q > kFewRows && rows_k > 0) {
        const TilePlan plan(nseq, max_q, max_k, rows_k, heads, head_dim, r.doc_k != nullptr);
        char *at = static_cast<char *>(ws);
        p.splits = plan.splits;
        p.doc_range = reinterpret_cast<int2 *>(at);
        at += plan.docs;
        if (plan.ordered) {
            p.tile_found = reinterpret_cast<int4 *>(at);
            p.tile_order = p.tile_found + plan.tiles;
            p.tile_count = reinterpret_cast<int *>(p.tile_order + plan.tiles);
        }
        at += plan.order;
        p.part_o = reinterpret_cast<float *>(at);
        p.part_ml = reinterpret_cast<float2 *>(at + plan.o);
        return masked_attention_tiles(ctx, p, head_dim, dtype);
    }
    if (max_k <= kFewKeys) return masked_attention_rows(ctx, p, head_dim, dtype);
    const PiecePlan plan(nseq, max_q, max_k, rows_k, heads, kv_heads, head_dim);
    p.item_rows = plan.item_rows;
    p.piece = plan.piece;
    p.most_pieces = plan.most_pieces;
    p.blocks = plan.blocks;
    p.parts = plan.parts;
    p.part_o = static_cast<float *>(ws);
    p.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(ws) + plan.o);
    return masked_attention_pieces(ctx, p, head_dim, dtype);
}
