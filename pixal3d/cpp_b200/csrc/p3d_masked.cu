// C ABI entry of the masked attention (kernels in p3d_masked_rows.cu and
// p3d_masked_fmha.cuh).
#include <algorithm>
#include <cmath>

#include "p3d_masked.cuh"

namespace p3d {
int masked_attention_rows(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype);
// Ranges that the key tiles of `items` items are cut into, 0 for a block an item.
int masked_rows_ranges(int64_t items, int64_t max_k, int group, int head_dim);
int masked_tiles_bf16_64(p3d_ctx *ctx, const MaskedParams &p, int dtype);
int masked_tiles_bf16_128(p3d_ctx *ctx, const MaskedParams &p, int dtype);
int masked_tiles_f16_64(p3d_ctx *ctx, const MaskedParams &p, int dtype);
int masked_tiles_f16_128(p3d_ctx *ctx, const MaskedParams &p, int dtype);

namespace {

// Up to this many queries a sequence go to the kernel that takes them one by one.
constexpr int64_t kFewRows = 8;

// Smallest and largest document number of every key block, a warp a block.
__global__ void __launch_bounds__(256) doc_range_kernel(const MaskedParams p) {
    pdl_wait();
    pdl_trigger();
    const SeqRange sr = seq_range(p, blockIdx.y);
    const int lane = threadIdx.x & 31, step = gridDim.x * 8;
    for (int b = blockIdx.x * 8 + (threadIdx.x >> 5); b * 64 < sr.lk; b += step) {
        const int j = b * 64 + lane;
        const int a = p.doc_k[sr.k0 + min(j, sr.lk - 1)], c = p.doc_k[sr.k0 + min(j + 32, sr.lk - 1)];
        const int lo = __reduce_min_sync(0xffffffffu, min(a, c)), hi = __reduce_max_sync(0xffffffffu, max(a, c));
        if (lane == 0) p.doc_range[doc_block(sr, blockIdx.y) + b] = make_int2(lo, hi);
    }
}

// Many queries: the documents' block ranges, then the tensor-core kernel.
int masked_attention_tiles(p3d_ctx *ctx, const MaskedParams &p, int head_dim, int dtype) {
    if (p.doc_k) {
        const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(ceil_div(std::max<int64_t>(p.max_k, 1), 8 * 64), 1024));
        P3D_CUDA(ctx, launch_pdl(doc_range_kernel, dim3(blocks, p.nseq), dim3(256), 0, ctx->stream, p));
        const int rc = check_launch(ctx, "doc_range");
        if (rc) return rc;
    }
    if (dtype == P3D_BF16) return head_dim == 64 ? masked_tiles_bf16_64(ctx, p, dtype) : masked_tiles_bf16_128(ctx, p, dtype);
    return head_dim == 64 ? masked_tiles_f16_64(ctx, p, dtype) : masked_tiles_f16_128(ctx, p, dtype);
}

size_t align256(size_t b) { return (b + 255) / 256 * 256; }

// Ranges of the rows kernel and the bytes of its parts' sums and (maximum, sum).
int rows_parts(int nseq, int64_t max_q, int64_t max_k, int heads, int kv_heads, int head_dim, size_t &o, size_t &ml) {
    const int group = heads / kv_heads, per = group > 8 ? 16 : 8;
    const int64_t items = static_cast<int64_t>(nseq) * max_q * kv_heads * ceil_div(group, per);
    const int ranges = masked_rows_ranges(items, max_k, group, head_dim);
    const size_t parts = static_cast<size_t>(ranges + items) * per;
    o = align256(parts * head_dim * sizeof(float));
    ml = align256(parts * sizeof(float2));
    return ranges;
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" size_t p3d_masked_attention_workspace(int nseq, int64_t max_q, int64_t max_k, int64_t rows_q, int64_t rows_k,
                                                 int heads, int kv_heads, int head_dim, int documents) {
    if (nseq <= 0 || max_q <= 0 || max_k < 0 || rows_q <= 0 || rows_k < 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0) return 0;
    if (max_q > kFewRows) return documents ? align256(static_cast<size_t>(rows_k / 64 + nseq + 1) * sizeof(int2)) : 0;
    size_t o, ml;
    return rows_parts(nseq, max_q, max_k, heads, kv_heads, head_dim, o, ml) ? o + ml : 0;
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
    P3D_REQUIRE(ctx, r.softcap >= 0.0f && std::isfinite(r.softcap), "p3d_masked_attention: softcap must be finite, 0 for none");
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
        p.doc_range = static_cast<int2 *>(ws);
        return masked_attention_tiles(ctx, p, head_dim, dtype);
    }
    size_t o, ml;
    p.head_tiles = static_cast<int>(ceil_div(p.group, p.group > 8 ? 16 : 8));
    p.ranges = rows_parts(nseq, max_q, max_k, heads, kv_heads, head_dim, o, ml);
    p.part_o = static_cast<float *>(ws);
    p.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(ws) + o);
    return masked_attention_rows(ctx, p, head_dim, dtype);
}
