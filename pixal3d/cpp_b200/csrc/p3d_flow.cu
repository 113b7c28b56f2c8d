// Device-resident SLat flow model and flow-Euler/CFG sampler.
//
// Mirrors slat_flow_forward_f32 (src/slat_flow.cpp:161-249) and
// SLatFlowModel::sample (src/slat_flow.cpp:1401-1447) with
// flow_euler_sample_f32 (src/flow_sampler.cpp:245-343), but keeps every
// tensor in HBM for the whole sampling run:
//   - weights are converted once to bf16 GEMM operands (biases, norms and
//     the modulation MLP stay f32);
//   - the coordinate topology (batch offsets, neighbour maps, downsample
//     maps) is built once per coordinate set in p3d_flow_prepare;
//   - CFG runs as ONE batched forward: batch items [0, I) are the
//     conditional images, [I, 2I) the unconditional copies (zeros
//     condition), so velocity halves are contiguous and the Euler/CFG update
//     is a single fused kernel;
//   - the sampler keeps its t schedule and a step counter on the device, so
//     one step (forward + update) is captured once as a CUDA graph and
//     replayed for every remaining step.
// Residual stream h is f32; GEMM operands f16 (or bf16); accumulation f32.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <unordered_map>
#include <vector>

#include "p3d_common.cuh"

extern "C" int p3d_layernorm_modulate(p3d_ctx *, const float *, int64_t, int, float, const float *, const float *,
                                      const float *, int64_t, const int32_t *, int, void *, int);
extern "C" int p3d_qk_rmsnorm_rope(p3d_ctx *, void *, int64_t, int64_t, int, int, const float *, const int32_t *,
                                   float, float, int);
extern "C" int p3d_group_norm_silu(p3d_ctx *, const float *, int64_t, int, int, float, const float *, const float *,
                                   const int32_t *, int, int, double *, void *, int);
extern "C" int64_t p3d_downsample_grid_ints(int, int, int, int, int);

namespace p3d {
namespace {

unsigned blocks_for(int64_t n, int per) { return static_cast<unsigned>(ceil_div(n, per)); }

// ------------------------------------------------------ small kernels

// Sinusoidal timestep embedding cos||sin, dim 256, period 1e4
// (timestep_embedding, src/flow.cpp:92-123).  t_b = mult * ts[base + b*stride]
// where base = 4 * (*counter) when counter is given (sampler schedule).
__global__ void temb_freq_kernel(const float *ts, int stride, const int *counter, float mult, int batch, int dim,
                                 float *out) {
    const int b = blockIdx.x, i = threadIdx.x;
    const int half = dim / 2;
    if (i >= half) return;
    const int base = counter ? 4 * (*counter) : 0;
    const float t = mult * ts[base + b * stride];
    const float log_period = 9.210340371976184f;  // (float)log(10000.0)
    const float frac = static_cast<float>(i) / static_cast<float>(half);
    const float arg = t * expf(-log_period * frac);
    out[b * dim + i] = cosf(arg);
    out[b * dim + half + i] = sinf(arg);
}

// y[b, n] = act_out(bias[n] + sum_k W[n, k] * act_in(x[b, k])) for B <= 16
// rows; one warp per output feature.  act: 0 none, 1 silu (x/(1+e^-x)),
// 2 silu in the sign-split form of src/slat_flow.cpp:79-83.
__device__ __forceinline__ float act_f(float v, int act) {
    if (act == 1) return v * (1.0f / (1.0f + expf(-v)));
    if (act == 2) {
        if (v >= 0.0f) return v / (1.0f + expf(-v));
        const float e = expf(v);
        return v * e / (1.0f + e);
    }
    return v;
}

// y[r, n] = act_out(bias[n] + sum_k W[n, k] act_in(x[r, k])) for a few rows
// (timestep MLP, modulation): one warp per output n, W rows read coalesced
// with 4 loads in flight per lane; act_in(x) is applied once per block into
// shared memory (rows * K floats, dynamic).
template <int B>
__global__ void small_linear_kernel(const float *__restrict__ x, int K, const float *__restrict__ W,
                                    const float *__restrict__ bias, int N, float *__restrict__ y, int act_in,
                                    int act_out, int rows) {
    extern __shared__ float xs[];  // [rows][K]
    for (int i = threadIdx.x; i < rows * K; i += blockDim.x) xs[i] = act_f(x[i], act_in);
    __syncthreads();
    const int n = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (n >= N) return;
    const int lane = threadIdx.x & 31;
    float acc[B];
#pragma unroll
    for (int b = 0; b < B; ++b) acc[b] = 0.0f;
    const float *w = W + static_cast<int64_t>(n) * K;
    int k = lane;
    for (; k + 96 < K; k += 128) {
        const float w0 = __ldg(w + k), w1 = __ldg(w + k + 32), w2 = __ldg(w + k + 64), w3 = __ldg(w + k + 96);
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (b < rows) {
                const float *xb = xs + b * K + k;
                acc[b] += w0 * xb[0] + w1 * xb[32] + w2 * xb[64] + w3 * xb[96];
            }
    }
    for (; k < K; k += 32) {
        const float wv = __ldg(w + k);
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (b < rows) acc[b] += wv * xs[b * K + k];
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
        const float s = warp_sum(acc[b]);
        if (lane == 0 && b < rows) y[b * N + n] = act_f(s + (bias ? bias[n] : 0.0f), act_out);
    }
}

int small_linear(p3d_ctx *ctx, const float *x, int rows, int K, const float *W, const float *b, int N, float *y,
                 int act_in, int act_out) {
    // up to 4 rows per call, rows * K floats of shared memory (<= 48 KB)
    const int per_call = std::min(4, (48 * 1024 / 4) / std::max(K, 1));
    if (per_call < 1) return set_error(ctx, P3D_ERR_UNSUPPORTED, "small_linear: K too large");
    for (int r0 = 0; r0 < rows; r0 += per_call) {
        const int r = rows - r0 < per_call ? rows - r0 : per_call;
        const size_t smem = sizeof(float) * static_cast<size_t>(r) * K;
        small_linear_kernel<4><<<blocks_for(N, 8), 256, smem, ctx->stream>>>(
            x + static_cast<int64_t>(r0) * K, K, W, b, N, y + static_cast<int64_t>(r0) * N, act_in, act_out, r);
        int rc = check_launch(ctx, "small_linear");
        if (rc) return rc;
    }
    return P3D_OK;
}

// mods[b, j] = block_mod[j] + tmod[b, j]
__global__ void add_mod_kernel(const float *bm, const float *tmod, int batch, int six_c, float *mods) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= static_cast<int64_t>(batch) * six_c) return;
    mods[i] = bm[i % six_c] + tmod[i];
}

// f32 [n, in] -> 16-bit [n, in_pad] (zero padded).
template <typename T>
__global__ void pad16_kernel(const float *x, int64_t n, int in, int in_pad, T *out, const int32_t *rows) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n * in_pad) return;
    const int64_t r = i / in_pad;
    const int c = static_cast<int>(i - r * in_pad);
    const int64_t src = rows ? rows[r] : r;  // rows: gather x[rows[r]] into row r
    out[i] = from_f32<T>(c < in ? x[src * in + c] : 0.0f);
}

int pad16(p3d_ctx *ctx, const float *x, int64_t n, int in, int in_pad, void *out, int dtype,
          const int32_t *rows = nullptr) {
    if (n * in_pad == 0) return P3D_OK;
    const unsigned grid = blocks_for(n * in_pad, 256);
    if (dtype == P3D_BF16)
        pad16_kernel<__nv_bfloat16><<<grid, 256, 0, ctx->stream>>>(x, n, in, in_pad, static_cast<__nv_bfloat16 *>(out),
                                                                   rows);
    else
        pad16_kernel<__half><<<grid, 256, 0, ctx->stream>>>(x, n, in, in_pad, static_cast<__half *>(out), rows);
    return check_launch(ctx, "pad16");
}

// Prepare-time checks and offsets, written into one int32 summary so that
// prepare reads everything it needs back with a single copy:
//   [0] batch-order fault (1 when some row's batch is outside [0, batch) or
//       decreases), [1] the context's device fault flag,
//   [2, 2 + B]  fine-level batch offsets, [3 + B, 3 + 2B] trunk offsets,
//   [4 + 2B] trunk rows.
__global__ void check_batch_kernel(const int4 *__restrict__ coords, int64_t n, int batch, int32_t *summary) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int b = coords[i].x;
    if (b < 0 || b >= batch || (i > 0 && coords[i - 1].x > b)) summary[0] = 1;
}

// off[b] = first row of batch item b among the *m rows (sorted by batch);
// off[batch] = *m, also written to *m_out.
__global__ void offsets_dev_kernel(const int4 *__restrict__ coords, const int64_t *m, int batch, int32_t *off,
                                   int32_t *m_out) {
    const int b = blockIdx.x * blockDim.x + threadIdx.x;
    if (b > batch) return;
    const int64_t n = *m;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (coords[mid].x < b) lo = mid + 1; else hi = mid;
    }
    off[b] = static_cast<int32_t>(b == batch ? n : lo);
    if (b == batch && m_out) *m_out = static_cast<int32_t>(n);
}

__global__ void copy_fault_kernel(const int *fault, int32_t *dst) { *dst = *fault; }

// coords_out[i] = coords_in[perm[i]]
__global__ void gather_coords_kernel(const int4 *__restrict__ in, const int32_t *__restrict__ perm, int64_t n,
                                     int4 *__restrict__ out) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i < n) out[i] = in[perm[i]];
}

// out[rows[i]][c] = y[i][c]: fine rows back to the caller's order.
__global__ void scatter_rows_kernel(const float *__restrict__ y, const int32_t *__restrict__ rows, int64_t n, int C,
                                    float *__restrict__ out) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n * C) return;
    const int64_t r = i / C;
    out[static_cast<int64_t>(rows[r]) * C + (i - r * C)] = y[i];
}

// Sinusoidal absolute 3D PE added to h (no reference; benchmark config 1/2):
// per axis a, fd = C/6 frequencies f_i = 10000^(-i/fd): [sin(c_a f_i), cos(c_a f_i)].
__global__ void ape_add_kernel(float *h, const int4 *coords, int64_t n, int C) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n * C) return;
    const int64_t r = i / C;
    const int c = static_cast<int>(i - r * C);
    const int fd = C / 6;
    if (c >= 6 * fd) return;
    const int a = c / (2 * fd), j = c % (2 * fd);
    const int f = j % fd;
    const int4 cc = coords[r];
    const int coord = a == 0 ? cc.y : (a == 1 ? cc.z : cc.w);
    const float freq = 1.0f / powf(10000.0f, static_cast<float>(f) / static_cast<float>(fd));
    const float arg = static_cast<float>(coord) * freq;
    h[i] += j < fd ? sinf(arg) : cosf(arg);
}

// Sampler: schedule rows are {t, t_next, guidance, unused}.
__global__ void euler_sched_stats_kernel(const float *__restrict__ x, const float *__restrict__ vp,
                                         const float *__restrict__ vn, int64_t n, int C,
                                         const int32_t *__restrict__ offsets, int nbatch, const float *sched,
                                         const int *counter, float sigma_min, double *__restrict__ stats) {
    const float *s = sched + 4 * (*counter);
    cfg_stats_rows(x, vp, vn, n, C, offsets, nbatch, s[0], s[2], sigma_min, stats);
}

__global__ void euler_sched_kernel(float *__restrict__ x, const float *__restrict__ vp, const float *__restrict__ vn,
                                   int64_t n, int C, const int32_t *__restrict__ offsets, int nbatch,
                                   const float *sched, const int *counter, float gr, float sigma_min,
                                   const double *__restrict__ stats, float *__restrict__ x_model, int ldm) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n * C) return;
    const float *s = sched + 4 * (*counter);
    const float t = s[0], dt = s[0] - s[1], g = s[2];
    const float p = vp[i];
    float pred = g * p + (1.0f - g) * vn[i];
    if (stats) {
        const int64_t row = i / C;
        const int b = batch_of_row(offsets, nbatch, row);
        const double cnt = static_cast<double>(offsets[b + 1] - offsets[b]) * C;
        const double m0 = stats[4 * b] / cnt, m1 = stats[4 * b + 2] / cnt;
        const float sp = static_cast<float>(sqrt(fmax(stats[4 * b + 1] / cnt - m0 * m0, 0.0)));
        const float sc = static_cast<float>(sqrt(fmax(stats[4 * b + 3] / cnt - m1 * m1, 0.0)));
        const float ratio = sc != 0.0f ? sp / sc : 1.0f;
        const float a = 1.0f - sigma_min, bb = sigma_min + a * t;
        float x0 = a * x[i] - bb * pred;
        x0 = gr * (x0 * ratio) + (1.0f - gr) * x0;
        pred = (a * x[i] - x0) / bb;
    }
    const float nx = x[i] - dt * pred;
    x[i] = nx;
    // next forward's input: conditional and unconditional copies (rows of
    // ldm >= C columns; columns [C, ldm) hold the fixed concat condition)
    const int64_t r = i / C, c = i - r * C;
    x_model[r * ldm + c] = nx;
    x_model[(n + r) * ldm + c] = nx;
}

__global__ void advance_kernel(int *counter) { *counter += 1; }

}  // namespace
}  // namespace p3d

using namespace p3d;

namespace {

struct DevBlock {
    float *modulation = nullptr, *qkv_b = nullptr, *q_gamma = nullptr, *k_gamma = nullptr, *out_b = nullptr;
    float *norm2_w = nullptr, *norm2_b = nullptr, *cq_b = nullptr, *ckv_b = nullptr, *cq_gamma = nullptr;
    float *ck_gamma = nullptr, *co_b = nullptr, *proj_b = nullptr, *mlp0_b = nullptr, *mlp2_b = nullptr;
    uint16_t *qkv_w = nullptr, *out_w = nullptr, *cq_w = nullptr, *ckv_w = nullptr, *co_w = nullptr;
    uint16_t *proj_w = nullptr, *mlp0_w = nullptr, *mlp2_w = nullptr;
};

struct DevRes {
    float *gn1_w = nullptr, *gn1_b = nullptr, *conv1_b = nullptr, *gn2_w = nullptr, *gn2_b = nullptr,
          *conv2_b = nullptr;
    uint16_t *conv1_w = nullptr, *conv2_w = nullptr;
};

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

}  // namespace

struct p3d_flow {
    p3d_ctx *ctx = nullptr;
    p3d_flow_hparams hp{};
    int C = 0, in_pad = 0, cond_pad = 0, proj_pad = 0;
    std::vector<void *> allocs;  // weights: freed with the flow
    // Topology + workspaces, one buffer per member pointer (keyed by its
    // address).  prepare() reuses a buffer while it is large enough, so a new
    // coordinate set of the same or smaller size rebinds no pointer.
    struct PoolBuf {
        void *ptr = nullptr;
        size_t bytes = 0;
    };
    std::unordered_map<void *, PoolBuf> pool;
    bool pool_grew = false;
    bool in_prepare = false;
    // weights
    uint16_t *input_w = nullptr, *output_w = nullptr;
    float *input_b = nullptr, *output_b = nullptr, *t_w0 = nullptr, *t_b0 = nullptr, *t_w2 = nullptr, *t_b2 = nullptr,
          *mod_w = nullptr, *mod_b = nullptr;
    std::vector<DevBlock> blocks;
    std::vector<DevRes> io_in, io_out;
    // topology
    bool prepared = false;
    int batch = 0;
    int64_t n = 0, nt = 0, T = 0, max_fine = 0, max_trunk = 0, max_ctx = 0;
    int32_t *coords = nullptr, *trunk_coords = nullptr, *fine_off = nullptr, *trunk_off = nullptr, *ctx_off = nullptr;
    int32_t *nbr = nullptr, *parent = nullptr, *child = nullptr;
    // fine level in neighbour-pattern order: fine row i is the caller's row
    // perm[i] (null: caller order); conv taps per 256-row tile
    int32_t *perm = nullptr;
    uint32_t *fine_taps = nullptr;
    int32_t *summary = nullptr;  // prepare's device-side checks and offsets (check_batch_kernel)
    int32_t *order_ws = nullptr;  // p3d_conv_row_order scratch (pooled)
    float *out_tmp = nullptr;
    // workspaces
    float *h = nullptr, *hf = nullptr, *ftmp = nullptr, *tfreq = nullptr, *temb = nullptr, *temb2 = nullptr,
          *tmod = nullptr, *mods = nullptr, *x_model = nullptr, *vel = nullptr, *sched = nullptr, *ts = nullptr;
    // 16-bit operand buffers (dt = P3D_F16 or P3D_BF16)
    uint16_t *xn = nullptr, *qkv = nullptr, *attn = nullptr, *mlp = nullptr, *kv = nullptr, *cq = nullptr,
             *ctx_bf = nullptr, *proj_bf = nullptr, *x_in = nullptr, *fbf = nullptr;
    int dt = P3D_F16;
    double *stats = nullptr;
    float *rope = nullptr;  // [nt][32] (cos, sin) of the trunk coordinates, head_dim 64 only
    int *counter = nullptr;
    float *x_state = nullptr, *proj_model = nullptr;  // sampler-owned copies of x / proj
    cudaStream_t stream = nullptr;
    std::string error;
    int64_t launches_per_step = 0;
    std::vector<int32_t> h_fine_off, h_ctx_off, h_trunk_off;  // host copies of the batch / condition offsets
    int32_t *hash_ws = nullptr, *down_grid = nullptr;  // prepare-time scratch (pooled)
    int64_t *down_m = nullptr;
    // Shape of the topology the cached step graph was captured for.
    std::vector<int64_t> graph_shape;
    // Cached CUDA graph of one sampler step; it reads only the buffers above,
    // so it stays valid across sample() calls until prepare() rebinds them or
    // a captured scalar (rescale, sigma_min) changes.
    cudaGraphExec_t step_graph = nullptr;
    float graph_gr = -1.0f, graph_sigma = -1.0f;

    template <typename T>
    int alloc(T **p, int64_t count) {
        if (count <= 0) count = 1;
        const size_t bytes = sizeof(T) * static_cast<size_t>(count);
        if (in_prepare) {
            PoolBuf &b = pool[reinterpret_cast<void *>(p)];
            if (b.bytes < bytes) {
                if (b.ptr) cudaFree(b.ptr);
                b.ptr = nullptr;
                b.bytes = 0;
                pool_grew = true;
                cudaError_t e = cudaMalloc(&b.ptr, bytes);
                if (e != cudaSuccess)
                    return set_error(ctx, P3D_ERR_CUDA, std::string("cudaMalloc: ") + cudaGetErrorString(e));
                b.bytes = bytes;
            }
            *p = static_cast<T *>(b.ptr);
            return P3D_OK;
        }
        *p = nullptr;
        cudaError_t e = cudaMalloc(reinterpret_cast<void **>(p), bytes);
        if (e != cudaSuccess) return set_error(ctx, P3D_ERR_CUDA, std::string("cudaMalloc: ") + cudaGetErrorString(e));
        allocs.push_back(*p);
        return P3D_OK;
    }
    void reset_topology();
    void drop_graph() {
        if (step_graph) cudaGraphExecDestroy(step_graph);
        step_graph = nullptr;
        graph_shape.clear();
    }
    ~p3d_flow() {
        if (stream) cudaStreamSynchronize(stream);
        drop_graph();
        for (auto &kv : pool) cudaFree(kv.second.ptr);
        for (void *p : allocs) cudaFree(p);
        if (stream) cudaStreamDestroy(stream);
    }
};

namespace {


int upload16(p3d_flow *f, const float *src, int64_t rows, int64_t cols, int64_t cols_pad, uint16_t **dst) {
    if (!src) return set_error(f->ctx, P3D_ERR_INVALID, "missing SLat flow weight");
    int rc = f->alloc(dst, rows * cols_pad);
    if (rc) return rc;
    return pad16(f->ctx, src, rows, static_cast<int>(cols), static_cast<int>(cols_pad), *dst, f->dt);
}

int copy_f32(p3d_flow *f, const float *src, int64_t count, float **dst, bool required = true) {
    if (!src) {
        *dst = nullptr;
        return required ? set_error(f->ctx, P3D_ERR_INVALID, "missing SLat flow tensor") : P3D_OK;
    }
    int rc = f->alloc(dst, count);
    if (rc) return rc;
    P3D_CUDA(f->ctx, cudaMemcpyAsync(*dst, src, sizeof(float) * count, cudaMemcpyDeviceToDevice, f->ctx->stream));
    return P3D_OK;
}

#define P3D_TRY(expr)          \
    do {                       \
        int rc_ = (expr);      \
        if (rc_) return rc_;   \
    } while (0)

// ----------------------------------------------------------- the forward
// Runs on ctx->stream (the flow's stream while sampling).  x: f32 [n, in].
// ts / ts_stride / counter / mult feed the timestep embedding.
int forward_impl(p3d_flow *f, const float *x, const float *ts, int ts_stride, const int *counter, float mult,
                 const float *proj, float *out) {
    p3d_ctx *ctx = f->ctx;
    const p3d_flow_hparams &hp = f->hp;
    const int C = f->C, H = hp.num_heads, B = f->batch;
    const int64_t n = f->n, nt = f->nt;
    const bool io = hp.io_resblocks > 0;
    const int dt = f->dt;
    // timestep MLP -> SiLU -> 6C modulation (src/slat_flow.cpp:208-222)
    temb_freq_kernel<<<B, 128, 0, ctx->stream>>>(ts, ts_stride, counter, mult, B, 256, f->tfreq);
    P3D_TRY(check_launch(ctx, "temb_freq"));
    P3D_TRY(small_linear(ctx, f->tfreq, B, 256, f->t_w0, f->t_b0, C, f->temb, 0, 1));
    P3D_TRY(small_linear(ctx, f->temb, B, C, f->t_w2, f->t_b2, C, f->temb2, 0, 0));
    P3D_TRY(small_linear(ctx, f->temb2, B, C, f->mod_w, f->mod_b, 6 * C, f->tmod, 2, 0));
    // input linear
    P3D_TRY(pad16(ctx, x, n, hp.in_channels, f->in_pad, f->x_in, dt, io ? f->perm : nullptr));
    float *hin = io ? f->hf : f->h;
    P3D_TRY(p3d_linear(ctx, f->x_in, f->in_pad, f->input_w, dt, f->input_b, n, C, f->in_pad, hin, C, P3D_F32, P3D_EPI_NONE,
                       nullptr, 0, nullptr, 0));
    if (io) {
        for (const DevRes &r : f->io_in) {
            P3D_TRY(p3d_group_norm_silu(ctx, f->hf, n, C, hp.groups, 1e-5f, r.gn1_w, r.gn1_b, f->fine_off, B, 1,
                                        f->stats, f->fbf, dt));
            P3D_TRY(p3d_subm_conv3d_taps(ctx, f->fbf, n, C, f->nbr, r.conv1_w, dt, r.conv1_b, C, f->ftmp, C, P3D_F32,
                                         P3D_EPI_NONE, nullptr, 0, nullptr, 0, f->fine_taps));
            P3D_TRY(p3d_group_norm_silu(ctx, f->ftmp, n, C, hp.groups, 1e-5f, r.gn2_w, r.gn2_b, f->fine_off, B, 1,
                                        f->stats, f->fbf, dt));
            P3D_TRY(p3d_subm_conv3d_taps(ctx, f->fbf, n, C, f->nbr, r.conv2_w, dt, r.conv2_b, C, f->hf, C, P3D_F32,
                                         P3D_EPI_RESIDUAL, nullptr, 0, nullptr, 0, f->fine_taps));
        }
        P3D_TRY(p3d_downsample_mean(ctx, f->hf, nt, C, 2, f->child, P3D_F32, f->h));
    }
    if (hp.pe_mode == 1) {
        ape_add_kernel<<<blocks_for(nt * C, 256), 256, 0, ctx->stream>>>(f->h, reinterpret_cast<const int4 *>(f->trunk_coords),
                                                                        nt, C);
        P3D_TRY(check_launch(ctx, "ape_add"));
    }
    const int hd = C / H;
    const float attn_scale = 1.0f / sqrtf(static_cast<float>(hd));
    const int mlp = hp.mlp_hidden;
    if (hp.proj_mode && proj) {
        P3D_TRY(pad16(ctx, proj, nt, hp.proj_in_channels, f->proj_pad, f->proj_bf, dt));
    }
    for (std::size_t bi = 0; bi < f->blocks.size(); ++bi) {
        const DevBlock &bw = f->blocks[bi];
        add_mod_kernel<<<blocks_for(static_cast<int64_t>(B) * 6 * C, 256), 256, 0, ctx->stream>>>(
            bw.modulation, f->tmod, B, 6 * C, f->mods);
        P3D_TRY(check_launch(ctx, "add_mod"));
        // self-attention branch (src/sparse_transformer.cpp:194-235)
        P3D_TRY(p3d_layernorm_modulate(ctx, f->h, nt, C, hp.norm_eps, nullptr, nullptr, f->mods, 6 * C, f->trunk_off,
                                       B, f->xn, dt));
        const int32_t *rope_coords = hp.pe_mode == 0 ? f->trunk_coords : nullptr;
        const bool fuse_heads = hd == 64;
        if (fuse_heads && (hp.qk_rms_norm || rope_coords)) {
            // q/k RMS norm and RoPE in the GEMM epilogue, from the f32 accumulators
            P3D_TRY(p3d_linear_headnorm(ctx, f->xn, C, bw.qkv_w, dt, bw.qkv_b, nt, 3 * C, C, f->qkv, 3 * C, dt,
                                        hp.qk_rms_norm ? 2 * C : 0, bw.q_gamma, rope_coords ? 2 * C : 0, f->rope));
        } else {
            P3D_TRY(p3d_linear(ctx, f->xn, C, bw.qkv_w, dt, bw.qkv_b, nt, 3 * C, C, f->qkv, 3 * C, dt, P3D_EPI_NONE,
                               nullptr, 0, nullptr, 0));
        }
        if (!fuse_heads && (hp.qk_rms_norm || rope_coords)) {
            P3D_TRY(p3d_qk_rmsnorm_rope(ctx, f->qkv, nt, 3 * C, H, C / H, hp.qk_rms_norm ? bw.q_gamma : nullptr,
                                        rope_coords, hp.rope_freq_min, hp.rope_freq_base, dt));
            P3D_TRY(p3d_qk_rmsnorm_rope(ctx, f->qkv + C, nt, 3 * C, H, C / H, hp.qk_rms_norm ? bw.k_gamma : nullptr,
                                        rope_coords, hp.rope_freq_min, hp.rope_freq_base, dt));
        }
        P3D_TRY(p3d_varlen_attention(ctx, f->qkv, 3 * C, f->qkv + C, 3 * C, f->qkv + 2 * C, 3 * C, f->attn, C,
                                     f->trunk_off, f->trunk_off, B, f->max_trunk, nt, nt, H, C / H, attn_scale, dt));
        P3D_TRY(p3d_linear(ctx, f->attn, C, bw.out_w, dt, bw.out_b, nt, C, C, f->h, C, P3D_F32, P3D_EPI_RESIDUAL,
                           f->mods + 2 * C, 6 * C, f->trunk_off, B));
        // cross-attention branch (:237-275)
        P3D_TRY(p3d_layernorm_modulate(ctx, f->h, nt, C, hp.norm_eps, bw.norm2_w, bw.norm2_b, nullptr, 0, nullptr, 0,
                                       f->xn, dt));
        if (fuse_heads && hp.qk_rms_norm_cross) {
            P3D_TRY(p3d_linear_headnorm(ctx, f->xn, C, bw.cq_w, dt, bw.cq_b, nt, C, C, f->cq, C, dt, C, bw.cq_gamma, 0,
                                        nullptr));
        } else {
            P3D_TRY(p3d_linear(ctx, f->xn, C, bw.cq_w, dt, bw.cq_b, nt, C, C, f->cq, C, dt, P3D_EPI_NONE, nullptr, 0,
                               nullptr, 0));
            if (hp.qk_rms_norm_cross)
                P3D_TRY(p3d_qk_rmsnorm_rope(ctx, f->cq, nt, C, H, C / H, bw.cq_gamma, nullptr, 1.0f, 10000.0f, dt));
        }
        // this block's condition keys/values: computed once per condition (compute_kv)
        const uint16_t *kvb = f->kv + static_cast<int64_t>(bi) * f->T * 2 * C;
        P3D_TRY(p3d_varlen_attention(ctx, f->cq, C, kvb, 2 * C, kvb + C, 2 * C, f->attn, C, f->trunk_off,
                                     f->ctx_off, B, f->max_trunk, nt, f->T, H, C / H, attn_scale, dt));
        P3D_TRY(p3d_linear(ctx, f->attn, C, bw.co_w, dt, bw.co_b, nt, C, C, f->h, C, P3D_F32, P3D_EPI_RESIDUAL, nullptr, 0,
                           nullptr, 0));
        if (hp.proj_mode && proj)
            P3D_TRY(p3d_linear(ctx, f->proj_bf, f->proj_pad, bw.proj_w, dt, bw.proj_b, nt, C, f->proj_pad, f->h, C,
                               P3D_F32, P3D_EPI_RESIDUAL, nullptr, 0, nullptr, 0));
        // MLP branch (:277-290)
        P3D_TRY(p3d_layernorm_modulate(ctx, f->h, nt, C, hp.norm_eps, nullptr, nullptr, f->mods + 3 * C, 6 * C,
                                       f->trunk_off, B, f->xn, dt));
        P3D_TRY(p3d_linear(ctx, f->xn, C, bw.mlp0_w, dt, bw.mlp0_b, nt, mlp, C, f->mlp, mlp, dt, P3D_EPI_GELU_TANH,
                           nullptr, 0, nullptr, 0));
        P3D_TRY(p3d_linear(ctx, f->mlp, mlp, bw.mlp2_w, dt, bw.mlp2_b, nt, C, mlp, f->h, C, P3D_F32, P3D_EPI_RESIDUAL,
                           f->mods + 5 * C, 6 * C, f->trunk_off, B));
    }
    float *hout = f->h;
    if (io) {
        P3D_TRY(p3d_upsample_nearest(ctx, f->h, n, C, f->parent, P3D_F32, f->hf));
        for (const DevRes &r : f->io_out) {
            P3D_TRY(p3d_group_norm_silu(ctx, f->hf, n, C, hp.groups, 1e-5f, r.gn1_w, r.gn1_b, f->fine_off, B, 1,
                                        f->stats, f->fbf, dt));
            P3D_TRY(p3d_subm_conv3d_taps(ctx, f->fbf, n, C, f->nbr, r.conv1_w, dt, r.conv1_b, C, f->ftmp, C, P3D_F32,
                                         P3D_EPI_NONE, nullptr, 0, nullptr, 0, f->fine_taps));
            P3D_TRY(p3d_group_norm_silu(ctx, f->ftmp, n, C, hp.groups, 1e-5f, r.gn2_w, r.gn2_b, f->fine_off, B, 1,
                                        f->stats, f->fbf, dt));
            P3D_TRY(p3d_subm_conv3d_taps(ctx, f->fbf, n, C, f->nbr, r.conv2_w, dt, r.conv2_b, C, f->hf, C, P3D_F32,
                                         P3D_EPI_RESIDUAL, nullptr, 0, nullptr, 0, f->fine_taps));
        }
        hout = f->hf;
    }
    // final LayerNorm (eps 1e-5, src/slat_flow.cpp:244-248) + output linear
    uint16_t *xfin = io ? f->fbf : f->xn;
    P3D_TRY(p3d_layernorm_modulate(ctx, hout, n, C, 1e-5f, nullptr, nullptr, nullptr, 0, nullptr, 0, xfin, dt));
    float *y = (io && f->perm) ? f->out_tmp : out;
    P3D_TRY(p3d_linear(ctx, xfin, C, f->output_w, dt, f->output_b, n, hp.out_channels, C, y, hp.out_channels, P3D_F32,
                       P3D_EPI_NONE, nullptr, 0, nullptr, 0));
    if (y != out) {
        scatter_rows_kernel<<<blocks_for(n * hp.out_channels, 256), 256, 0, ctx->stream>>>(y, f->perm, n,
                                                                                          hp.out_channels, out);
        P3D_TRY(check_launch(ctx, "scatter_rows"));
    }
    return P3D_OK;
}

struct StreamSwap {
    p3d_ctx *ctx;
    cudaStream_t saved;
    StreamSwap(p3d_ctx *c, cudaStream_t s) : ctx(c), saved(c->stream) { ctx->stream = s; }
    ~StreamSwap() { ctx->stream = saved; }
};

}  // namespace

void p3d_flow::reset_topology() {
    prepared = false;
    n = nt = T = max_fine = max_trunk = max_ctx = 0;
    coords = trunk_coords = fine_off = trunk_off = ctx_off = nbr = parent = child = perm = nullptr;
    fine_taps = nullptr;
    summary = order_ws = nullptr;
    out_tmp = nullptr;
    h = hf = ftmp = tfreq = temb = temb2 = tmod = mods = x_model = vel = sched = ts = x_state = proj_model = nullptr;
    xn = qkv = attn = mlp = kv = cq = ctx_bf = proj_bf = x_in = fbf = nullptr;
    stats = nullptr;
    counter = nullptr;
    rope = nullptr;
    hash_ws = down_grid = nullptr;
    down_m = nullptr;
    h_trunk_off.clear();
}

// Sinusoidal absolute 3D position embedding added to f32 rows (no
// reference: the benchmark configs' "sinusoidal 3D absolute PE").
extern "C" int p3d_ape_add(p3d_ctx *ctx, const int32_t *coords, int64_t n, int channels, float *x) {
    if (!ctx) return P3D_ERR_INVALID;
    P3D_REQUIRE(ctx, coords && x && channels > 0 && n >= 0, "p3d_ape_add: bad argument");
    P3D_REQUIRE(ctx, (reinterpret_cast<uintptr_t>(coords) & 15) == 0, "p3d_ape_add: coords must be 16-byte aligned");
    if (n == 0) return P3D_OK;
    DeviceGuard dg(ctx->device);
    ape_add_kernel<<<blocks_for(n * channels, 256), 256, 0, ctx->stream>>>(x, reinterpret_cast<const int4 *>(coords), n,
                                                                          channels);
    return check_launch(ctx, "ape_add");
}

extern "C" int p3d_timestep_mlp(p3d_ctx *ctx, const float *timesteps, int batch, int channels, const float *w0,
                                const float *b0, const float *w2, const float *b2, const float *mod_w,
                                const float *mod_b, float *scratch, float *tmod) {
    if (!ctx) return P3D_ERR_INVALID;
    P3D_REQUIRE(ctx, timesteps && w0 && b0 && w2 && b2 && mod_w && mod_b && scratch && tmod && batch > 0 &&
                         channels > 0,
                "p3d_timestep_mlp: bad argument");
    DeviceGuard dg(ctx->device);
    float *freq = scratch, *t1 = scratch + static_cast<int64_t>(batch) * 256, *t2 = t1 + static_cast<int64_t>(batch) * channels;
    temb_freq_kernel<<<batch, 128, 0, ctx->stream>>>(timesteps, 1, nullptr, 1.0f, batch, 256, freq);
    P3D_TRY(check_launch(ctx, "temb_freq"));
    P3D_TRY(small_linear(ctx, freq, batch, 256, w0, b0, channels, t1, 0, 1));
    P3D_TRY(small_linear(ctx, t1, batch, channels, w2, b2, channels, t2, 0, 0));
    return small_linear(ctx, t2, batch, channels, mod_w, mod_b, 6 * channels, tmod, 2, 0);
}

extern "C" int p3d_flow_create(p3d_ctx *ctx, const p3d_flow_hparams *hp, const p3d_flow_weights *w, p3d_flow **out) {
    if (!ctx || !hp || !w || !out) return P3D_ERR_INVALID;
    DeviceGuard dg(ctx->device);
    *out = nullptr;
    const int C = hp->model_channels;
    P3D_REQUIRE(ctx, C > 0 && hp->num_heads > 0 && C % hp->num_heads == 0 && C / hp->num_heads == 64,
                "p3d_flow_create: head_dim must be 64");
    P3D_REQUIRE(ctx, C % 64 == 0, "p3d_flow_create: model_channels must be a multiple of 64");
    P3D_REQUIRE(ctx, hp->in_channels > 0 && hp->out_channels > 0 && hp->cond_channels > 0 && hp->num_blocks > 0,
                "invalid SLat flow hyperparameters");
    P3D_REQUIRE(ctx, hp->mlp_hidden > 0 && hp->mlp_hidden % 8 == 0, "p3d_flow_create: mlp_hidden must be a multiple of 8");
    P3D_REQUIRE(ctx, !hp->proj_mode || hp->proj_in_channels > 0, "SLat flow projection channels must be positive");
    P3D_REQUIRE(ctx, !(hp->proj_mode && hp->io_resblocks > 0), "p3d_flow_create: proj mode with io stages is undefined");
    P3D_REQUIRE(ctx, hp->io_resblocks == 0 || (hp->groups > 0 && C % hp->groups == 0),
                "p3d_flow_create: groups must divide model_channels");
    P3D_REQUIRE(ctx, w->blocks, "missing SLat flow block weights");
    p3d_flow *f = new p3d_flow();
    f->ctx = ctx;
    f->hp = *hp;
    f->C = C;
    f->in_pad = static_cast<int>(round_up(hp->in_channels, 8));
    f->cond_pad = static_cast<int>(round_up(hp->cond_channels, 8));
    f->proj_pad = static_cast<int>(round_up(hp->proj_in_channels > 0 ? hp->proj_in_channels : 8, 8));
    f->dt = hp->operand_dtype == P3D_BF16 ? P3D_BF16 : P3D_F16;
    auto fail = [&](int rc) {
        delete f;
        return rc;
    };
    int rc;
    if ((rc = upload16(f, w->input_w, C, hp->in_channels, f->in_pad, &f->input_w))) return fail(rc);
    if ((rc = copy_f32(f, w->input_b, C, &f->input_b))) return fail(rc);
    if ((rc = copy_f32(f, w->t_w0, static_cast<int64_t>(C) * 256, &f->t_w0))) return fail(rc);
    if ((rc = copy_f32(f, w->t_b0, C, &f->t_b0))) return fail(rc);
    if ((rc = copy_f32(f, w->t_w2, static_cast<int64_t>(C) * C, &f->t_w2))) return fail(rc);
    if ((rc = copy_f32(f, w->t_b2, C, &f->t_b2))) return fail(rc);
    if ((rc = copy_f32(f, w->mod_w, static_cast<int64_t>(6) * C * C, &f->mod_w))) return fail(rc);
    if ((rc = copy_f32(f, w->mod_b, 6 * C, &f->mod_b))) return fail(rc);
    if ((rc = upload16(f, w->output_w, hp->out_channels, C, C, &f->output_w))) return fail(rc);
    if ((rc = copy_f32(f, w->output_b, hp->out_channels, &f->output_b))) return fail(rc);
    const int mlp = hp->mlp_hidden;
    for (int i = 0; i < hp->num_blocks; ++i) {
        const p3d_block_weights &s = w->blocks[i];
        DevBlock d;
        if ((rc = copy_f32(f, s.modulation, 6 * C, &d.modulation))) return fail(rc);
        if ((rc = upload16(f, s.qkv_w, 3 * C, C, C, &d.qkv_w))) return fail(rc);
        if ((rc = copy_f32(f, s.qkv_b, 3 * C, &d.qkv_b))) return fail(rc);
        if (hp->qk_rms_norm) {
            // q and k gammas side by side: one [2C] vector for the fused qkv epilogue
            if (!s.q_gamma || !s.k_gamma) return fail(set_error(ctx, P3D_ERR_INVALID, "missing SLat flow tensor"));
            if ((rc = f->alloc(&d.q_gamma, 2 * C))) return fail(rc);
            d.k_gamma = d.q_gamma + C;
            if (cudaMemcpyAsync(d.q_gamma, s.q_gamma, sizeof(float) * C, cudaMemcpyDeviceToDevice, ctx->stream) !=
                    cudaSuccess ||
                cudaMemcpyAsync(d.k_gamma, s.k_gamma, sizeof(float) * C, cudaMemcpyDeviceToDevice, ctx->stream) !=
                    cudaSuccess)
                return fail(set_error(ctx, P3D_ERR_CUDA, "p3d_flow_create: gamma copy failed"));
        }
        if ((rc = upload16(f, s.out_w, C, C, C, &d.out_w))) return fail(rc);
        if ((rc = copy_f32(f, s.out_b, C, &d.out_b))) return fail(rc);
        if ((rc = copy_f32(f, s.norm2_w, C, &d.norm2_w))) return fail(rc);
        if ((rc = copy_f32(f, s.norm2_b, C, &d.norm2_b))) return fail(rc);
        if ((rc = upload16(f, s.cq_w, C, C, C, &d.cq_w))) return fail(rc);
        if ((rc = copy_f32(f, s.cq_b, C, &d.cq_b))) return fail(rc);
        if ((rc = upload16(f, s.ckv_w, 2 * C, hp->cond_channels, f->cond_pad, &d.ckv_w))) return fail(rc);
        if ((rc = copy_f32(f, s.ckv_b, 2 * C, &d.ckv_b))) return fail(rc);
        if ((rc = copy_f32(f, s.cq_gamma, C, &d.cq_gamma, hp->qk_rms_norm_cross != 0))) return fail(rc);
        if ((rc = copy_f32(f, s.ck_gamma, C, &d.ck_gamma, hp->qk_rms_norm_cross != 0))) return fail(rc);
        if ((rc = upload16(f, s.co_w, C, C, C, &d.co_w))) return fail(rc);
        if ((rc = copy_f32(f, s.co_b, C, &d.co_b))) return fail(rc);
        if (hp->proj_mode) {
            if ((rc = upload16(f, s.proj_w, C, hp->proj_in_channels, f->proj_pad, &d.proj_w))) return fail(rc);
            if ((rc = copy_f32(f, s.proj_b, C, &d.proj_b))) return fail(rc);
        }
        if ((rc = upload16(f, s.mlp0_w, mlp, C, C, &d.mlp0_w))) return fail(rc);
        if ((rc = copy_f32(f, s.mlp0_b, mlp, &d.mlp0_b))) return fail(rc);
        if ((rc = upload16(f, s.mlp2_w, C, mlp, mlp, &d.mlp2_w))) return fail(rc);
        if ((rc = copy_f32(f, s.mlp2_b, C, &d.mlp2_b))) return fail(rc);
        f->blocks.push_back(d);
    }
    for (int side = 0; side < 2; ++side) {
        const p3d_resblock_weights *src = side == 0 ? w->io_in : w->io_out;
        std::vector<DevRes> &dst = side == 0 ? f->io_in : f->io_out;
        for (int i = 0; i < hp->io_resblocks; ++i) {
            if (!src) return fail(set_error(ctx, P3D_ERR_INVALID, "missing io resblock weights"));
            const p3d_resblock_weights &s = src[i];
            DevRes d;
            const int64_t cw = static_cast<int64_t>(27) * C;
            if ((rc = copy_f32(f, s.gn1_w, C, &d.gn1_w))) return fail(rc);
            if ((rc = copy_f32(f, s.gn1_b, C, &d.gn1_b))) return fail(rc);
            if ((rc = upload16(f, s.conv1_w, cw, C, C, &d.conv1_w))) return fail(rc);
            if ((rc = copy_f32(f, s.conv1_b, C, &d.conv1_b))) return fail(rc);
            if ((rc = copy_f32(f, s.gn2_w, C, &d.gn2_w))) return fail(rc);
            if ((rc = copy_f32(f, s.gn2_b, C, &d.gn2_b))) return fail(rc);
            if ((rc = upload16(f, s.conv2_w, cw, C, C, &d.conv2_w))) return fail(rc);
            if ((rc = copy_f32(f, s.conv2_b, C, &d.conv2_b))) return fail(rc);
            dst.push_back(d);
        }
    }
    if (cudaStreamCreateWithFlags(&f->stream, cudaStreamNonBlocking) != cudaSuccess)
        return fail(set_error(ctx, P3D_ERR_CUDA, "cudaStreamCreate failed"));
    if (cudaStreamSynchronize(ctx->stream) != cudaSuccess)
        return fail(set_error(ctx, P3D_ERR_CUDA, "weight upload failed"));
    *out = f;
    return P3D_OK;
}

extern "C" int p3d_flow_destroy(p3d_flow *flow) {
    if (flow) {
        DeviceGuard dg(flow->ctx->device);
        cudaStreamSynchronize(flow->stream);
        delete flow;
    }
    return P3D_OK;
}

extern "C" int p3d_flow_prepare(p3d_flow *f, const int32_t *coords, int64_t n, int batch, int sx, int sy, int sz,
                                const int64_t *ctx_offsets_host) {
    if (!f) return P3D_ERR_INVALID;
    p3d_ctx *ctx = f->ctx;
    DeviceGuard dg(ctx->device);
    P3D_REQUIRE(ctx, coords && ctx_offsets_host && n > 0 && batch > 0, "p3d_flow_prepare: bad argument");
    // Rebinding reuses the previous coordinate set's buffers where they are
    // large enough; the cached step graph survives only if no buffer moved and
    // the topology's sizes and offsets are unchanged.  Weights stay resident.
    if (f->stream) P3D_CUDA(ctx, cudaStreamSynchronize(f->stream));
    f->reset_topology();
    f->pool_grew = false;
    struct PrepScope {
        p3d_flow *f;
        explicit PrepScope(p3d_flow *ff) : f(ff) { f->in_prepare = true; }
        ~PrepScope() { f->in_prepare = false; }
    } prep_scope(f);
    const p3d_flow_hparams &hp = f->hp;
    const int C = f->C;
    f->batch = batch;
    f->n = n;
    // Topology on the device; one copy of `summary` brings back what the host
    // needs (the batch check, the fault flag, batch offsets, trunk size): one
    // synchronisation per prepare.
    std::vector<int32_t> coff(batch + 1);
    for (int b = 0; b <= batch; ++b) coff[b] = static_cast<int32_t>(ctx_offsets_host[b]);
    for (int b = 0; b < batch; ++b) {
        if (coff[b + 1] <= coff[b]) return set_error(ctx, P3D_ERR_INVALID, "sparse cross-attention has an empty key sequence");
        f->max_ctx = std::max<int64_t>(f->max_ctx, coff[b + 1] - coff[b]);
    }
    f->T = coff[batch];
    f->h_ctx_off = coff;
    P3D_REQUIRE(ctx, (reinterpret_cast<uintptr_t>(coords) & 15) == 0, "p3d_flow_prepare: coords must be 16-byte aligned");
    const int64_t nsum = 2 * static_cast<int64_t>(batch) + 5;
    P3D_TRY(f->alloc(&f->summary, nsum));
    P3D_CUDA(ctx, cudaMemsetAsync(f->summary, 0, sizeof(int32_t) * nsum, ctx->stream));
    const int4 *cin = reinterpret_cast<const int4 *>(coords);
    check_batch_kernel<<<blocks_for(n, 256), 256, 0, ctx->stream>>>(cin, n, batch, f->summary);
    P3D_TRY(check_launch(ctx, "check_batch"));
    P3D_TRY(f->alloc(&f->fine_off, batch + 1));
    P3D_TRY(p3d_batch_offsets(ctx, coords, n, batch, f->fine_off));
    P3D_TRY(f->alloc(&f->ctx_off, batch + 1));
    P3D_CUDA(ctx, cudaMemcpyAsync(f->ctx_off, coff.data(), sizeof(int32_t) * (batch + 1), cudaMemcpyHostToDevice,
                                  ctx->stream));
    P3D_TRY(f->alloc(&f->coords, n * 4));
    const bool io = hp.io_resblocks > 0;
    if (io) {
        // Fine level: rows of each batch item stably sorted by neighbour
        // pattern inside chunks of P3D_CONV_ORDER_CHUNK_ROWS caller rows
        // (device radix sort), so a 256-row conv tile shares its missing taps
        // and the conv skips them while the tiles in flight keep the caller
        // order's locality; the input rows are gathered through perm and the
        // output rows scattered back.
        P3D_TRY(f->alloc(&f->nbr, 27 * n));
        const size_t wsb = p3d_neighbor_map27_workspace(n);
        P3D_TRY(f->alloc(&f->hash_ws, static_cast<int64_t>((wsb + 3) / 4)));
        P3D_TRY(p3d_neighbor_map27_ws(ctx, coords, n, f->hash_ws, wsb, f->nbr));
        const size_t owb = p3d_conv_row_order_workspace(n, batch, P3D_CONV_ORDER_CHUNK_ROWS);
        P3D_TRY(f->alloc(&f->order_ws, static_cast<int64_t>((owb + 3) / 4)));
        P3D_TRY(f->alloc(&f->perm, n));
        P3D_TRY(p3d_conv_row_order(ctx, coords, f->nbr, n, batch, P3D_CONV_ORDER_CHUNK_ROWS, f->order_ws, owb, f->perm));
        gather_coords_kernel<<<blocks_for(n, 256), 256, 0, ctx->stream>>>(cin, f->perm, n,
                                                                          reinterpret_cast<int4 *>(f->coords));
        P3D_TRY(check_launch(ctx, "gather_coords"));
        P3D_TRY(f->alloc(&f->out_tmp, n * hp.out_channels));
        P3D_TRY(p3d_neighbor_map27_ws(ctx, f->coords, n, f->hash_ws, wsb, f->nbr));
        P3D_TRY(f->alloc(&f->fine_taps, (n + 255) / 256));
        P3D_TRY(p3d_conv_tile_taps(ctx, f->nbr, n, f->fine_taps));
        // 2x downsample topology and the trunk's batch offsets
        const int64_t gints = p3d_downsample_grid_ints(batch, sx, sy, sz, 2);
        P3D_TRY(f->alloc(&f->trunk_coords, n * 4));
        P3D_TRY(f->alloc(&f->parent, n));
        P3D_TRY(f->alloc(&f->child, n * 8));
        P3D_TRY(f->alloc(&f->down_grid, gints));
        P3D_TRY(f->alloc(&f->down_m, 1));
        P3D_TRY(p3d_downsample_topology(ctx, f->coords, n, batch, sx, sy, sz, 2, f->down_grid, f->trunk_coords,
                                        f->parent, f->child, f->down_m));
        P3D_TRY(f->alloc(&f->trunk_off, batch + 1));
        offsets_dev_kernel<<<blocks_for(batch + 1, 128), 128, 0, ctx->stream>>>(
            reinterpret_cast<const int4 *>(f->trunk_coords), f->down_m, batch, f->trunk_off, f->summary + 4 + 2 * batch);
        P3D_TRY(check_launch(ctx, "trunk_offsets"));
        P3D_CUDA(ctx, cudaMemcpyAsync(f->summary + 3 + batch, f->trunk_off, sizeof(int32_t) * (batch + 1),
                                      cudaMemcpyDeviceToDevice, ctx->stream));
    } else {
        P3D_CUDA(ctx, cudaMemcpyAsync(f->coords, coords, sizeof(int32_t) * n * 4, cudaMemcpyDeviceToDevice, ctx->stream));
    }
    P3D_CUDA(ctx, cudaMemcpyAsync(f->summary + 2, f->fine_off, sizeof(int32_t) * (batch + 1), cudaMemcpyDeviceToDevice,
                                  ctx->stream));
    copy_fault_kernel<<<1, 1, 0, ctx->stream>>>(ctx->fault, f->summary + 1);
    P3D_TRY(check_launch(ctx, "copy_fault"));
    std::vector<int32_t> sum(static_cast<size_t>(nsum));
    P3D_CUDA(ctx, cudaMemcpyAsync(sum.data(), f->summary, sizeof(int32_t) * nsum, cudaMemcpyDeviceToHost, ctx->stream));
    P3D_CUDA(ctx, cudaStreamSynchronize(ctx->stream));  // the one synchronisation of prepare
    if (sum[1]) return p3d_ctx_check(ctx);  // a topology kernel latched a fault (duplicate, hash, key range)
    if (sum[0]) return set_error(ctx, P3D_ERR_INVALID, "sparse coordinates must be contiguous by batch");
    std::vector<int32_t> off(sum.begin() + 2, sum.begin() + 3 + batch);
    for (int b = 0; b < batch; ++b) f->max_fine = std::max<int64_t>(f->max_fine, off[b + 1] - off[b]);
    f->h_fine_off = off;
    if (io) {
        f->nt = sum[4 + 2 * batch];
        f->h_trunk_off.assign(sum.begin() + 3 + batch, sum.begin() + 4 + 2 * batch);
        for (int b = 0; b < batch; ++b)
            f->max_trunk = std::max<int64_t>(f->max_trunk, f->h_trunk_off[b + 1] - f->h_trunk_off[b]);
        P3D_TRY(f->alloc(&f->hf, n * C));
        P3D_TRY(f->alloc(&f->ftmp, n * C));
        P3D_TRY(f->alloc(&f->fbf, n * C));
        P3D_TRY(f->alloc(&f->stats, 3 * batch * hp.groups + 4 * batch));
    } else {
        f->nt = n;
        f->trunk_coords = f->coords;
        f->trunk_off = f->fine_off;
        f->max_trunk = f->max_fine;
        f->h_trunk_off = off;
        P3D_TRY(f->alloc(&f->stats, 4 * batch));
    }
    const int64_t nt = f->nt;
    P3D_TRY(f->alloc(&f->h, nt * C));
    P3D_TRY(f->alloc(&f->xn, std::max(nt, n) * C));
    P3D_TRY(f->alloc(&f->qkv, nt * 3 * C));
    P3D_TRY(f->alloc(&f->attn, nt * C));
    P3D_TRY(f->alloc(&f->cq, nt * C));
    P3D_TRY(f->alloc(&f->mlp, nt * hp.mlp_hidden));
    P3D_TRY(f->alloc(&f->kv, static_cast<int64_t>(hp.num_blocks) * f->T * 2 * C));  // all blocks' K/V
    P3D_TRY(f->alloc(&f->ctx_bf, f->T * f->cond_pad));
    P3D_TRY(f->alloc(&f->proj_bf, nt * f->proj_pad));
    P3D_TRY(f->alloc(&f->x_in, n * f->in_pad));
    P3D_TRY(f->alloc(&f->tfreq, batch * 256));
    P3D_TRY(f->alloc(&f->temb, batch * C));
    P3D_TRY(f->alloc(&f->temb2, batch * C));
    P3D_TRY(f->alloc(&f->tmod, batch * 6 * C));
    P3D_TRY(f->alloc(&f->mods, batch * 6 * C));
    P3D_TRY(f->alloc(&f->x_model, n * hp.in_channels));
    P3D_TRY(f->alloc(&f->vel, n * hp.out_channels));
    P3D_TRY(f->alloc(&f->ts, batch));
    P3D_TRY(f->alloc(&f->counter, 1));
    P3D_TRY(f->alloc(&f->sched, 4 * 4096));
    P3D_TRY(f->alloc(&f->x_state, n * hp.in_channels));
    if (hp.proj_mode) P3D_TRY(f->alloc(&f->proj_model, n * hp.proj_in_channels));
    if (hp.pe_mode == 0 && C / hp.num_heads == 64) {
        P3D_TRY(f->alloc(&f->rope, nt * 64));
        P3D_TRY(p3d_rope_table(ctx, f->trunk_coords, nt, 64, hp.rope_freq_min, hp.rope_freq_base, f->rope));
    }
    // Work issued here runs on ctx->stream; sampling orders the flow's own
    // stream after it with an event, and forward runs on ctx->stream.
    std::vector<int64_t> shape = {n, f->nt, f->T, batch, f->max_fine, f->max_trunk, f->max_ctx};
    shape.insert(shape.end(), off.begin(), off.end());
    shape.insert(shape.end(), coff.begin(), coff.end());
    shape.insert(shape.end(), f->h_trunk_off.begin(), f->h_trunk_off.end());
    if (f->pool_grew || shape != f->graph_shape) f->drop_graph();
    f->graph_shape = shape;
    f->prepared = true;
    return P3D_OK;
}

namespace {
int load_ctx(p3d_flow *f, const void *ctx_feats, int ctx_dtype) {
    p3d_ctx *ctx = f->ctx;
    const int cc = f->hp.cond_channels;
    if (ctx_dtype == P3D_F32) return pad16(ctx, static_cast<const float *>(ctx_feats), f->T, cc, f->cond_pad, f->ctx_bf, f->dt);
    P3D_REQUIRE(ctx, ctx_dtype == f->dt, "p3d_flow: 16-bit condition must use the model's operand dtype");
    P3D_REQUIRE(ctx, cc == f->cond_pad, "p3d_flow: 16-bit condition needs cond_channels % 8 == 0");
    P3D_CUDA(ctx, cudaMemcpyAsync(f->ctx_bf, ctx_feats, sizeof(uint16_t) * f->T * cc, cudaMemcpyDeviceToDevice,
                                  ctx->stream));
    return P3D_OK;
}
}  // namespace

namespace {
// Cross-attention keys/values of every block from the loaded condition
// tokens (ctx_bf): they depend on neither the timestep nor the latents, so
// a sampling run computes them once, outside the per-step graph.
int compute_kv(p3d_flow *f) {
    p3d_ctx *ctx = f->ctx;
    const p3d_flow_hparams &hp = f->hp;
    const int C = f->C, H = hp.num_heads, dt = f->dt;
    for (std::size_t bi = 0; bi < f->blocks.size(); ++bi) {
        const DevBlock &bw = f->blocks[bi];
        uint16_t *kvb = f->kv + static_cast<int64_t>(bi) * f->T * 2 * C;
        if (C / H == 64 && hp.qk_rms_norm_cross) {
            P3D_TRY(p3d_linear_headnorm(ctx, f->ctx_bf, f->cond_pad, bw.ckv_w, dt, bw.ckv_b, f->T, 2 * C, f->cond_pad,
                                        kvb, 2 * C, dt, C, bw.ck_gamma, 0, nullptr));
        } else {
            P3D_TRY(p3d_linear(ctx, f->ctx_bf, f->cond_pad, bw.ckv_w, dt, bw.ckv_b, f->T, 2 * C, f->cond_pad, kvb,
                               2 * C, dt, P3D_EPI_NONE, nullptr, 0, nullptr, 0));
            if (hp.qk_rms_norm_cross)
                P3D_TRY(p3d_qk_rmsnorm_rope(ctx, kvb, f->T, 2 * C, H, C / H, bw.ck_gamma, nullptr, 1.0f, 10000.0f, dt));
        }
    }
    return P3D_OK;
}
}  // namespace

extern "C" int p3d_flow_forward(p3d_flow *f, const float *x, const float *timesteps, const void *ctx_feats,
                                int ctx_dtype, const float *proj, float *out) {
    if (!f) return P3D_ERR_INVALID;
    p3d_ctx *ctx = f->ctx;
    DeviceGuard dg(ctx->device);
    P3D_REQUIRE(ctx, f->prepared, "p3d_flow_forward: call p3d_flow_prepare first");
    P3D_REQUIRE(ctx, x && timesteps && ctx_feats && out, "SLat flow input, timestep, or context shape mismatch");
    P3D_REQUIRE(ctx, !f->hp.proj_mode || proj, "SLat flow projection context shape mismatch");
    P3D_TRY(load_ctx(f, ctx_feats, ctx_dtype));
    P3D_TRY(compute_kv(f));
    return forward_impl(f, x, timesteps, 1, nullptr, 1.0f, proj, out);
}

extern "C" int p3d_flow_sample(p3d_flow *f, float *x, const void *ctx_feats, int ctx_dtype, const float *proj,
                               const p3d_sampler_config *cfg) {
    return p3d_flow_sample_concat(f, x, ctx_feats, ctx_dtype, proj, nullptr, 0, cfg);
}

extern "C" int p3d_flow_sample_concat(p3d_flow *f, float *x, const void *ctx_feats, int ctx_dtype, const float *proj,
                                      const float *concat, int concat_channels, const p3d_sampler_config *cfg) {
    if (!f || !cfg) return P3D_ERR_INVALID;
    p3d_ctx *ctx = f->ctx;
    DeviceGuard dg(ctx->device);
    P3D_REQUIRE(ctx, f->prepared, "p3d_flow_sample: call p3d_flow_prepare first");
    P3D_REQUIRE(ctx, x && ctx_feats, "p3d_flow_sample: null pointer");
    P3D_REQUIRE(ctx, f->batch % 2 == 0, "p3d_flow_sample: batch must be 2 x images (conditional, unconditional)");
    P3D_REQUIRE(ctx, concat_channels >= 0 && (concat_channels == 0) == (concat == nullptr),
                "SLat flow concat condition shape or coordinates mismatch");
    P3D_REQUIRE(ctx, f->hp.in_channels == f->hp.out_channels + concat_channels,
                concat_channels ? "SLat stage concat condition does not match model input metadata"
                                : "p3d_flow_sample: in/out channels differ");
    P3D_REQUIRE(ctx, !f->hp.proj_mode || proj, "SLat flow projection context shape mismatch");
    P3D_REQUIRE(ctx, cfg->steps > 0 && cfg->steps < 4096 && cfg->sigma_min >= 0.0f && cfg->sigma_min < 1.0f &&
                         cfg->rescale_t > 0.0f && cfg->guidance_rescale >= 0.0f &&
                         cfg->guidance_interval_min <= cfg->guidance_interval_max,
                "invalid flow Euler sampler configuration");
    const int I = f->batch / 2;
    const int64_t half = f->h_fine_off[I];
    P3D_REQUIRE(ctx, 2 * half == f->n, "p3d_flow_sample: unconditional half must mirror the conditional half");
    const int ch = f->hp.out_channels;   // sampler state columns
    const int ldm = f->hp.in_channels;   // model input: [state | concat]
    // t schedule (src/flow_sampler.cpp:268-286), computed in f32 like the reference
    std::vector<float> sched(4 * (cfg->steps + 1), 0.0f);
    const float steps = static_cast<float>(cfg->steps);
    for (int s = 0; s < cfg->steps; ++s) {
        const float lin = 1.0f - static_cast<float>(s) / steps;
        const float den = 1.0f + (cfg->rescale_t - 1.0f) * lin;
        const float t = cfg->rescale_t * lin / den;
        const float nl = 1.0f - static_cast<float>(s + 1) / steps;
        const float nden = 1.0f + (cfg->rescale_t - 1.0f) * nl;
        const float tn = cfg->rescale_t * nl / nden;
        if (!(den > 0.0f) || !(nden > 0.0f))
            return set_error(ctx, P3D_ERR_INVALID, "flow Euler timestep schedule is not finite");
        const bool in_interval = t >= cfg->guidance_interval_min && t <= cfg->guidance_interval_max;
        sched[4 * s] = t;
        sched[4 * s + 1] = tn;
        sched[4 * s + 2] = in_interval ? cfg->guidance_strength : 1.0f;
    }
    StreamSwap swap(ctx, f->stream);
    cudaEvent_t ev;
    P3D_CUDA(ctx, cudaEventCreateWithFlags(&ev, cudaEventDisableTiming));
    cudaEventRecord(ev, swap.saved);  // order after the caller's stream
    cudaStreamWaitEvent(f->stream, ev, 0);
    int rc = P3D_OK;
    auto body = [&]() -> int {
        P3D_CUDA(ctx, cudaMemcpyAsync(f->sched, sched.data(), sizeof(float) * sched.size(), cudaMemcpyHostToDevice,
                                      f->stream));
        P3D_CUDA(ctx, cudaMemsetAsync(f->counter, 0, sizeof(int), f->stream));
        // condition: conditional tokens for items [0, I), zeros for [I, 2I)
        P3D_TRY(load_ctx(f, ctx_feats, ctx_dtype));
        const int64_t z0 = f->h_ctx_off[I], z1 = f->h_ctx_off[f->batch];
        P3D_CUDA(ctx, cudaMemsetAsync(f->ctx_bf + z0 * f->cond_pad, 0, sizeof(uint16_t) * (z1 - z0) * f->cond_pad,
                                      f->stream));
        P3D_TRY(compute_kv(f));
        if (f->hp.proj_mode) {
            const int64_t hp_rows = half * f->hp.proj_in_channels;
            P3D_CUDA(ctx, cudaMemcpyAsync(f->proj_model, proj, sizeof(float) * hp_rows, cudaMemcpyDeviceToDevice,
                                          f->stream));
            P3D_CUDA(ctx, cudaMemsetAsync(f->proj_model + hp_rows, 0, sizeof(float) * hp_rows, f->stream));
        }
        // sampler state and model input [x | concat; x | concat] (the concat
        // condition is the same for both branches, src/slat_flow.cpp:1427-1441)
        P3D_CUDA(ctx, cudaMemcpyAsync(f->x_state, x, sizeof(float) * half * ch, cudaMemcpyDeviceToDevice, f->stream));
        for (int b = 0; b < 2; ++b) {
            float *dst = f->x_model + b * half * ldm;
            P3D_CUDA(ctx, cudaMemcpy2DAsync(dst, sizeof(float) * ldm, x, sizeof(float) * ch, sizeof(float) * ch, half,
                                            cudaMemcpyDeviceToDevice, f->stream));
            if (concat_channels)
                P3D_CUDA(ctx, cudaMemcpy2DAsync(dst + ch, sizeof(float) * ldm, concat, sizeof(float) * concat_channels,
                                                sizeof(float) * concat_channels, half, cudaMemcpyDeviceToDevice,
                                                f->stream));
        }
        const bool rescale = cfg->guidance_rescale > 0.0f;
        const float gr = cfg->guidance_rescale, sigma = cfg->sigma_min;
        auto one_step = [&]() -> int {
            P3D_TRY(forward_impl(f, f->x_model, f->sched, 0, f->counter, 1000.0f, f->proj_model, f->vel));
            const float *vp = f->vel, *vn = f->vel + half * ch;
            if (rescale) {
                P3D_CUDA(ctx, cudaMemsetAsync(f->stats, 0, sizeof(double) * 4 * I, f->stream));
                euler_sched_stats_kernel<<<blocks_for(ceil_div(half, kStatsRowsPerWarp), 8), 256, 0, f->stream>>>(
                    f->x_state, vp, vn, half, ch, f->fine_off, I, f->sched, f->counter, sigma, f->stats);
                P3D_TRY(check_launch(ctx, "euler_stats"));
            }
            euler_sched_kernel<<<blocks_for(half * ch, 256), 256, 0, f->stream>>>(
                f->x_state, vp, vn, half, ch, f->fine_off, I, f->sched, f->counter, gr, sigma,
                rescale ? f->stats : nullptr, f->x_model, ldm);
            P3D_TRY(check_launch(ctx, "euler_sched"));
            advance_kernel<<<1, 1, 0, f->stream>>>(f->counter);
            return check_launch(ctx, "advance");
        };
        int first = 0;
        if (cfg->use_graph && f->step_graph && (f->graph_gr != gr || f->graph_sigma != sigma)) {
            cudaGraphExecDestroy(f->step_graph);
            f->step_graph = nullptr;
        }
        if (cfg->use_graph && !f->step_graph) {
            // One eager step (first launches of every kernel happen outside
            // capture), then capture one step for replay.
            const int64_t l0 = ctx->launches;
            P3D_TRY(one_step());
            f->launches_per_step = ctx->launches - l0;
            first = 1;
            if (cfg->steps > 1) {
                cudaGraph_t graph = nullptr;
                P3D_CUDA(ctx, cudaStreamBeginCapture(f->stream, cudaStreamCaptureModeThreadLocal));
                const int rc_cap = one_step();
                const cudaError_t e = cudaStreamEndCapture(f->stream, &graph);
                if (rc_cap) {
                    if (graph) cudaGraphDestroy(graph);
                    return rc_cap;
                }
                if (e != cudaSuccess) return set_error(ctx, P3D_ERR_CUDA, std::string("capture: ") + cudaGetErrorString(e));
                const cudaError_t ie = cudaGraphInstantiate(&f->step_graph, graph, 0);
                cudaGraphDestroy(graph);
                if (ie != cudaSuccess) {
                    f->step_graph = nullptr;
                    return set_error(ctx, P3D_ERR_CUDA, "cudaGraphInstantiate failed");
                }
                f->graph_gr = gr;
                f->graph_sigma = sigma;
            }
        }
        for (int s = first; s < cfg->steps; ++s) {
            if (cfg->use_graph && f->step_graph) {
                P3D_CUDA(ctx, cudaGraphLaunch(f->step_graph, f->stream));
                ctx->count_launches(f->launches_per_step);
            } else {
                const int64_t l0 = ctx->launches;
                P3D_TRY(one_step());
                f->launches_per_step = ctx->launches - l0;
            }
        }
        P3D_CUDA(ctx, cudaMemcpyAsync(x, f->x_state, sizeof(float) * half * ch, cudaMemcpyDeviceToDevice, f->stream));
        return P3D_OK;
    };
    rc = body();
    cudaEventRecord(ev, f->stream);
    cudaStreamWaitEvent(swap.saved, ev, 0);
    cudaEventDestroy(ev);
    return rc;
}

extern "C" int64_t p3d_flow_launches_per_step(const p3d_flow *f) { return f ? f->launches_per_step : 0; }
