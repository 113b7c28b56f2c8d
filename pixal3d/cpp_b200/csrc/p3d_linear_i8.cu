// Matrix product of 8-bit integers with scales for each row and channel.
//
//   y[i, j] = act( (float(sum_k x[i, k] w[j, k]) xs[i]) ws[j] + bias[j] )
//
// The sum is exact in 32-bit integers (k <= 131071 keeps 128 * 128 * k below
// 2^31); it is rounded once to f32 (24 bits), then scaled in f32.
//
// More than a few rows run on the tensor cores (tcgen05.mma kind::i8, 32-bit
// integer accumulators in TMEM).  CTA = 18 warps, persistent over the tiles:
//   warps 0-15  epilogue: four per TMEM lane quarter, each its share of the
//               columns; lane = row; scales, bias, activation, then boxes of
//               32 rows x 64 bytes staged in shared memory and written by TMA
//   warp  16    TMEM allocator, one thread issues the MMAs
//   warp  17    one thread issues the TMA loads
// BK = 128 bytes (one swizzle atom row), four MMAs of K = 32 a stage; two
// accumulators in TMEM, so a tile's epilogue runs under the next one's MMAs.
// Every wait is bounded.
//
// What bounds it, 8184 x 1024 x 4096 to bf16 (68.6 Gop): 33.3 us = 2060 Top/s,
// with GELU 38.3; the MMAs alone take 22.5 us (3055 Top/s), with their loads
// 24.8.  The rest is the epilogue's share of shared memory and issue slots,
// which at K = 1024 is one pass over 64 KB for eight stages.  Tried where GELU
// took the hardware tanh (35.0 us): eight epilogue warps instead of 16 43.1 us
// (their loads' latency showed), 4 KB staging slots and so three stages instead
// of four 37.7, CTA pairs (cta_group::2, half the loads of w) 38.3 (without GELU
// 35.4 against 33.1) and 2 % faster at 8184 x 4096 x 4096 (101.0 / 102.7 us), so
// there are none.
#include <algorithm>
#include <cstring>

#include "p3d_common.cuh"

namespace p3d {
namespace {

struct I8Params {
    const int8_t *x, *w;
    int64_t ldx, ldw;
    const float *xs, *ws, *bias;
    void *out;
    int64_t ldo;
    const float *gate;
    int64_t gate_ld;
    const int32_t *batch_offsets;
    int nbatch;
    int64_t M, N;
    int K;
    int out_dtype;
    int epi;
    int *fault;
    int tma_out;    // the output is a TMA target (16-byte base and pitch)
    int wide_cols;  // w_scale and bias start on 16-byte boundaries
};

// GELU, tanh form, as x sigmoid(2 y): a few 2^-23 of the result and of its slope.
// (0.5 x (1 + tanh(y)) by the hardware tanh is 2^-12 |x| off wherever the two
// cancel: 20 % of the value at x = -3, in 16 bits too.)
__device__ __forceinline__ float gelu_f(float x) {
    const float y = 0.7978845608028654f * fmaf(0.044715f * x, x * x, x);
    return __fdividef(x, 1.0f + __expf(-2.0f * y));
}

__device__ __forceinline__ float act_f(float v, int epi) {
    if (epi & P3D_EPI_GELU_TANH) return gelu_f(v);
    if (epi & P3D_EPI_SILU) return silu_f(v);
    return v;
}

__device__ __forceinline__ void store_one(const I8Params &p, int64_t row, int64_t col, float v) {
    if (p.epi & P3D_EPI_RESIDUAL) {
        float g = 1.0f;
        if (p.gate) g = p.gate[static_cast<int64_t>(batch_of_row(p.batch_offsets, p.nbatch, row)) * p.gate_ld + col];
        static_cast<float *>(p.out)[row * p.ldo + col] += g * v;
        return;
    }
    if (p.out_dtype == P3D_F32)
        static_cast<float *>(p.out)[row * p.ldo + col] = v;
    else if (p.out_dtype == P3D_BF16)
        static_cast<__nv_bfloat16 *>(p.out)[row * p.ldo + col] = __float2bfloat16_rn(v);
    else
        static_cast<__half *>(p.out)[row * p.ldo + col] = __float2half_rn(v);
}

// 16 bytes of a row from byte k on.  The word that holds the row's end is read
// whole (rows start on 16-byte boundaries, so it lies in the same allocation).
__device__ __forceinline__ int4 load16(const int8_t *row, int k) { return __ldg(reinterpret_cast<const int4 *>(row + k)); }
// Bytes at or past K to zero; one operand is enough.
__device__ __forceinline__ int4 trim16(const int4 &v, int k, int K) {
    auto keep = [&](int w, int n) { return n >= 4 ? w : n <= 0 ? 0 : static_cast<int>(static_cast<uint32_t>(w) & ((1u << (8 * n)) - 1u)); };
    const int n = K - k;
    return n >= 16 ? v : make_int4(keep(v.x, n), keep(v.y, n - 4), keep(v.z, n - 8), keep(v.w, n - 12));
}

// Few rows: a warp takes NC channels and MR rows, its lanes stride over k.
constexpr int kRowThreads = 128;
template <int MR, int NC>
__global__ void __launch_bounds__(kRowThreads) linear_i8_rows_kernel(const I8Params p) {
    const int lane = threadIdx.x & 31;
    const int64_t col0 = (static_cast<int64_t>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5)) * NC;
    const int64_t row0 = static_cast<int64_t>(blockIdx.y) * MR;
    pdl_wait();
    pdl_trigger();
    if (col0 >= p.N) return;
    const int rows = static_cast<int>(min(static_cast<int64_t>(MR), p.M - row0));
    const int cols = static_cast<int>(min(static_cast<int64_t>(NC), p.N - col0));
    int acc[MR][NC];
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[r][c] = 0;
    // rows and channels past the last are the last again: no branch inside
    const int8_t *xr[MR], *wr[NC];
#pragma unroll
    for (int r = 0; r < MR; ++r) xr[r] = p.x + (row0 + min(r, rows - 1)) * p.ldx;
#pragma unroll
    for (int c = 0; c < NC; ++c) wr[c] = p.w + (col0 + min(c, cols - 1)) * p.ldw;
#pragma unroll 2
    for (int k = lane * 16; k < p.K; k += 512) {
        int4 b[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) b[c] = trim16(load16(wr[c], k), k, p.K);
#pragma unroll
        for (int r = 0; r < MR; ++r) {
            const int4 a = load16(xr[r], k);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                acc[r][c] = __dp4a(a.x, b[c].x, acc[r][c]);
                acc[r][c] = __dp4a(a.y, b[c].y, acc[r][c]);
                acc[r][c] = __dp4a(a.z, b[c].z, acc[r][c]);
                acc[r][c] = __dp4a(a.w, b[c].w, acc[r][c]);
            }
        }
    }
    // lane r * NC + c finishes output (r, c)
    int mine = 0;
#pragma unroll
    for (int r = 0; r < MR; ++r)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int s = __reduce_add_sync(0xffffffffu, acc[r][c]);
            if (lane == r * NC + c) mine = s;
        }
    const int r = lane / NC, c = lane % NC;
    if (r < rows && c < cols) {
        const int64_t row = row0 + r, col = col0 + c;
        const float bias = p.bias ? p.bias[col] : 0.0f;
        store_one(p, row, col, act_f(fmaf(static_cast<float>(mine) * p.xs[row], p.ws[col], bias), p.epi));
    }
}

template <int MR, int NC>
int launch_rows(p3d_ctx *ctx, const I8Params &p) {
    static_assert(MR * NC <= 32, "one lane an output");
    dim3 grid(static_cast<unsigned>(ceil_div(p.N, kRowThreads / 32 * NC)), static_cast<unsigned>(ceil_div(p.M, MR)));
    P3D_CUDA(ctx, launch_pdl(linear_i8_rows_kernel<MR, NC>, grid, dim3(kRowThreads), 0, ctx->stream, p));
    return check_launch(ctx, "linear_i8_rows");
}

// D(tmem) (+)= A(smem) B(smem)^T, 8-bit integers, 32-bit integer accumulators.
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor, kind::i8: D s32 (2 at bits 4-5), A and B signed (1
// at bits 7-9 and 10-12), both K-major, N >> 3 at 17-22, M >> 4 at 24-28.
constexpr uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

constexpr int kTileM = 128;   // rows of one CTA
constexpr int kBK = 128;      // bytes of k a stage
constexpr int kEpiWarps = 16;
constexpr int kMmaWarp = kEpiWarps, kTmaWarp = kEpiWarps + 1;
constexpr int kThreadsT = 32 * (kEpiWarps + 2);

// One epilogue warp's staging: 32 rows x 64 bytes (32 16-bit or 16 f32
// columns) in the 64-byte swizzle (16-byte chunk c of row r at c ^ (r / 2 % 4),
// so the eight lanes of a store phase hit eight different bank groups).
constexpr int kSlotBytes = 2048;

template <int BN>
struct TileCfg {
    static constexpr int COLS = BN * 4 / kEpiWarps < 32 ? 32 : BN * 4 / kEpiWarps;  // accumulator columns of one epilogue warp
    static constexpr int DRAIN = 4 * (BN / COLS);                                   // epilogue warps that work
    static constexpr int A_BYTES = kTileM * kBK;
    static constexpr int B_BYTES = BN * kBK;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int EPI = DRAIN * kSlotBytes;
    static constexpr int FIT = (232448 - EPI - 1024 - 512) / STAGE;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int TMEM = 2 * BN;  // two accumulators
    static constexpr int SMEM = STAGES * STAGE + EPI + 1024 + 512;
    static_assert(TMEM == 128 || TMEM == 256 || TMEM == 512, "TMEM columns");
};

// Two values of gelu_f for 16-bit outputs: the exponential and the reciprocal
// approximate, 2^-21 of the result together (8184 x 1024 x 4096 to bf16: 38.3 us;
// one reciprocal for both 37.8, a cubic and a Newton step in its place 39.1, the
// hardware tanh 34.8).
__device__ __forceinline__ F2 gelu2(const F2 &x) {
    constexpr float c0 = -2.0f * 1.4426950408889634f * 0.7978845608028654f, c1 = c0 * 0.044715f;
    const F2 y = mul2(fma2(mul2(x, x), F2(c1, c1), F2(c0, c0)), x);
    float a, b;
    y.get(a, b);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
    const F2 d = add2(F2(a, b), F2(1.0f, 1.0f));
    d.get(a, b);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
    return mul2(x, F2(a, b));
}

// 32 accumulators of one row to outputs, columns col0.. (ncols of them exist).
// wide: the whole chunk exists and scales and bias lie on 16-byte boundaries.
__device__ __forceinline__ void finish32(const I8Params &p, float (&v)[32], float xs, int64_t row, int64_t col0, int ncols,
                                         bool wide) {
    const F2 xs2(xs, xs);
    const bool fast_gelu = (p.epi & P3D_EPI_GELU_TANH) && p.out_dtype != P3D_F32;
#pragma unroll
    for (int h = 0; h < 32; h += 16) {  // scales and bias of 16 columns at a time: their loads are in flight together
        float s[16], b[16];
        if (wide) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 t = __ldg(reinterpret_cast<const float4 *>(p.ws + col0 + h + i));
                s[i] = t.x, s[i + 1] = t.y, s[i + 2] = t.z, s[i + 3] = t.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = h + i < ncols ? __ldg(p.ws + col0 + h + i) : 0.0f;
        }
        if (!p.bias) {
#pragma unroll
            for (int i = 0; i < 16; ++i) b[i] = 0.0f;
        } else if (wide) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 t = __ldg(reinterpret_cast<const float4 *>(p.bias + col0 + h + i));
                b[i] = t.x, b[i + 1] = t.y, b[i + 2] = t.z, b[i + 3] = t.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) b[i] = h + i < ncols ? __ldg(p.bias + col0 + h + i) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            float &v0 = v[h + i], &v1 = v[h + i + 1];
            const F2 acc(static_cast<float>(__float_as_int(v0)), static_cast<float>(__float_as_int(v1)));
            const F2 r = fma2(mul2(acc, xs2), F2(s[i], s[i + 1]), F2(b[i], b[i + 1]));
            r.get(v0, v1);
        }
    }
    if (fast_gelu) {
#pragma unroll
        for (int i = 0; i < 32; i += 2) gelu2(F2(v[i], v[i + 1])).get(v[i], v[i + 1]);
    }
    if ((p.epi & P3D_EPI_GELU_TANH) && !fast_gelu) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = gelu_f(v[i]);
    } else if (p.epi & P3D_EPI_SILU) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = silu_f(v[i]);
    }
    if ((p.epi & P3D_EPI_RESIDUAL) && p.gate) {
        const float *g = p.gate + static_cast<int64_t>(batch_of_row(p.batch_offsets, p.nbatch, row)) * p.gate_ld + col0;
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= i < ncols ? __ldg(g + i) : 0.0f;
    }
}

__device__ __forceinline__ void prefetch_l1(const void *p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

// One epilogue warp's columns of an accumulator: rows row0 .. row0 + 31 (lane
// = row), columns n0 .. n0 + COLS - 1.
template <int COLS>
__device__ __forceinline__ void epilogue_i8(const I8Params &p, const CUtensorMap *tmo, uint32_t tacc, int64_t row0, int lane,
                                            int64_t n0, float xs, uint8_t *buf) {
    const int64_t row = row0 + lane;
    const bool f32 = p.out_dtype == P3D_F32;
    // 64 bytes of each row (lane) to columns col..
    auto put = [&](const uint4 *w, int64_t col) {
        if (p.tma_out && lane == 0) bulk_wait_read<0>();  // the slot's last box has been read
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; ++c) *reinterpret_cast<uint4 *>(buf + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) = w[c];
        if (p.tma_out) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (p.epi & P3D_EPI_RESIDUAL)
                    tma_reduce_add_2d(tmo, buf, static_cast<int>(col), static_cast<int>(row0));
                else
                    tma_store_2d(tmo, buf, static_cast<int>(col), static_cast<int>(row0));
                bulk_commit();
            }
            return;
        }
        // rows that start off a 16-byte boundary: consecutive lanes write
        // consecutive elements of a row
        __syncwarp();
        const int64_t rows = p.M - row0 < 32 ? p.M - row0 : 32;
        if (f32) {
            const int e = lane & 15;
            if (col + e < p.N) {
#pragma unroll 4
                for (int r = lane >> 4; r < rows; r += 2) {
                    const float y = *reinterpret_cast<const float *>(buf + r * 64 + (((e >> 2) ^ ((r >> 1) & 3)) << 4) + (e & 3) * 4);
                    float *o = static_cast<float *>(p.out) + (row0 + r) * p.ldo + col + e;
                    *o = p.epi & P3D_EPI_RESIDUAL ? *o + y : y;
                }
            }
        } else if (col + lane < p.N) {
            uint16_t *o = static_cast<uint16_t *>(p.out) + row0 * p.ldo + col + lane;
#pragma unroll 4
            for (int r = 0; r < rows; ++r, o += p.ldo)
                *o = *reinterpret_cast<const uint16_t *>(buf + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
        }
    };
    auto emit = [&](float(&v)[32], int c) {
        const int64_t col0 = n0 + c;
        const int ncols = static_cast<int>(p.N - col0 < 32 ? p.N - col0 : 32);
        finish32(p, v, xs, row < p.M ? row : p.M - 1, col0, ncols, p.wide_cols && ncols == 32);
        if (f32) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (col0 + 16 * h >= p.N) break;
                uint4 w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = make_uint4(__float_as_uint(v[16 * h + 4 * e]), __float_as_uint(v[16 * h + 4 * e + 1]),
                                      __float_as_uint(v[16 * h + 4 * e + 2]), __float_as_uint(v[16 * h + 4 * e + 3]));
                put(w, col0 + 16 * h);
            }
        } else {
            const bool bf = p.out_dtype == P3D_BF16;
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
                w[e] = bf ? pack2<__nv_bfloat16>(v[2 * e], v[2 * e + 1]) : pack2<__half>(v[2 * e], v[2 * e + 1]);
            uint4 u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
            put(u, col0);
        }
    };
    float v[32];
#pragma unroll 1
    for (int c = 0; c < COLS; c += 32) {
        if (n0 + c >= p.N) break;  // the whole warp
        __syncwarp();
        tmem_ld32(tacc + c, v);
        tmem_ld_wait_regs(v);
        emit(v, c);
    }
}

template <int BN>
__global__ void __launch_bounds__(kThreadsT, 1)
    linear_i8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                     const __grid_constant__ CUtensorMap tmap_o, const I8Params p) {
    using C = TileCfg<BN>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *smem_a = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    uint8_t *smem_b = smem_a + STAGES * C::A_BYTES;
    uint8_t *smem_o = smem_b + STAGES * C::B_BYTES;
    uint64_t *full = reinterpret_cast<uint64_t *>(smem_o + C::EPI);
    uint64_t *empty = full + STAGES;
    uint64_t *tfull = empty + STAGES;  // [2]
    uint64_t *tempty = tfull + 2;      // [2]
    uint64_t *done = tempty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t first = blockIdx.x, step = gridDim.x;
    const int64_t n_tiles = (p.N + BN - 1) / BN;
    const int64_t tiles = (p.M + kTileM - 1) / kTileM * n_tiles;
    const int kbs = (p.K + kBK - 1) / kBK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], C::DRAIN);
        }
        mbar_init(done, 1);
        fence_barrier_init();
        prefetch_tmap(&tmap_a);
        prefetch_tmap(&tmap_b);
        if (p.tma_out) prefetch_tmap(&tmap_o);
    }
    if (warp == kMmaWarp) {
        tmem_alloc(tmem_slot, C::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();

    if (warp == kTmaWarp) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int64_t t = first; t < tiles && ok; t += step) {
                const int m0 = static_cast<int>(t / n_tiles * kTileM);
                const int n0 = static_cast<int>(t % n_tiles * BN);
                for (int kb = 0; kb < kbs; ++kb) {
                    if (!(ok = mbar_wait(&empty[stage], phase ^ 1, p.fault))) break;
                    uint8_t *a = smem_a + stage * C::A_BYTES, *b = smem_b + stage * C::B_BYTES;
                    mbar_arrive_expect_tx(&full[stage], C::STAGE);
                    tma_load_2d(a, &tmap_a, &full[stage], kb * kBK, m0);
                    tma_load_2d(b, &tmap_b, &full[stage], kb * kBK, n0);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_i8(kTileM, BN);
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true, issued = false;
            for (int64_t t = first; t < tiles && ok; t += step) {
                if (!(ok = mbar_wait(&tempty[acc], acc_phase ^ 1, p.fault))) break;
                tc_fence_after();
                for (int kb = 0; kb < kbs; ++kb) {
                    if (!(ok = mbar_wait(&full[stage], phase, p.fault))) break;
                    tc_fence_after();
                    const uint32_t a = smem_u32(smem_a + stage * C::A_BYTES), b = smem_u32(smem_b + stage * C::B_BYTES);
#pragma unroll
                    for (int kk = 0; kk < kBK / 32; ++kk)
                        umma_i8(tmem + acc * BN, sw128_desc(a + kk * 32), sw128_desc(b + kk * 32), idesc,
                                      (kb > 0 || kk > 0) ? 1u : 0u);
                    issued = true;
                    umma_commit(&empty[stage]);
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (!ok) break;
                umma_commit(&tfull[acc]);
                acc ^= 1;
                if (acc == 0) acc_phase ^= 1;
            }
            if (issued) {  // no MMA is in flight when the TMEM is freed
                umma_commit(done);
                mbar_wait(done, 0, p.fault);
            }
        }
        __syncwarp();
    } else if (warp < C::DRAIN) {
        const int q = warp & 3, h = warp >> 2;
        uint8_t *buf = smem_o + warp * kSlotBytes;
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int64_t t = first; t < tiles; t += step) {
            const int64_t m0 = t / n_tiles * kTileM + q * 32, n0 = t % n_tiles * BN + h * C::COLS;
            // what the epilogue reads comes while the MMAs run
            const float xs = m0 + lane < p.M ? __ldg(p.xs + m0 + lane) : 0.0f;
            if (lane * 8 < C::COLS && n0 + lane * 8 < p.N) {
                prefetch_l1(p.ws + n0 + lane * 8);
                if (p.bias) prefetch_l1(p.bias + n0 + lane * 8);
            }
            if (!warp_wait<false>(&tfull[acc], acc_phase, p.fault)) break;
            tc_fence_after();
            if (m0 < p.M)
                epilogue_i8<C::COLS>(p, &tmap_o, tmem + acc * BN + h * C::COLS + (static_cast<uint32_t>(q * 32) << 16), m0,
                                     lane, n0, xs, buf);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[acc]);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
        }
        if (p.tma_out && lane == 0) bulk_wait_all();  // the staging stays until the stores have read it
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, C::TMEM);
}

// Operand map: rows x k bytes, boxes of 128 bytes x box_rows, 128-byte
// swizzle; bytes from k on read as zero.
int make_tmap_i8(p3d_ctx *ctx, CUtensorMap *map, const int8_t *base, int64_t rows, int64_t k, int64_t ld, int box_rows) {
    EncodeFn fn = get_encode_fn();
    if (!fn) return set_error(ctx, P3D_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    cuuint32_t box[2] = {kBK, static_cast<cuuint32_t>(box_rows)};
    cuuint32_t es[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(base), dims, strides, box, es,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(ctx, P3D_ERR_CUDA, "cuTensorMapEncodeTiled (8-bit) failed: " + std::to_string(r));
    return P3D_OK;
}

// Output map: boxes of 32 rows x 64 bytes, 64-byte swizzle.
int make_tmap_i8_out(p3d_ctx *ctx, CUtensorMap *map, const I8Params &p) {
    EncodeFn fn = get_encode_fn();
    if (!fn) return set_error(ctx, P3D_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    const bool f32 = p.out_dtype == P3D_F32;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.N), static_cast<cuuint64_t>(p.M)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.ldo) * dtype_size(p.out_dtype)};
    cuuint32_t box[2] = {f32 ? 16u : 32u, 32};
    cuuint32_t es[2] = {1, 1};
    const CUtensorMapDataType dt = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : (p.out_dtype == P3D_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
    CUresult r = fn(map, dt, 2, p.out, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                    CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(ctx, P3D_ERR_CUDA, "cuTensorMapEncodeTiled (output) failed: " + std::to_string(r));
    return P3D_OK;
}

template <int BN>
int launch_tiles(p3d_ctx *ctx, I8Params p) {
    using C = TileCfg<BN>;
    CUtensorMap ta, tb, to;
    std::memset(&to, 0, sizeof(to));
    int rc = make_tmap_i8(ctx, &ta, p.x, p.M, p.K, p.ldx, kTileM);
    if (rc || (rc = make_tmap_i8(ctx, &tb, p.w, p.N, p.K, p.ldw, BN))) return rc;
    const int64_t es = static_cast<int64_t>(dtype_size(p.out_dtype));
    p.tma_out = reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.ldo * es % 16 == 0 && p.ldo >= p.N;
    if (p.tma_out && (rc = make_tmap_i8_out(ctx, &to, p))) return rc;
    p.wide_cols = ((reinterpret_cast<uintptr_t>(p.ws) | reinterpret_cast<uintptr_t>(p.bias)) & 15) == 0;
    P3D_CUDA(ctx, cudaFuncSetAttribute(linear_i8_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    const int64_t tiles = ceil_div(p.M, kTileM) * ceil_div(p.N, BN);
    const int ctas = static_cast<int>(std::min<int64_t>(tiles, ctx->num_sms));
    P3D_CUDA(ctx, launch_pdl(linear_i8_kernel<BN>, dim3(ctas), dim3(kThreadsT), C::SMEM, ctx->stream, ta, tb, to, p));
    return check_launch(ctx, "linear_i8");
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" int p3d_linear_i8(p3d_ctx *ctx, const int8_t *x, int64_t ldx, const float *x_scale, const int8_t *w,
                             int64_t ldw, const float *w_scale, const float *bias, int64_t m, int64_t n, int64_t k,
                             void *out, int64_t ldo, int out_dtype, int epilogue, const float *gate, int64_t gate_ld,
                             const int32_t *batch_offsets, int nbatch) {
    if (!ctx) return P3D_ERR_INVALID;
    P3D_REQUIRE(ctx, x && x_scale && w && w_scale && out, "p3d_linear_i8: null pointer");
    P3D_REQUIRE(ctx, m >= 0 && n > 0 && k > 0 && m < (int64_t(1) << 31) && n < (int64_t(1) << 31), "p3d_linear_i8: bad shape");
    if (k > 131071)
        return set_error(ctx, P3D_ERR_UNSUPPORTED, "p3d_linear_i8: k above 131071 could overflow the 32-bit sums");
    P3D_REQUIRE(ctx, ldx >= k && ldw >= k && ldx % 16 == 0 && ldw % 16 == 0,
                "p3d_linear_i8: ldx and ldw must be multiples of 16, at least k");
    P3D_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0,
                "p3d_linear_i8: x and w must be 16-byte aligned");
    P3D_REQUIRE(ctx, ldo >= n || m <= 1, "p3d_linear_i8: ldo < n");
    P3D_REQUIRE(ctx, out_dtype == P3D_F32 || is_16bit(out_dtype), "p3d_linear_i8: bad out_dtype");
    P3D_REQUIRE(ctx, reinterpret_cast<uintptr_t>(out) % dtype_size(out_dtype) == 0, "p3d_linear_i8: out not aligned to its elements");
    P3D_REQUIRE(ctx, (epilogue & ~(P3D_EPI_GELU_TANH | P3D_EPI_SILU | P3D_EPI_RESIDUAL)) == 0 &&
                         (epilogue & (P3D_EPI_GELU_TANH | P3D_EPI_SILU)) != (P3D_EPI_GELU_TANH | P3D_EPI_SILU),
                "p3d_linear_i8: at most one activation");
    P3D_REQUIRE(ctx, !(epilogue & P3D_EPI_RESIDUAL) || out_dtype == P3D_F32,
                "p3d_linear_i8: residual epilogue needs f32 out");
    P3D_REQUIRE(ctx, !gate || ((epilogue & P3D_EPI_RESIDUAL) && batch_offsets && nbatch > 0),
                "p3d_linear_i8: gate needs the residual epilogue and batch offsets");
    if (m == 0) return P3D_OK;
    DeviceGuard on(ctx->device);
    I8Params p{x, w, ldx, ldw, x_scale, w_scale, bias, out, ldo, gate, gate_ld, batch_offsets, nbatch,
               m, n, static_cast<int>(k), out_dtype, epilogue, ctx->fault, 0, 0};
    // Few outputs: the rows kernel runs about 1.5 us + m n k / 21e6 us (16e6
    // for short k; k at least 512, a warp's stride), the tiles 3.6 us + 0.0022
    // us k (their ring of TMA loads).  m x k x n, rows against tiles: 120 x 333
    // x 777 4.80 / 4.91 us, 200 x 100 x 600 5.74 / 4.08, 64 x 1024 x 1024 4.69 /
    // 5.58, 16 x 1024 x 6144 6.24 / 6.74, 32 x 4096 x 1024 7.7 / 12.5.
    const int64_t kk = std::max<int64_t>(k, 512);
    if (m * n * kk < std::min<int64_t>(111000 * kk - 21000000, 47000 * kk + 45000000)) {
        // Rows and channels a warp: as many as leave the GPU enough warps.  us
        // with the choice and with 1 x 1 / 4 x 2: 1 x 1024 x 6144 2.16 (2.54 /
        // 3.19), 2 x 1024 x 6144 2.33 (3.69 / 3.19), 2 x 4096 x 1024 3.04 (3.18
        // / 3.98), 4 x 1024 x 6144 2.77 (6.87 / 3.20), 4 x 4096 x 1024 3.31
        // (3.41 / 4.03), 16 x 4096 x 1024 4.69 (7.62 / the choice).
        const bool wide = n >= 4096;
        if (m == 2 && wide) return launch_rows<2, 4>(ctx, p);
        if (m > 2 && m <= 4 && wide) return launch_rows<4, 4>(ctx, p);
        if (m > 2 && ceil_div(n, 2) * ceil_div(m, 4) >= 1024) return launch_rows<4, 2>(ctx, p);
        return launch_rows<1, 2>(ctx, p);
    }
    // The tile width of the fewest waves, a 128- and a 64-column tile costing
    // 0.78 and 0.69 of a 256-column one (8184 x 4096 x 1024: 11.4, 10.1 and
    // 14.6 us a wave).
    const int64_t mt = ceil_div(m, kTileM);
    auto cost = [&](int bn, double tile) { return tile * static_cast<double>(ceil_div(mt * ceil_div(n, bn), ctx->num_sms)); };
    const double c64 = cost(64, 0.69), c128 = cost(128, 0.78), c256 = cost(256, 1.0);
    if (c64 < c128 && c64 < c256) return launch_tiles<64>(ctx, p);
    if (c128 < c256) return launch_tiles<128>(ctx, p);
    return launch_tiles<256>(ctx, p);
}
