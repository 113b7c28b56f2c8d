// Output side shared by the tcgen05 GEMM kernels: warp-uniform waits, rows
// staged in shared memory and written as TMA boxes, and the tensor maps.
#pragma once

#include "p3d_common.cuh"

namespace p3d {

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, or null where the driver lacks it.
EncodeFn get_encode_fn();
// Output map of the TMA epilogue (defined with the 16-bit operand maps).
int make_tmap_out(p3d_ctx *ctx, CUtensorMap *map, void *base, int dtype, uint64_t rows, uint64_t cols, uint64_t ld);

// One staging slot: a 32-row x 128-byte box (32 f32 or 64 16-bit columns) in
// the 128-byte swizzle.
constexpr int EPI_SLOT_BYTES = 4096;

template <typename T>
__device__ __forceinline__ void store16(T *o, const float (&v)[32], int ncols) {
    if (ncols == 32 && ((reinterpret_cast<uintptr_t>(o) & 15) == 0)) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            uint4 pk;
            pk.x = pack2<T>(v[i], v[i + 1]);
            pk.y = pack2<T>(v[i + 2], v[i + 3]);
            pk.z = pack2<T>(v[i + 4], v[i + 5]);
            pk.w = pack2<T>(v[i + 6], v[i + 7]);
            *reinterpret_cast<uint4 *>(o + i) = pk;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < ncols) o[i] = from_f32<T>(v[i]);
    }
}

// Staging slot for the next box: wait until the box last issued from this
// slot (two boxes ago) has been read by the TMA unit.
template <int SLOTS>
__device__ __forceinline__ uint8_t *acquire_slot(uint8_t *wbuf, int slot, int lane) {
    if (lane == 0) bulk_wait_read<SLOTS - 1>();
    __syncwarp();
    return wbuf + slot * EPI_SLOT_BYTES;
}

// This lane's 32 values as row `lane` of the slot, in the 128-byte swizzle
// (16-byte chunk c of a 128-byte row at c ^ (row & 7)).  f32: the whole
// 128-byte row; 16-bit: half `half` (columns 32*half .. +31) of a 64-column row.
__device__ __forceinline__ void stage_row(int out_dtype, uint8_t *buf, int lane, const float (&v)[32], int half) {
    uint8_t *rowp = buf + lane * 128;
    if (out_dtype == P3D_F32) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
            *reinterpret_cast<float4 *>(rowp + ((c ^ (lane & 7)) << 4)) =
                make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
        return;
    }
    const bool bf = out_dtype == P3D_BF16;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint4 pk;
        pk.x = bf ? pack2<__nv_bfloat16>(v[8 * c], v[8 * c + 1]) : pack2<__half>(v[8 * c], v[8 * c + 1]);
        pk.y = bf ? pack2<__nv_bfloat16>(v[8 * c + 2], v[8 * c + 3]) : pack2<__half>(v[8 * c + 2], v[8 * c + 3]);
        pk.z = bf ? pack2<__nv_bfloat16>(v[8 * c + 4], v[8 * c + 5]) : pack2<__half>(v[8 * c + 4], v[8 * c + 5]);
        pk.w = bf ? pack2<__nv_bfloat16>(v[8 * c + 6], v[8 * c + 7]) : pack2<__half>(v[8 * c + 6], v[8 * c + 7]);
        *reinterpret_cast<uint4 *>(rowp + (((4 * half + c) ^ (lane & 7)) << 4)) = pk;
    }
}

// Lane 0 writes the staged 32-row box at (col0, row0): a TMA store, or (the
// residual epilogue, or part of a tile cut by the split schedule) a TMA
// reduce-add into the f32 output.  Rows >= M and columns >= N of the box are
// clipped by the tensor map's bounds.
template <int SLOTS>
__device__ __forceinline__ void issue_box(const CUtensorMap *tmo, const uint8_t *buf, int lane, int64_t col0,
                                          int64_t row0, int &slot, bool reduce) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
        if (reduce)
            tma_reduce_add_2d(tmo, buf, static_cast<int>(col0), static_cast<int>(row0));
        else
            tma_store_2d(tmo, buf, static_cast<int>(col0), static_cast<int>(row0));
        bulk_commit();
    }
    slot = SLOTS == 1 ? 0 : slot ^ 1;
}

// Warp-uniform bounded wait: lane 0 polls, the warp follows its verdict.
template <bool CLUSTER>
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int *fault) {
    int ok = 1;
    if ((threadIdx.x & 31) == 0)
        ok = (CLUSTER ? mbar_wait_cluster(bar, parity, fault) : mbar_wait(bar, parity, fault)) ? 1 : 0;
    return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

}  // namespace p3d
