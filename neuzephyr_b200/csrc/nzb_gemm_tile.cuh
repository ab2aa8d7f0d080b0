// Operand tiles of the fp16 tensor-core kernels: tensor maps, TMA loads of one k block and the bits of the
// shared-memory descriptors, for K-major and MN-major operand copies.
#pragma once
#include <cuda_fp16.h>

#include "nzb_internal.h"
#include "nzb_ptx.cuh"

namespace nzb {

// Operand tile loads for one k block. K-major: one box of `rows` x 64 k. MN-major: rows/64
// boxes of 64 (m or n) x 64 k, 8192 bytes apart, which is the layout the MN-major
// descriptor below walks (leading byte offset 8192, 1024 bytes per 8-k group).
template <int ROWS>
__device__ __forceinline__ void load_operand(uint8_t* dst, const CUtensorMap* tm, int32_t mn, int32_t k0, int32_t row0,
                                             int32_t z, uint64_t* bar) {
    using namespace ptx;
    if (mn) {
#pragma unroll
        for (int j = 0; j < ROWS / 64; j++) tma_load_3d(dst + j * 8192, tm, row0 + j * 64, k0, z, bar);
    } else {
        tma_load_3d(dst, tm, k0, row0, z, bar);
    }
}
template <int ROWS>
__device__ __forceinline__ void load_operand_pair(uint8_t* dst, const CUtensorMap* tm, int32_t mn, int32_t k0,
                                                  int32_t row0, int32_t z, uint32_t leader_bar) {
    using namespace ptx;
    if (mn) {
#pragma unroll
        for (int j = 0; j < ROWS / 64; j++) tma_load_3d_pair(dst + j * 8192, tm, row0 + j * 64, k0, z, leader_bar);
    } else {
        tma_load_3d_pair(dst, tm, k0, row0, z, leader_bar);
    }
}

// Descriptor bits above the start address for a SWIZZLE_128B operand tile.
//   K-major: rows of 128 bytes, 8-row groups 1024 bytes apart (leading offset unused: 1).
//   MN-major: 64-element blocks 8192 bytes apart (leading), 8-k groups 1024 bytes apart (stride).
__device__ __forceinline__ uint64_t desc_high_bits(int32_t mn) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>(mn ? (8192 >> 4) : 1) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// Descriptor address units (16 bytes) per 16-wide k step: 32 bytes along a K-major row,
// 16 rows of 128 bytes in an MN-major tile.
__device__ __forceinline__ uint32_t desc_kstep(int32_t mn) { return mn ? 128u : 2u; }

static inline int make_operand_map(CUtensorMap* map, const __half* base, int64_t K, int64_t Kp, int64_t rows, int64_t nmat,
                            int box_rows) {
    EncodeTiledFn enc;
    int rc = get_encode_tiled(&enc);
    if (rc != NZB_OK) return rc;
    cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)rows, (cuuint64_t)nmat};
    cuuint64_t strides[2] = {(cuuint64_t)Kp * 2, (cuuint64_t)rows * (cuuint64_t)Kp * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NZB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return NZB_OK;
}

// MN-major operand copy [nmat][K][ld]: dimension 0 runs along m (or n), boxes are 64 x 64.
static inline int make_operand_map_mn(CUtensorMap* map, const __half* base, int64_t K, int64_t extent, int64_t ld,
                               int64_t nmat) {
    EncodeTiledFn enc;
    int rc = get_encode_tiled(&enc);
    if (rc != NZB_OK) return rc;
    cuuint64_t dims[3] = {(cuuint64_t)extent, (cuuint64_t)K, (cuuint64_t)nmat};
    cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)K * (cuuint64_t)ld * 2};
    cuuint32_t box[3] = {64, 64, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(NZB_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
    return NZB_OK;
}

}  // namespace nzb
