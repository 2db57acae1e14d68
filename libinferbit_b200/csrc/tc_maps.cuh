// Tensor maps for the kernels that load tiles with TMA: the driver's encoder, and the two-dimensional byte matrices they use.
#pragma once
#include "common.cuh"
#include <cudaTypedefs.h>

using TensorMapEncodeFn = PFN_cuTensorMapEncodeTiled_v12000;
// NULL where the driver has none
inline TensorMapEncodeFn tensor_map_encoder() {
    static TensorMapEncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) { cudaGetLastError(); f = nullptr; }
        return (TensorMapEncodeFn)f;
    }();
    return fn;
}
// rows x cols bytes, rows `pitch` bytes apart, in boxes of box_rows x 128 bytes with the 128-byte swizzle; what lies outside reads as zeros
inline bool tensor_map_bytes(CUtensorMap* map, const void* base, long rows, long cols, long pitch, int box_rows) {
    const cuuint64_t dims[2] = { (cuuint64_t)cols, (cuuint64_t)rows }, strides[1] = { (cuuint64_t)pitch };
    const cuuint32_t box[2] = { 128, (cuuint32_t)box_rows }, es[2] = { 1, 1 };
    return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// into this block's shared memory, the bytes reported to a barrier of either block of a pair
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
