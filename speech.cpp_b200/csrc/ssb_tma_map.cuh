// Tensor maps over the pages of a key-value cache, and the TMA loads that use them (no multicast).
#pragma once

#include <cfloat>
#include <cmath>

#include <cuda.h>
#include <cudaTypedefs.h>

#include "ssb_kernels.h"
#include "ssb_tma.cuh"

namespace ssb {
namespace {

__device__ __forceinline__ void tma_load_5d(void * dst, const CUtensorMap * map, int x, int slot, int half, int head, int page,
                                            uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(slot), "r"(half), "r"(head), "r"(page), "r"(smem_addr(bar))
        : "memory");
}

template <typename Fn> inline Fn driver_function(const char * name) {
    void * p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint(name, &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<Fn>(p);
}

// The maps of the keys' and the values' pool as [page][head][column block][slot][128 bytes]: a copy brings `slots` positions of one head, `blocks`
// column blocks (64 bf16 or 32 fp32 elements) one after the other, each position's 128 bytes swizzled by its
// row's low three bits. Its innermost coordinate is always 0, so every copy starts on a 16-byte boundary where the
// base and the strides are multiples of 16.
inline bool page_maps(CUtensorMap * maps, const KvArgs & kv, int dim, int slots, int blocks, int element_bytes) {
    static const auto encode = driver_function<PFN_cuTensorMapEncodeTiled_v12000>("cuTensorMapEncodeTiled");
    static const auto readdress = driver_function<PFN_cuTensorMapReplaceAddress_v12000>("cuTensorMapReplaceAddress");
    if (!encode || !readdress) return false;
    const cuuint64_t es = (cuuint64_t) element_bytes, width = 128 / es;
    // the strides of axes of one entry are never used, but have to be valid
    const cuuint64_t head_stride = kv.kv_heads > 1 ? (cuuint64_t) kv.head_stride * es : 16;
    const cuuint64_t page_stride = kv.pages > 1 ? (cuuint64_t) kv.page_stride * es : 16;
    const cuuint64_t dims[5] = {width, (cuuint64_t) kv.page_size, (cuuint64_t) dim / width, (cuuint64_t) kv.kv_heads, (cuuint64_t) kv.pages};
    const cuuint64_t strides[4] = {(cuuint64_t) kv.position_stride * es, 128, head_stride, page_stride};
    const cuuint32_t box[5] = {(cuuint32_t) width, (cuuint32_t) slots, (cuuint32_t) blocks, 1, 1};
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    if (encode(&maps[0], element_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 5, kv.k, dims, strides,
               box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    maps[1] = maps[0];
    return readdress(&maps[1], kv.v) == CUDA_SUCCESS;
}

// Whether TMA can read this cache and the kernels that use it these rows. They hide a position by a score of -inf before the scale,
// which has to stay -inf: a scale next to 0, or 0, is the general kernel's.
inline bool tma_takes(const AttendArgs & a, int element_bytes) {
    const KvArgs & kv = a.kv;
    constexpr int64_t kMaxStride = (int64_t) 1 << 37;  // elements: tensor maps take strides below 2^40 bytes
    const int es = element_bytes, unit = 16 / es;
    return (kv.head_dim == 64 || kv.head_dim == 128) && a.vec_q && kv.pages > 0 && std::fabs(a.scale_log2) >= FLT_MIN &&
           (reinterpret_cast<uintptr_t>(kv.k) | reinterpret_cast<uintptr_t>(kv.v)) % 16 == 0 && kv.position_stride % unit == 0 &&
           (kv.kv_heads == 1 || kv.head_stride % unit == 0) && (kv.pages == 1 || (kv.page_stride > 0 && kv.page_stride % unit == 0)) &&
           kv.position_stride < kMaxStride && kv.head_stride < kMaxStride && kv.page_stride < kMaxStride;
}

}  // namespace
}  // namespace ssb
