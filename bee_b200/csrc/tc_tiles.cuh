// What the tensor-core products share: the order in which a persistent grid
// visits output tiles, and TMA maps of 16-bit matrices.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "common.cuh"

namespace bee_b200 {

constexpr int kGroupM = 16;

__device__ __forceinline__ void grouped_tile(int t, int m_tiles, int n_tiles, int& mb, int& nb) {
    const int per_group = kGroupM * n_tiles;
    const int group = t / per_group;
    const int first_m = group * kGroupM;
    const int gsize = min(m_tiles - first_m, kGroupM);
    const int r = t - group * per_group;
    mb = first_m + r % gsize;
    nb = r / gsize;
}

// K order of a persistent CTA's i-th tile: forward for even i, backward for odd
// i.  The CTAs move through their tiles together, so the tiles of one wave
// start on the K blocks the previous wave (which shares their A panels under
// the grouped raster) read last, while those are still in L2.  The MMA side
// accumulates in iteration order whatever the coordinate.
__device__ __forceinline__ int k_block(int kb, int i, int num_kb) { return (i & 1) ? num_kb - 1 - kb : kb; }

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

// 3-D tensor map of 16-bit elements (bf16, or f16 when `f16`) {inner, outer,
// batch} with 128-byte swizzle.
inline int make_map(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t outer, uint64_t batch,
                    uint64_t row_stride, uint64_t batch_stride, uint32_t box_inner, uint32_t box_outer,
                    bool f16 = false) {
    auto enc = encode_fn();
    if (!enc) return fail(cudaErrorNotSupported, "cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[3] = {inner, outer, batch};
    cuuint64_t strides[2] = {row_stride * 2, batch_stride * 2};
    cuuint32_t box[3] = {box_inner, box_outer, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                     const_cast<void*>(ptr), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(cudaErrorInvalidValue, "tensor map encoding failed (CUresult %d)", int(r));
    return 0;
}

}  // namespace bee_b200
