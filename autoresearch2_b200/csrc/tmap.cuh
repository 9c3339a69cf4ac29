// Host side of the tensor-core kernels of glu.cu and fp8mm.cu: tensor maps,
// resident clusters, the raster of their tiles.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <stdio.h>

#include <atomic>

#include "common.cuh"

namespace sffn {

constexpr int P_GROUP_M = 8;  // pair-tile rows per raster group

// Tiles in groups of P_GROUP_M rows of tiles, so that the clusters running at
// once share operand tiles in L2.
__device__ __forceinline__ void pair_raster(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int per_group = P_GROUP_M * tiles_n;
    const int group = tile / per_group;
    const int first_m = group * P_GROUP_M;
    const int gsize = min(tiles_m - first_m, P_GROUP_M);
    const int r = tile - group * per_group;
    tm = first_m + r % gsize;
    tn = r / gsize;
}

inline PFN_cuTensorMapEncodeTiled_v12000 tmap_encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void* p = nullptr;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
        return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p)
                                                                    : nullptr;
    }();
    return fn;
}

// `inner` contiguous elements a row, `outer` rows `ld` elements apart.
inline int tmap_2d(CUtensorMap* m, CUtensorMapDataType type, int esize, const void* base, long long inner, long long outer,
                   long long ld, int box_inner, int box_outer, CUtensorMapSwizzle swizzle) {
    const auto fn = tmap_encoder();
    if (!fn) {
        set_error_text("cuTensorMapEncodeTiled entry point not found");
        return SFFN_ERR_CUDA;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    const cuuint64_t strides[1] = {(cuuint64_t)(ld * esize)};
    const cuuint32_t box[2] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(m, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        char msg[200];
        snprintf(msg, sizeof(msg), "cuTensorMapEncodeTiled -> %d (base %p dims %lld x %lld ld %lld box %d x %d)", (int)r,
                 base, inner, outer, ld, box_inner, box_outer);
        set_error_text(msg);
        return SFFN_ERR_CUDA;
    }
    return SFFN_OK;
}

// Scale tiles [tiles][32 * bt] rows of 16 bytes; boxes of one block tile's 32 rows
// in `count` row tiles (zeros past the last one, whose values are zero too).
inline int scale_map(CUtensorMap* m, const void* p, long long tiles, long long bt, int count) {
    const auto fn = tmap_encoder();
    const cuuint64_t dims[3] = {4, (cuuint64_t)(bt * 32), (cuuint64_t)tiles};
    const cuuint64_t strides[2] = {16, (cuuint64_t)(bt * 512)};
    const cuuint32_t box[3] = {4, 32, (cuuint32_t)count}, estr[3] = {1, 1, 1};
    if (!fn || fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(p), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
        set_error_text("cuTensorMapEncodeTiled failed for the scale tiles");
        return SFFN_ERR_CUDA;
    }
    return SFFN_OK;
}

// The current device's multiprocessors; 0 unless it is sm_100.  Asked of the
// driver once a device.
inline int sm100_sms() {
    static std::atomic<int> known[64];  // sms + 1, 0: not asked yet
    int dev = 0, major = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev < 64)
        if (const int k = known[dev].load(std::memory_order_relaxed)) return k - 1;
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    if (major != 10) sms = 0;
    if (dev < 64) known[dev].store(sms + 1, std::memory_order_relaxed);
    return sms;
}

// A kernel's shared-memory limit, raised once a device.
struct SmemOnce {
    std::atomic<uint64_t> done{0};
    template <typename K>
    cudaError_t set(K kernel, int smem) {
        int dev = 0;
        if (const cudaError_t e = cudaGetDevice(&dev)) return e;
        const uint64_t bit = dev < 64 ? 1ull << dev : 0;
        if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
        return e;
    }
};

// Clusters of `size` CTAs of this kernel that are resident at once (one CTA fills an SM).
template <typename K>
int resident_clusters(K kernel, int threads, int smem, int size) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)size * 128);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)size;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, (void*)kernel, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = sm100_sms() / size;
    }
    return n > 0 ? n : 1;
}
template <typename K>
int resident_pairs(K kernel, int threads, int smem) {
    return resident_clusters(kernel, threads, smem, 2);
}

}  // namespace sffn
