// Epilogue output of the tensor-core kernels through shared memory: a warp's 32
// rows x 32 columns of 16-bit values (lane = row, 16 packed words).
#pragma once

#include "sm100.cuh"

namespace sffn {

// Into a 2 KB buffer, in the layout of a tensor map with 64-byte swizzle
// (16-byte chunk ch of row r at r * 64 + 16 * (ch ^ ((r >> 1) & 3))).
// 16 of the 32 columns:
__device__ __forceinline__ void stage16(unsigned char* sbuf, int lane, int half, const uint32_t* w) {
    const uint32_t rb = smem_u32(sbuf) + (uint32_t)lane * 64u;
    const int sw = (lane >> 1) & 3;
#pragma unroll
    for (int ch = 0; ch < 2; ++ch)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(rb + 16u * (uint32_t)((2 * half + ch) ^ sw)), "r"(w[4 * ch]),
                     "r"(w[4 * ch + 1]), "r"(w[4 * ch + 2]), "r"(w[4 * ch + 3])
                     : "memory");
}
__device__ __forceinline__ void stage32(unsigned char* sbuf, int lane, const uint32_t (&w)[16]) {
    stage16(sbuf, lane, 0, w);
    stage16(sbuf, lane, 1, w + 8);
}

// A warp's R staging buffers, used in turn: each store is a bulk group of its own,
// and a buffer is written again once the store that used it has read it, with
// the R - 1 later ones still under way.  (Waiting for the last store each time
// made the epilogue, not the products, the bound of a 768-wide K.)
template <int R>
struct StageRing {
    unsigned char* base;
    int at = 0;
    __device__ __forceinline__ explicit StageRing(unsigned char* p) : base(p) {}

    // The block by one bulk-tensor store (whole 64-byte row segments; clipped at the
    // tensor's edges).
    __device__ __forceinline__ void store(const CUtensorMap* tmap, int lane, const uint32_t (&w)[16], int col, int row0) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(R - 1) : "memory");
        __syncwarp();
        unsigned char* sbuf = base + at * 2048;
        at = at + 1 == R ? 0 : at + 1;
        stage32(sbuf, lane, w);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(tmap, sbuf, col, row0);
            bulk_commit_group();
        }
    }
};

// The same where the rows' stride or start suit no tensor map: lane = column,
// row by row.  (A lane writing its own row, 2 bytes of 32 rows an instruction,
// took 45 us for a 1023 x 1777 result.)
__device__ __forceinline__ void stage_store_plain(uint16_t* out, long long ld, int rows, int cols, unsigned char* sbuf, int lane,
                                                  const uint32_t (&w)[16], int col, int row0) {
    __syncwarp();
    stage32(sbuf, lane, w);
    __syncwarp();
    const uint32_t sb = smem_u32(sbuf) + 2u * (uint32_t)(lane & 7);
    const int ch = lane >> 3;
    uint16_t* p = out + (long long)row0 * ld + col + lane;
    const int n = min(32, rows - row0);
    if (col + lane < cols) {
#pragma unroll 8
        for (int r = 0; r < n; ++r) {
            uint16_t h;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(sb + (uint32_t)(r * 64 + 16 * (ch ^ ((r >> 1) & 3)))));
            p[r * ld] = h;
        }
    }
}

}  // namespace sffn
