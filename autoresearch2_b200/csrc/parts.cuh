// Products split over K: into how many parts, and their join.
#pragma once

#include <algorithm>

#include "fp8.cuh"

namespace sffn {

constexpr int P_PAIRS = 74;  // CTA pairs of a B200

inline long long tiles_of(long long M, long long N) { return (M + 255) / 256 * ((N + 255) / 256); }
inline long long part_ld(long long N) { return (N + 3) / 4 * 4; }

// A product of few 256 x 256 tiles leaves CTA pairs idle, so its k-blocks are dealt
// to more of them.  In us: rounds of tasks, each a part's blocks (`us` a block) and
// four more to fill the pipeline, and for parts their float32 traffic (written and
// read at the copy rate) and the second kernel (3 us).  Parts are whole multiples
// of `grain` blocks.
inline int split_of(long long M, long long N, long long nkb, int grain, double us) {
    const long long tiles = tiles_of(M, N), units = (nkb + grain - 1) / grain;
    double best = 0;
    int best_s = 1;
    for (int s = 1; s <= 32 && s <= units; ++s) {
        const long long per = (units + s - 1) / s;
        if ((units + per - 1) / per != s) continue;
        const long long rounds = (tiles * s + P_PAIRS - 1) / P_PAIRS;
        const double cost = (double)rounds * (double)(per * grain + 4) * us + (s > 1 ? 3.0 + 8.0 * (double)M * (double)N * s / 6.5e6 : 0);
        if (s == 1 || cost < best) best = cost, best_s = s;
    }
    return best_s;
}

namespace {

// C = the parts of a product split over K, added in their order.
template <int DT>
__global__ void __launch_bounds__(256)
    join_parts_kernel(const float* __restrict__ part, int splits, long long M, int N, long long ldp, uint16_t* __restrict__ out,
                      long long ldc, int vec) {
    const long long quads = ldp / 4, n = M * quads;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long row = i / quads;
        const int col = (int)(i - row * quads) * 4;
        const float4* p = reinterpret_cast<const float4*>(part + row * ldp + col);
        float4 s = __ldcs(p);
        for (int k = 1; k < splits; ++k) {
            const float4 v = __ldcs(p + k * (M * quads));
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
        uint16_t* o = out + row * ldc + col;
        const uint2 w = make_uint2(pack16x2<DT>(s.x, s.y), pack16x2<DT>(s.z, s.w));
        if (vec && col + 4 <= N) {
            *reinterpret_cast<uint2*>(o) = w;
        } else {
            if (col < N) o[0] = (uint16_t)w.x;
            if (col + 1 < N) o[1] = (uint16_t)(w.x >> 16);
            if (col + 2 < N) o[2] = (uint16_t)w.y;
            if (col + 3 < N) o[3] = (uint16_t)(w.y >> 16);
        }
    }
}

// part: [splits][M][part_ld(N)] -> out [M][ldc]
template <int DT>
int join_parts(const float* part, int splits, long long M, int N, void* out, long long ldc, cudaStream_t st) {
    const long long ldp = part_ld(N), quads = M * (ldp / 4);
    const int grid = (int)std::min<long long>((quads + 255) / 256, 148 * 8);
    const int vec = reinterpret_cast<uintptr_t>(out) % 8 == 0 && ldc % 4 == 0;
    join_parts_kernel<DT><<<grid, 256, 0, st>>>(part, splits, M, N, ldp, static_cast<uint16_t*>(out), ldc, vec);
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

}  // namespace
}  // namespace sffn
