// Products of up to 64 rows with long weights on the tcgen05 tensor cores:
// out[T, N] = x[T, K] W[N, K]^T in 16 bits or in the 8-bit block format, and the
// gated pair act(x Wg^T) * (x Wu^T).
//
// Bound by reading the weights once.  W's rows are the M of tcgen05.mma (128) and
// the tokens its N (48 or 64, those past the last hold anything), so that 8-bit operands
// need no conversion and tokens cost next to nothing.  A CTA takes a tile of 128
// rows of W (of Wg and of Wu); where tiles are few a cluster of up to 8 CTAs shares
// one, each a part of K, and every CTA adds the parts of its share of the tokens, in
// order, from its shared memory.  17 rows through 4096 x 14336 and back, bfloat16:
// 70 us, 5.1 TB/s, 64 rows 73 (256-row tiles: 87 and 91); 17 x 14336 x 4096 in 8 bits 18.1 us (20.2).
// What is left: 16 KB of W take a CTA 0.33 us, 50 GB/s, whatever K's place or the
// number of tokens (more stages, more issuers, separate sums for the products, and
// tiles of fewer rows on more CTAs made no difference; the tensor pipe is active 10
// to 16%), and tiles rarely deal out evenly over the multiprocessors.
//   warps 0-2 or 0-3  TMA issuers of W: a third of the k-blocks each, or half of Wg's or of Wu's
//   next 3 or 2       TMA issuers of x
//   next warp         tensor memory, scales (tcgen05.cp) and MMA issuer
//   warps 8-15        epilogue, thread = row of W, two a row for alternate 16 tokens
#include <cuda.h>
#include <string.h>

#include <algorithm>

#include "act.cuh"
#include "fp8.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace sffn {
namespace {

constexpr int R_THREADS = 512, R_EPI = 8;  // first epilogue warp
constexpr int R_W = 128 * 128;  // bytes of a stage's tile of one W

// NT: the tokens of a product, tcgen05.mma's N, 48 or 64.
template <bool FP8, int MATS, int NT>
struct Narrow {
    static constexpr int STAGES = MATS == 2 ? 4 : 6;
    static constexpr int ISSUERS = STAGES / 2;     // of each matrix: a stage belongs to one
    static constexpr int STAGE = MATS * R_W + NT * 128;
    static constexpr int SCALES = FP8 ? 1024 : 0;  // W's tile, x's
    // token rows for the parts of K: those of 8 more, where they fit, take any deal
    static constexpr int PLACES = MATS == 2 && NT == 64 ? 64 : NT + 8;
    static constexpr int PARTS = PLACES * MATS * 512;
    static constexpr int SMEM = STAGES * (STAGE + SCALES) + PARTS + 1024;
    static constexpr int ACC = MATS * NT;          // tensor memory columns, twice
    static constexpr int SCALE_COL = 2 * ACC;      // 8 columns a group of four k-blocks
    static_assert(SMEM <= 232448 - 1024 && SCALE_COL + (FP8 ? 8 * STAGES : 0) <= 512 && NT % 16 == 0, "");
};

struct NarrowArgs {
    int T, N;
    int tiles, nkb, per;  // tiles of 128 rows; k-blocks of 128 bytes, of a part (a multiple of 4 in 8 bits)
    uint16_t* out;
    long long ldo;
    uint32_t* status;
};

template <int DT>
__device__ constexpr uint32_t idesc_narrow(bool fp8, int n) {  // K-major operands, M = 128
    const uint32_t f = DT == SFFN_BF16 ? 1u : 0u;
    return ((uint32_t)(n >> 3) << 17) | (8u << 24) | (fp8 ? 1u << 23 : (1u << 4) | (f << 7) | (f << 10));
}
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void cp_scales(uint32_t taddr, uint64_t sdesc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

template <bool FP8, int DT, int MATS, int ACT, int NT>
__global__ void __launch_bounds__(R_THREADS, 1)
    narrow_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmW2,
                  const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmSW,
                  const __grid_constant__ CUtensorMap tmSX, const NarrowArgs args) {
    using C = Narrow<FP8, MATS, NT>;
    constexpr uint32_t IDESC = idesc_narrow<DT>(FP8, NT);
    constexpr int BK = FP8 ? 128 : 64;
    extern __shared__ __align__(1024) unsigned char narrow_smem[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(narrow_smem) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char* sscales = smem + C::STAGES * C::STAGE;
    float* parts = reinterpret_cast<float*>(sscales + C::STAGES * C::SCALES);  // [source][token][matrix][128]
    __shared__ __align__(8) uint64_t full_bar[C::STAGES], empty_bar[C::STAGES];
    __shared__ __align__(8) uint64_t tfull_bar[2], tempty_bar[2];
    __shared__ __align__(8) uint64_t came_bar, free_bar;  // the cluster's parts are in this CTA; this CTA's are read everywhere
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), size = cluster_size();
    const int first = (int)(blockIdx.x / size), stride = (int)(gridDim.x / size);
    const int kb0 = (int)rank * args.per, kb1 = min(args.nkb, kb0 + args.per);
    // Groups of four k-blocks, each cluster from another one on, so that they do not
    // all read the same part of x at once.
    const int groups = (kb1 - kb0 + 3) / 4, turn0 = (int)((long long)first * groups / stride);
    auto each_block = [&](auto&& f) {  // f(kb, first one); false: given up
        for (int i = 0; i < groups; ++i) {
            const int g = i + turn0 < groups ? i + turn0 : i + turn0 - groups;
            for (int kb = kb0 + 4 * g; kb < min(kb1, kb0 + 4 * g + 4); ++kb)
                if (!f(kb, i == 0 && kb == kb0 + 4 * g)) return false;
        }
        return true;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull_bar[a], 1);
            mbar_init(&tempty_bar[a], 8);
        }
        mbar_init(&came_bar, 8 * size);
        mbar_init(&free_bar, 8 * size);
        s_abort = 0;
        fence_mbar_init();
        prefetch_tmap(&tmW);
        prefetch_tmap(&tmX);
        if constexpr (MATS == 2) prefetch_tmap(&tmW2);
    }
    constexpr int X_WARP = C::ISSUERS * MATS, MMA_WARP = X_WARP + C::ISSUERS;
    __syncthreads();
    // The copies need no more; tensor memory and the cluster's other CTAs are waited
    // for where they are used.
    if (size > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    grid_dependents_start();

    if (warp < MMA_WARP) {
        // ------------------------------------------------------ producers --
        if (lane == 0) {
            const bool loads_x = warp >= X_WARP;
            const int mat = warp / C::ISSUERS, turn = warp % C::ISSUERS;
            if (loads_x) grid_dependency_wait();  // the kernel before may be writing x
            int armed[C::STAGES] = {0};
            int kc = 0, sgroup = -1;
            for (int tile = first; tile < args.tiles && !s_abort; tile += stride) {
                const bool whole = each_block([&](int kb, bool) {
                    const bool scales = FP8 && (kb & 3) == 0;
                    if (scales) sgroup = sgroup + 1 == C::STAGES ? 0 : sgroup + 1;
                    const int at = kc++, stage = at % C::STAGES;
                    if (at % C::ISSUERS != turn) return true;
                    if (!mbar_wait_bounded(&empty_bar[stage], (uint32_t)(at / C::STAGES & 1) ^ 1u)) {
                        atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                        s_abort = 1;
                        return false;
                    }
                    unsigned char* to = smem + stage * C::STAGE;
                    // Scale slots are as many as stages and a group has a k-block at least:
                    // the slot's last group lies a whole ring back.
                    unsigned char* ss = sscales + sgroup * C::SCALES;
                    if (loads_x) {
                        tma_load_2d(to + MATS * R_W, &tmX, kb * BK, 0, &full_bar[stage]);
                        if (scales) tma_load_2d(ss + 512, &tmSX, 0, (kb >> 2) * 32, &full_bar[stage]);
                    } else {
                        if (mat == 0) {
                            mbar_arrive_expect_tx(&full_bar[stage], (uint32_t)(MATS * R_W + args.T * 128 + (scales ? 1024 : 0)));
                            ++armed[stage];
                        }
                        tma_load_2d(to + mat * R_W, mat ? &tmW2 : &tmW, kb * BK, tile * 128, &full_bar[stage]);
                        if (scales) tma_load_3d(ss, &tmSW, 0, (kb >> 2) * 32, tile, &full_bar[stage]);
                    }
                    return true;
                });
                if (!whole) break;
            }
            // once the last phases armed here complete, no copy is still landing
            for (int s = 0; s < C::STAGES; ++s)
                if (armed[s]) (void)mbar_wait_bounded(&full_bar[s], (uint32_t)(armed[s] - 1) & 1u);
        }
        __syncwarp();
    } else if (warp == MMA_WARP) {
        // ----------------------------------------------------------- MMA --
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
        tc_fence_before();
        named_bar_sync(1, 9 * 32);
        tc_fence_after();
        const uint32_t tmem_base = s_tmem;
        if (lane == 0) {
            int stage = 0, acc = 0, sgroup = -1;
            uint32_t phase = 0, acc_phase = 0;
            for (int tile = first; tile < args.tiles && !s_abort; tile += stride) {
                bool fail = !mbar_wait_bounded(&tempty_bar[acc], acc_phase ^ 1u);
                tc_fence_after();
                const uint32_t d = tmem_base + (uint32_t)(acc * C::ACC);
                fail = fail || !each_block([&](int kb, bool start) {
                    if (!mbar_wait_bounded(&full_bar[stage], phase)) return false;
                    const uint32_t sw = smem_u32(smem + stage * C::STAGE), sx = sw + MATS * R_W;
                    if constexpr (FP8) {
                        if ((kb & 3) == 0) sgroup = sgroup + 1 == C::STAGES ? 0 : sgroup + 1;
                        const uint32_t ta = tmem_base + C::SCALE_COL + 8u * (uint32_t)sgroup, id = (uint32_t)kb & 3u;
                        if ((kb & 3) == 0) {
                            const uint32_t ss = smem_u32(sscales + sgroup * C::SCALES);
                            cp_scales(ta, smem_desc_rows16(ss));
                            cp_scales(ta + 4, smem_desc_rows16(ss + 512));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mma_mx(d, umma_desc_sw128(sw + 32 * j, 16, 1024), umma_desc_sw128(sx + 32 * j, 16, 1024),
                                   IDESC | (id << 4) | (id << 29), ta, ta + 4, !start || j ? 1u : 0u);
                    } else {
#pragma unroll
                        for (int m = 0; m < MATS; ++m)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                tc_mma_f16(d + m * NT, umma_desc_sw128(sw + m * R_W + 32 * j, 16, 1024),
                                           umma_desc_sw128(sx + 32 * j, 16, 1024), IDESC, !start || j ? 1u : 0u);
                    }
                    tc_commit(&empty_bar[stage]);
                    if (++stage == C::STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    return true;
                });
                if (fail) {
                    atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                    s_abort = 1;
                    break;
                }
                tc_commit(&tfull_bar[acc]);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp >= R_EPI) {
        // ------------------------------------------------------ epilogue --
        named_bar_sync(1, 9 * 32);
        tc_fence_after();
        const uint32_t tmem_base = s_tmem;
        if (size > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        grid_dependency_wait();
        const int ew = warp & 3, place = ew * 32 + lane, half = (warp - R_EPI) >> 2;
        // tokens are dealt to the cluster's CTAs in runs of `share`
        const int share = (args.T + (int)size - 1) / (int)size;
        const int mine = (int)rank * share, n = min(share, args.T - mine);
        int acc = 0;
        uint32_t acc_phase = 0, came = 0, read = 1;
        auto result = [&](const float (&v)[MATS]) {
            if constexpr (MATS == 2) return Elt<DT>::from_f(glu_act<ACT>(v[0]) * v[1]);
            else return Elt<DT>::from_f(v[0]);
        };
        for (int tile = first; tile < args.tiles; tile += stride) {
            const long long row = (long long)tile * 128 + place;
            const bool live = row < args.N;
            uint16_t* out = args.out + row;
            bool ok = __all_sync(FULL, mbar_wait_bounded(&tfull_bar[acc], acc_phase));
            if (ok && size > 1) ok = __all_sync(FULL, mbar_wait_bounded<true>(&free_bar, read));
            if (!ok && lane == 0) atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
            if (!ok || __any_sync(FULL, s_abort != 0)) break;
            read ^= 1u;
            tc_fence_after();
            const uint32_t t0 = tmem_base + ((uint32_t)(ew * 32) << 16) + (uint32_t)(acc * C::ACC);
#pragma unroll 1
            for (int t = half * 16; t < args.T; t += 32) {
                uint32_t r[MATS][16];
#pragma unroll
                for (int m = 0; m < MATS; ++m) tmem_ld16(t0 + m * NT + t, r[m]);
                tmem_wait_ld();
                if (size == 1) {
                    uint16_t* o = out + t * args.ldo;
#pragma unroll
                    for (int j = 0; j < 16; ++j, o += args.ldo) {
                        float v[MATS];
#pragma unroll
                        for (int m = 0; m < MATS; ++m) v[m] = __uint_as_float(r[m][j]);
                        if (t + j < args.T && live) *o = result(v);
                    }
                } else {
                    int owner = t / share, at = t - owner * share;
                    const uint32_t here = smem_u32(parts) + (((uint32_t)rank * share * MATS) * 128 + place) * 4;
                    uint32_t to = cluster_addr(here, (uint32_t)owner) + at * (MATS * 512);
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (t + j < args.T) {
#pragma unroll
                            for (int m = 0; m < MATS; ++m) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + m * 512), "r"(r[m][j]) : "memory");
                            to += MATS * 512;
                            if (++at == share) at = 0, ++owner, to = cluster_addr(here, (uint32_t)min(owner, (int)size - 1));
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty_bar[acc]);
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
            if (size > 1) {
                asm volatile("fence.acq_rel.cluster;" ::: "memory");
                __syncwarp();
                if (lane < (int)size) mbar_arrive_cluster(cluster_addr(smem_u32(&came_bar), (uint32_t)lane));
                if (!__all_sync(FULL, mbar_wait_bounded<true>(&came_bar, came))) {
                    if (lane == 0) atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                    break;
                }
                came ^= 1u;
#pragma unroll 4
                for (int at = half; at < n; at += 2) {
                    float v[MATS];
#pragma unroll
                    for (int m = 0; m < MATS; ++m) {
                        v[m] = parts[(at * MATS + m) * 128 + place];
                        for (uint32_t s = 1; s < size; ++s) v[m] += parts[(((int)s * share + at) * MATS + m) * 128 + place];
                    }
                    if (live) out[(mine + at) * args.ldo] = result(v);
                }
                __syncwarp();
                if (lane < (int)size) mbar_arrive_cluster(cluster_addr(smem_u32(&free_bar), (uint32_t)lane));
            }
        }
        __syncwarp();
    }
    // no CTA of the cluster leaves while another can reach its shared memory
    tc_fence_before();
    if (size > 1) {
        if (warp < R_EPI) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        cluster_sync();
    } else {
        __syncthreads();
    }
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(s_tmem, 512);
    }
}

// ------------------------------------------------------------------ host ----
// How many CTAs share a tile, 1 to 8, and how many clusters of them are
// launched (8192 x 512 of 17 rows by clusters of 1, 2, 4, 8: 45, 27, 17, 11 us).  In
// us: a k-block takes a CTA 0.33 a matrix, all weights come at 6 TB/s, and a tile's
// results take a few, more where parts are added.  `resident`: such clusters that run at once, asked of the
// driver once a kernel.
struct Share {
    int size, clusters, per;
};
template <typename K>
Share share_tiles(K kernel, int smem, std::atomic<int> (&resident)[8], long long tiles, long long nkb, int grain, int mats, int T, int places) {
    const long long units = (nkb + grain - 1) / grain;
    Share best{};
    double least = 0;
    for (int i = 0; i < 8; ++i) {
        const long long size = i + 1, per = (units + size - 1) / size;
        if ((units + per - 1) / per != size) continue;          // a CTA without a part
        if (size * ((T + size - 1) / size) > places) continue;  // no room for the parts
        int n = resident[i].load(std::memory_order_relaxed);
        if (!n) resident[i].store(n = resident_clusters(kernel, R_THREADS, smem, (int)size), std::memory_order_relaxed);
        const long long at_once = std::min<long long>(tiles, n), rounds = (tiles + n - 1) / n;
        const double block = std::max(0.33 * mats, (double)(mats * R_W * at_once * size) / 6e6);
        const double last = (i ? 3.0 : 1.0) + 0.03 * T;
        const double us = (double)rounds * std::max((double)(per * grain) * block, last) + last;
        if (!best.size || us < least) least = us, best = {(int)size, (int)at_once, (int)per * grain};
    }
    return best;
}

struct NarrowCall {
    int T;
    long long N, K;  // K elements
    const void* x;
    long long ldx;
    const void* w[2];
    long long ldw[2];
    const void *xs, *ws;
    uint16_t* out;
    long long ldo;
    bool after;
    uint32_t* status;
    cudaStream_t st;
};

template <bool FP8, int DT, int MATS, int ACT, int NT>
int launch_narrow_nt(const NarrowCall& c) {
    using S = Narrow<FP8, MATS, NT>;
    auto k = narrow_kernel<FP8, DT, MATS, ACT, NT>;
    static SmemOnce once;
    SFFN_CUDA_TRY(once.set(k, S::SMEM));
    constexpr int ES = FP8 ? 1 : 2, BK = 128 / ES;
    NarrowArgs a{};
    a.T = c.T, a.N = (int)c.N;
    a.nkb = (int)((c.K + BK - 1) / BK);
    a.out = c.out, a.ldo = c.ldo, a.status = c.status;
    a.tiles = (int)((c.N + 127) / 128);
    static std::atomic<int> resident[8];
    const Share share = share_tiles(k, S::SMEM, resident, a.tiles, a.nkb, FP8 ? 4 : 1, MATS, c.T, S::PLACES);
    a.per = share.per;
    const auto type = FP8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    const auto sw = CU_TENSOR_MAP_SWIZZLE_128B;
    CUtensorMap m[5];
    memset(m, 0, sizeof(m));
    for (int i = 0; i < MATS; ++i)
        if (int rc = tmap_2d(&m[i], type, ES, c.w[i], c.K, c.N, c.ldw[i], BK, 128, sw)) return rc;
    if (int rc = tmap_2d(&m[2], type, ES, c.x, c.K, c.T, c.ldx, BK, c.T, sw)) return rc;
    if constexpr (FP8) {
        const long long bt = fp8_block_tiles(c.K);
        if (int rc = scale_map(&m[3], c.ws, a.tiles, bt, 1)) return rc;
        if (int rc = tmap_2d(&m[4], CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, c.xs, 4, bt * 32, 4, 4, 32, CU_TENSOR_MAP_SWIZZLE_NONE)) return rc;
    }
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(share.clusters * share.size));
    config.blockDim = dim3(R_THREADS);
    config.dynamicSmemBytes = S::SMEM;
    config.stream = c.st;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)share.size, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = c.after ? 2 : 1;
    SFFN_CUDA_TRY(cudaLaunchKernelEx(&config, k, m[0], m[1], m[2], m[3], m[4], a));
    return SFFN_OK;
}

template <bool FP8, int DT, int MATS, int ACT>
int launch_narrow(const NarrowCall& c) {
    return c.T <= 48 ? launch_narrow_nt<FP8, DT, MATS, ACT, 48>(c) : launch_narrow_nt<FP8, DT, MATS, ACT, 64>(c);
}

template <int DT>
int launch_narrow_gated(int act, const NarrowCall& c) {
    switch (act) {
        case GLU_RELU: return launch_narrow<false, DT, 2, GLU_RELU>(c);
        case GLU_RELU2: return launch_narrow<false, DT, 2, GLU_RELU2>(c);
        case GLU_SILU: return launch_narrow<false, DT, 2, GLU_SILU>(c);
        default: return launch_narrow<false, DT, 2, GLU_GELU>(c);
    }
}

}  // namespace

int narrow_mm(int dtype, const void* x, long long ldx, const void* w, long long ldw, long long T, long long N, long long K, void* out,
              long long ldo, bool after, uint32_t* status, cudaStream_t st) {
    const NarrowCall c{(int)T, N, K, x, ldx, {w, nullptr}, {ldw, 0}, nullptr, nullptr, static_cast<uint16_t*>(out), ldo, after, status, st};
    return dtype == SFFN_BF16 ? launch_narrow<false, SFFN_BF16, 1, 0>(c) : launch_narrow<false, SFFN_F16, 1, 0>(c);
}

int narrow_glu(int dtype, int act, const void* x, long long ldx, const void* wg, long long ldwg, const void* wu, long long ldwu, long long T,
               long long D, long long F, void* h, long long ldh, uint32_t* status, cudaStream_t st) {
    const NarrowCall c{(int)T, F, D, x, ldx, {wg, wu}, {ldwg, ldwu}, nullptr, nullptr, static_cast<uint16_t*>(h), ldh, false, status, st};
    return dtype == SFFN_BF16 ? launch_narrow_gated<SFFN_BF16>(act, c) : launch_narrow_gated<SFFN_F16>(act, c);
}

int narrow_fp8(const void* x, long long ldx, const void* x_scales, const void* w, long long ldw, const void* w_scales, long long T, long long N,
               long long K, void* out, int out_dtype, long long ldo, bool after, uint32_t* status, cudaStream_t st) {
    const NarrowCall c{(int)T, N, K, x, ldx, {w, nullptr}, {ldw, 0}, x_scales, w_scales, static_cast<uint16_t*>(out), ldo, after, status, st};
    return out_dtype == SFFN_BF16 ? launch_narrow<true, SFFN_BF16, 1, 0>(c) : launch_narrow<true, SFFN_F16, 1, 0>(c);
}

}  // namespace sffn
