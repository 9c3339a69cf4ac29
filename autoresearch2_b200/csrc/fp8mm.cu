// Product of two matrices in the 8-bit block format (fp8.cuh):
// C[M, N] = A[M, K] B[N, K]^T, both with one power-of-two scale for each 128
// elements of a row, C in 16 bits.
//
// tcgen05.mma kind::mxf8f6f4 with block scaling: the tensor cores multiply each
// 32 products' sum by 2^(ea + eb) as they accumulate in float32, at the full
// 8-bit rate; the four 32-wide steps of a 128-wide k-block use the same scale
// byte.  One scale tile (128 rows x 4 blocks, 512 bytes) holds four k-blocks'
// scales, which the instruction's scale-id field picks.
//
// CTA pairs, persistent over 256 x 256 tiles; each CTA loads its 128 rows of A
// and of B (128 bytes of K a stage), its A scale tile and the two of B.
//   warps 0-5    TMA issuers of A and B, three each for every third k-block: one
//                thread's copies complete one after another, about one per trip to
//                L2, and a stage is multiplied in half of such a trip
//   warp 6       MMA issuer (leader): at every fourth k-block three tcgen05.cp bring
//                the next four's scales to tensor memory; four tcgen05.mma a stage
//   warp 7       allocates tensor memory and issues the copies of the scales, two for
//                four k-blocks
//   warps 8-15   epilogue, two warpgroups of 128 columns.  The accumulator takes
//                256 of 512 columns and the scales need some, so there is one:
//                the epilogue frees it fast, as 16-bit pairs in 128 spare
//                columns, and stores from there while the next tile runs.
// The 256 x 256 tile is as large as tensor memory allows: at 8 bits a stage's
// 32 KB a CTA feed 512 cycles of MMA, 64 bytes a cycle, and L2 delivers 40 to 45: its
// bound.  16384 x 8192 x 4096: 456 us, 2.4 PFLOP/s, 1.47 times the measured 16-bit
// rate (one issuer an operand, scales with every k-block: 490).  Few tiles
// and a long K are split over K: 256 x 4096 x 14336 32 us, 54 unsplit.
#include <cuda.h>
#include <string.h>

#include "fp8.cuh"
#include "parts.cuh"
#include "stage.cuh"
#include "tmap.cuh"

namespace sffn {
namespace {

constexpr int X_ISSUERS = 3;  // of each operand
constexpr int X_STAGES = 6;   // a multiple: a stage belongs to one issuer
constexpr int X_THREADS = 512;
constexpr int X_OPERAND = 128 * 128;             // bytes of one operand a stage and CTA
constexpr int X_STAGE = 2 * X_OPERAND;
constexpr int X_SCALES = 3 * 512;                // A's tile, B's two
constexpr int X_SMEM = X_STAGES * (X_STAGE + X_SCALES) + 8 * 2048 + 1024;
constexpr int X_PACK_COL = 256;                  // 64 columns per warpgroup
constexpr int X_SCALE_COL = 384;                 // 12 columns per stage: 4 of A, 8 of B
static_assert(X_SCALE_COL + 12 * X_STAGES <= 512, "tensor memory columns");
static_assert(X_SMEM <= 232448, "shared memory");

struct MmArgs {
    int M, N, K;
    int tiles_m, tiles_n;  // of 128 rows, of 256 columns
    int tiles_b;           // 128-row tiles of B
    int bt;                // scale tiles across K
    uint16_t* out;
    long long ldc;
    int vec_out;
    int splits, per_split;  // parts of K, k-blocks of each (a multiple of 4)
    float* part;            // splits > 1: [splits][M][ldp]
    long long ldp;
    uint32_t* status;
};

// kind::mxf8f6f4: e4m3 operands (format 0), K-major, ue8m0 scales (bit 23); the
// scale bytes used by A (bits 29, 30) and B (bits 4, 5).
__device__ constexpr uint32_t idesc_mx(int M, int N) {
    return ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void mma_mx_pair(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t sa, uint32_t sb,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
        : "memory");
}
// A 3-D box for a CTA pair, completing on the leader's barrier.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const void* tmap, int c0, int c1, int c2, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(leader_smem_addr(bar))
        : "memory");
}
// 32 rows of 16 bytes -> 4 tensor-memory columns, the same in each quarter of
// the lanes; in each CTA of the pair from its own shared memory.
__device__ __forceinline__ void cp_scales_pair(uint32_t taddr, uint64_t sdesc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}

template <int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(X_THREADS, 1)
    fp8_mm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                  const __grid_constant__ CUtensorMap tmC, const MmArgs args) {
    constexpr uint32_t IDESC = idesc_mx(256, 256);
    extern __shared__ __align__(1024) unsigned char x_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(x_smem_raw) + 1023) &
                                                           ~static_cast<uintptr_t>(1023));
    unsigned char* sscales = smem + X_STAGES * X_STAGE;
    __shared__ __align__(8) uint64_t full_bar[X_STAGES], empty_bar[X_STAGES];
    __shared__ __align__(8) uint64_t tfull_bar, tempty_bar;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_mp = (args.tiles_m + 1) / 2;
    const int tiles = tiles_mp * args.tiles_n;
    const int ntasks = tiles * args.splits;
    const int nkb = (args.K + 127) / 128;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int first_task = (int)cluster_id_x();
    const int task_stride = (int)cluster_count_x();
    // the tile of a task and its k-blocks; all tiles of one part of K run together
    auto locate = [&](int task, int& pm, int& tn, int& kb0, int& kb1) {
        const int sp = task / tiles;
        pair_raster(task - sp * tiles, tiles_mp, args.tiles_n, pm, tn);
        kb0 = sp * args.per_split;
        kb1 = min(nkb, kb0 + args.per_split);
        return sp;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < X_STAGES; ++s) {
            mbar_init(&full_bar[s], 1);   // the leader's arrive.expect_tx, for both CTAs' bytes
            mbar_init(&empty_bar[s], 1);  // one multicast commit a use
        }
        mbar_init(&tfull_bar, 1);
        mbar_init(&tempty_bar, 16);  // the 8 epilogue warps of both CTAs
        s_abort = 0;
        fence_mbar_init();
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
        prefetch_tmap(&tmSA);
        prefetch_tmap(&tmSB);
    }
    if (warp == 7) {
        tmem_alloc_pair(&s_tmem, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = s_tmem;

    if (warp < 6 || warp == 7) {
        // ------------------------------------------------------ producers --
        const int op = warp == 7 ? 2 : warp / X_ISSUERS;  // 0: A, 1: B, 2: scales
        if (lane == 0) {
            int armed[X_STAGES] = {0};
            long long kc = 0;
            int sgroup = 0;  // groups of up to four k-blocks with one tile of scales so far
            bool stop = false;
            for (int task = first_task; task < ntasks && !stop && !s_abort; task += task_stride) {
                int pm, tn, kb0, kb1;
                locate(task, pm, tn, kb0, kb1);
                const int arow = (pm * 2 + (int)rank) * 128;
                const int brow = tn * 256 + (int)rank * 128;
                for (int kb = kb0; kb < kb1; ++kb, ++kc) {
                    if (op == 2 ? (kb & 3) != 0 : (int)(kc % X_ISSUERS) != warp % X_ISSUERS) continue;
                    const int stage = (int)(kc % X_STAGES);
                    const uint32_t phase = (uint32_t)((kc / X_STAGES) & 1);
                    if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1u)) {
                        atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                        s_abort = 1;
                        stop = true;
                        break;
                    }
                    unsigned char* sa = smem + stage * X_STAGE;
                    if (op == 0) {
                        if (leader) {
                            mbar_arrive_expect_tx(&full_bar[stage], 2 * (X_STAGE + ((kb & 3) == 0 ? X_SCALES : 0)));
                            ++armed[stage];
                        }
                        tma_load_2d_pair(sa, &tmA, kb * 128, arow, &full_bar[stage]);
                    } else if (op == 1) {
                        tma_load_2d_pair(sa + X_OPERAND, &tmB, kb * 128, brow, &full_bar[stage]);
                    } else {
                        // Slots are as many as stages and a group has a k-block at
                        // least: the slot's last group lies a whole ring back, its
                        // tcgen05.cp before the commit waited for above.
                        unsigned char* ss = sscales + sgroup * X_SCALES;
                        tma_load_3d_pair(ss, &tmSA, 0, (kb >> 2) * 32, pm * 2 + (int)rank, &full_bar[stage]);
                        tma_load_3d_pair(ss + 512, &tmSB, 0, (kb >> 2) * 32, tn * 2, &full_bar[stage]);
                        sgroup = sgroup + 1 == X_STAGES ? 0 : sgroup + 1;
                    }
                }
            }
            // once the last phases armed here complete, no copy is still landing in either CTA
            if (leader && op == 0)
                for (int s = 0; s < X_STAGES; ++s)
                    if (armed[s]) (void)mbar_wait_bounded(&full_bar[s], (uint32_t)(armed[s] - 1) & 1u);
        }
        __syncwarp();
    } else if (warp == 6) {
        // ----------------------------------------------------------- MMA --
        if (lane == 0 && leader) {
            int stage = 0, it = 0, sgroup = -1;
            uint32_t phase = 0;
            for (int task = first_task; task < ntasks && !s_abort; task += task_stride, ++it) {
                int pm, tn, kb0, kb1;
                locate(task, pm, tn, kb0, kb1);
                if (!mbar_wait_bounded(&tempty_bar, ((uint32_t)it & 1u) ^ 1u)) {
                    atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                    s_abort = 1;
                    break;
                }
                tc_fence_after();
                bool ready = mbar_try_wait(&full_bar[stage], phase), fail = false;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!ready && !mbar_wait_bounded(&full_bar[stage], phase)) {
                        atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                        s_abort = 1;
                        fail = true;
                        break;
                    }
                    const uint32_t sa = smem_u32(smem + stage * X_STAGE), sb = sa + X_OPERAND;
                    if ((kb & 3) == 0) sgroup = sgroup + 1 == X_STAGES ? 0 : sgroup + 1;
                    // the group's own columns, free as its shared memory is
                    const uint32_t ta = tmem_base + X_SCALE_COL + 12u * (uint32_t)sgroup, tb = ta + 4u;
                    if ((kb & 3) == 0) {
                        const uint32_t ss = smem_u32(sscales + sgroup * X_SCALES);
                        cp_scales_pair(ta, smem_desc_rows16(ss));
                        cp_scales_pair(tb, smem_desc_rows16(ss + 512));
                        cp_scales_pair(tb + 4u, smem_desc_rows16(ss + 1024));
                    }
                    const uint32_t id = (uint32_t)kb & 3u;
                    const uint32_t idesc = IDESC | (id << 4) | (id << 29);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma_mx_pair(tmem_base, umma_desc_sw128(sa + 32 * j, 16, 1024), umma_desc_sw128(sb + 32 * j, 16, 1024),
                                    idesc, ta, tb, ((kb - kb0) | j) != 0 ? 1u : 0u);
                    tc_commit_pair_multicast(&empty_bar[stage], 0x3);
                    if (++stage == X_STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    ready = kb + 1 < kb1 && mbar_try_wait(&full_bar[stage], phase);
                }
                if (fail) break;
                tc_commit_pair_multicast(&tfull_bar, 0x3);
            }
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ------------------------------------------------------ epilogue --
        const int ew = warp & 3, wg = (warp - 8) >> 2;
        unsigned char* sbuf = sscales + X_STAGES * X_SCALES + (warp - 8) * 2048;
        StageRing<1> ring(sbuf);
        const uint32_t tempty_leader = leader_smem_addr(&tempty_bar);
        const uint32_t lane_base = tmem_base + ((uint32_t)(ew * 32) << 16);
        int it = 0;
        for (int task = first_task; task < ntasks; task += task_stride, ++it) {
            int pm, tn, kb0, kb1;
            const int sp = locate(task, pm, tn, kb0, kb1);
            const int row0 = (pm * 2 + (int)rank) * 128 + ew * 32, col0 = tn * 256 + wg * 128;
            const bool ok = __all_sync(FULL, mbar_wait_bounded(&tfull_bar, (uint32_t)it & 1u));
            if (!ok || __any_sync(FULL, s_abort != 0)) {
                if (lane == 0 && !ok) atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                break;
            }
            tc_fence_after();
            if (args.splits > 1) {  // float32 parts: each lane its row's 128 contiguous bytes
#pragma unroll 1
                for (int c = 0; c < 4 && row0 < args.M && col0 + c * 32 < args.N; ++c) {
                    uint32_t r[32];
                    tmem_ld32(lane_base + (uint32_t)(wg * 128 + c * 32), r);
                    tmem_wait_ld();
                    if (row0 + lane < args.M) {
                        float* p = args.part + ((long long)sp * args.M + row0 + lane) * args.ldp + col0 + c * 32;
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            if (col0 + c * 32 + 4 * q < args.ldp)  // ldp is a multiple of 4
                                reinterpret_cast<uint4*>(p)[q] = make_uint4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(tempty_leader);
                continue;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t r[32], w[16];
                tmem_ld32(lane_base + (uint32_t)(wg * 128 + c * 32), r);
                tmem_wait_ld();
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    w[q] = pack16x2<DT>(__uint_as_float(r[2 * q]), __uint_as_float(r[2 * q + 1]));
                tmem_st16(lane_base + (uint32_t)(X_PACK_COL + wg * 64 + c * 16), w);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty_leader);
            if (row0 >= args.M) continue;
#pragma unroll 1
            for (int c = 0; c < 4 && col0 + c * 32 < args.N; ++c) {
                uint32_t w[16];
                tmem_ld16(lane_base + (uint32_t)(X_PACK_COL + wg * 64 + c * 16), w);
                tmem_wait_ld();
                const int col = col0 + c * 32;
                if (args.vec_out) {
                    ring.store(&tmC, lane, w, col, row0);
                } else {
                    stage_store_plain(args.out, args.ldc, args.M, args.N, sbuf, lane, w, col, row0);
                }
            }
        }
        if (lane == 0) bulk_wait_group0();
        __syncwarp();
    }
    // neither CTA leaves while the other can touch its shared or tensor memory
    tc_fence_before();
    cluster_sync();
    if (warp == 7) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

template <int DT>
int launch_mm(const void* a, long long lda, const void* as, const void* b, long long ldb, const void* bs, MmArgs args,
              cudaStream_t st) {
    CUtensorMap ta, tb, tsa, tsb, tc;
    memset(&tc, 0, sizeof(tc));
    const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const auto sw = CU_TENSOR_MAP_SWIZZLE_128B;
    if (int rc = tmap_2d(&ta, u8, 1, a, args.K, args.M, lda, 128, 128, sw)) return rc;
    if (int rc = tmap_2d(&tb, u8, 1, b, args.K, args.N, ldb, 128, 128, sw)) return rc;
    if (int rc = scale_map(&tsa, as, args.tiles_m, args.bt, 1)) return rc;
    if (int rc = scale_map(&tsb, bs, args.tiles_b, args.bt, 2)) return rc;
    if (args.vec_out && args.splits == 1)
        if (int rc = tmap_2d(&tc, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, args.out, args.N, args.M, args.ldc, 32, 32,
                             CU_TENSOR_MAP_SWIZZLE_64B))
            return rc;
    auto k = fp8_mm_kernel<DT>;
    static SmemOnce once;
    SFFN_CUDA_TRY(once.set(k, X_SMEM));
    static const int pairs = resident_pairs(k, X_THREADS, X_SMEM);
    const long long tasks = (long long)((args.tiles_m + 1) / 2) * args.tiles_n * args.splits;
    const int clusters = (int)std::min<long long>(tasks, pairs);
    k<<<clusters * 2, X_THREADS, X_SMEM, st>>>(ta, tb, tsa, tsb, tc, args);
    SFFN_CHECK_LAUNCH();
    return args.splits > 1 ? join_parts<DT>(args.part, args.splits, args.M, args.N, args.out, args.ldc, st) : SFFN_OK;
}

// Parts of K: a 128-wide k-block of a pair takes about 0.45 us, four share a scale tile.
int split8(long long M, long long N, long long K) { return split_of(M, N, (K + 127) / 128, 4, 0.45); }

// Coordinates and scale rows are 32-bit in the tensor maps.
bool mm_sizes_ok(long long M, long long N, long long K) {
    const long long most = 0x7FFFFF00;
    return M <= most && N <= most && K <= most && (M + 127) / 128 * fp8_block_tiles(K) * 32 <= 0x7FFFFFFF &&
           (N + 127) / 128 * fp8_block_tiles(K) * 32 <= 0x7FFFFFFF && tiles_of(M, N) <= 0x1FFFFFF;
}

}  // namespace
}  // namespace sffn

using namespace sffn;

extern "C" size_t sffn_fp8_mm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0 || !mm_sizes_ok(M, N, K)) return 0;
    const int s = split8(M, N, K);
    return s > 1 ? (size_t)s * (size_t)M * (size_t)part_ld(N) * 4 : 0;
}

extern "C" int sffn_fp8_mm(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb,
                           const void* b_scales, int64_t M, int64_t N, int64_t K, void* C, int c_dtype, int64_t ldc,
                           void* workspace, size_t workspace_bytes, uint32_t* status_dev, void* stream) {
    if (c_dtype != SFFN_BF16 && c_dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (M < 0 || N < 0 || K <= 0) return SFFN_ERR_ARG;
    if (M == 0 || N == 0) return SFFN_OK;
    if (!a || !a_scales || !b || !b_scales || !C || !status_dev || lda < K || ldb < K || ldc < N) return SFFN_ERR_ARG;
    if (!mm_sizes_ok(M, N, K)) return SFFN_ERR_TOO_LARGE;
    if (!aligned16(a) || !aligned16(b) || !aligned16(a_scales) || !aligned16(b_scales) || lda % 16 || ldb % 16 ||
        reinterpret_cast<uintptr_t>(C) % 2 || !aligned16(workspace))
        return SFFN_ERR_ALIGN;
    const size_t need = sffn_fp8_mm_workspace_bytes(M, N, K);
    if (need && (!workspace || workspace_bytes < need)) return SFFN_ERR_WORKSPACE;
    DeviceScope scope;
    if (int rc = scope.bind(a)) return rc;
    if (!sm100_sms()) return SFFN_ERR_DEVICE;
    MmArgs args{};
    args.M = (int)M;
    args.N = (int)N;
    args.K = (int)K;
    args.tiles_m = (int)((M + 127) / 128);
    args.tiles_n = (int)((N + 255) / 256);
    args.tiles_b = (int)((N + 127) / 128);
    args.bt = (int)fp8_block_tiles(K);
    args.out = static_cast<uint16_t*>(C);
    args.ldc = ldc;
    args.vec_out = aligned16(C) && ldc % 8 == 0;
    args.splits = split8(M, N, K);
    const int nkb = (int)((K + 127) / 128);
    args.per_split = ((nkb + 3) / 4 + args.splits - 1) / args.splits * 4;
    args.part = static_cast<float*>(workspace);
    args.ldp = part_ld(N);
    args.status = status_dev;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return c_dtype == SFFN_BF16 ? launch_mm<SFFN_BF16>(a, lda, a_scales, b, ldb, b_scales, args, st)
                                : launch_mm<SFFN_F16>(a, lda, a_scales, b, ldb, b_scales, args, st);
}
