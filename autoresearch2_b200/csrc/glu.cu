// The gated feed-forward block h = act(x Wg^T) * (x Wu^T), y = h W2^T, and the
// products of its backward, in bfloat16 or float16 on the tcgen05 tensor cores.
//
// Bound by the tensor cores under the power limit where K is long (UP of 8192 x
// 4096 x 14336: 1.54 ms, 1250 TF), by the operands' way from L2 where it is short:
// at 32768 x 768 x 2048 UP reads 1.57 GB of tiles from L2 in 165 us, 9.5 TB/s, the
// rate that plain products of this K have too (32768 x 768 x 2304: 96 us).  DGRAD takes
// 167 us there with nothing saturated: 0.13 GB of g and u and 0.4 GB of results beside
// 0.8 GB of tiles, in all 6.5 TB/s read from L2, DRAM at half its rate, tensor pipe 30%,
// issue slots 38%.  What holds it is not known; its epilogue waits twice every 32
// columns for its own stores to be read.
//
// One kernel: CTA pairs (tcgen05.mma.cta_group::2, 256 x 256 tiles, float32
// accumulation in tensor memory, two accumulators), persistent over tiles;
// operands by TMA in a ring of 64-wide k-blocks, either major order, so no
// operand is transposed.
//   warps 0,2 / 3 and the last  issuers of A / B (even / odd k-blocks)
//   warp 1                      MMA issuer (leader CTA)
//   warp 2                      also tensor memory
//   warps 4-11 or 4-19          epilogue, two or four warpgroups; thread = accumulator row
// Epilogues:
//   STORE  C in 16 bits; or, split over K, float32 parts that a second kernel
//          adds in order (few tiles and a long K: weight gradients).  K may run
//          on into a second pair of operands: dx = dg Wg + du Wu is one product.
//   UP     the pair's B rows are 128 of Wg (leader's shared memory) and the
//          same 128 of Wu (peer's), so the accumulator holds g and u of 128
//          columns side by side: h is formed here from the unrounded g and u,
//          and g and u are kept for the backward in 16 bits or in the 8-bit
//          block format (a tile's 128 columns are one block).
//   DGRAD  dh = dy W2; reads g and u as they were kept and writes
//          dg = dh u act'(g), du = dh act(g) and h = act(g) u (for dW2): dh
//          itself is never stored.
#include <cuda.h>
#include <string.h>

#include <algorithm>

#include "act.cuh"
#include "fp8.cuh"
#include "parts.cuh"
#include "stage.cuh"
#include "tmap.cuh"

namespace sffn {
namespace {

enum { P_STORE = 0, P_UP = 1, P_DGRAD = 2 };
enum { KEEP_NONE = 0, KEEP_16 = 1, KEEP_8 = 2 };

constexpr int P_BK = 64;
// Warps of the epilogue: eight store, sixteen where they compute as well: chains of
// conversions, exponentials and reciprocals, and copies to wait for (with eight, UP
// and DGRAD of 32768 x 768 x 2048 took 173 and 178 us instead of 165 and 167).
template <int EPI>
constexpr int p_epi() { return EPI == P_STORE ? 8 : 16; }
template <int EPI>
constexpr int p_threads() { return (5 + p_epi<EPI>()) * 32; }
constexpr int P_OPERAND = 128 * P_BK * 2;  // bytes of one operand a stage and CTA
constexpr int P_STAGE = 2 * P_OPERAND;
// Even counts: the issuers take alternate k-blocks.
template <int EPI>
constexpr int p_stages() { return EPI == P_STORE ? 6 : 4; }
// Bytes an epilogue warp has for staging: STORE two blocks of 32 x 32, UP three
// (h, g, u; in 8 bits g and u share one, the third is for the amax), DGRAD two
// and its g and u as kept.
template <int EPI>
constexpr int p_own() { return EPI == P_STORE ? 4096 : 6144; }
template <int EPI>
constexpr int p_smem() { return p_stages<EPI>() * P_STAGE + p_epi<EPI>() * p_own<EPI>() + 1024; }
static_assert(p_smem<P_STORE>() <= 227 * 1024 - 1024 && p_smem<P_UP>() <= 227 * 1024 - 1024, "shared memory");

struct PairArgs {
    int M, N;
    int tiles_m, tiles_n;  // of 128 rows; of 256 accumulator columns (UP: 128 columns of h)
    int nkb1, nkb;         // k-blocks of the first pair of operands, and of both
    int splits, per_split;
    uint16_t* out;  // STORE
    long long ldc;
    int vec_out;
    float* part;  // STORE, splits > 1: [splits][M][ldp]
    long long ldp;
    int keep;
    uint8_t *gs, *us;  // KEEP_8: scale tiles of g and u
    int bt;  // scale tiles across a row
    uint32_t* status;
};

template <int DT>
__device__ constexpr uint32_t idesc16(bool a_mn, bool b_mn) {
    const uint32_t f = DT == SFFN_BF16 ? 1u : 0u;  // both operands of one type
    return (1u << 4) | (f << 7) | (f << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(256 >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
}

// Four scaled values as four e4m3 bytes.
__device__ __forceinline__ uint32_t fp8_four(Float2 lo, Float2 hi) {
    const float2 a = split2(lo), b = split2(hi);
    return (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
           ((uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16);
}

template <int DT, bool A_MN, bool B_MN, int EPI, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(p_threads<EPI>(), 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmA2, const __grid_constant__ CUtensorMap tmB2,
                const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmC2,
                const __grid_constant__ CUtensorMap tmC3, const __grid_constant__ CUtensorMap tmG,
                const __grid_constant__ CUtensorMap tmU, const PairArgs args) {
    constexpr int NST = p_stages<EPI>();
    constexpr uint32_t IDESC = idesc16<DT>(A_MN, B_MN);
    constexpr uint32_t MN_LBO = P_BK * 128;  // MN-major: 64-element blocks of 64 K rows x 128 bytes
    constexpr int TILE_N = EPI == P_UP ? 128 : 256;
    constexpr int EW = p_epi<EPI>(), WG_N = TILE_N / (EW / 4);  // epilogue warps; columns of a warpgroup
    extern __shared__ __align__(1024) unsigned char p_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p_smem_raw) + 1023) &
                                                           ~static_cast<uintptr_t>(1023));
    __shared__ __align__(8) uint64_t full_bar[NST], empty_bar[NST];
    __shared__ __align__(8) uint64_t tfull_bar[2], tempty_bar[2];
    __shared__ __align__(8) uint64_t kept_bar[EW];  // DGRAD: each epilogue warp's g and u have come
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles_mp = (args.tiles_m + 1) / 2;
    const int ntasks = tiles_mp * args.tiles_n * args.splits;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int first_task = (int)cluster_id_x();
    const int task_stride = (int)cluster_count_x();
    // the tile of a task and its k-blocks
    auto locate = [&](int task, int& pm, int& tn, int& kb0, int& kb1) {
        int sp = 0;
        // all tiles of one part of K run together: they share its operands in L2
        // (2304 x 768 of 32768 in 5 parts: 113 -> 106 us)
        if (EPI == P_STORE && args.splits > 1) {
            const int tiles = tiles_mp * args.tiles_n;
            sp = task / tiles;
            task -= sp * tiles;
        }
        pair_raster(task, tiles_mp, args.tiles_n, pm, tn);
        kb0 = sp * args.per_split;
        kb1 = min(args.nkb, kb0 + args.per_split);
        return sp;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < NST; ++s) {
            mbar_init(&full_bar[s], 1);   // the leader's arrive.expect_tx, for both CTAs' bytes
            mbar_init(&empty_bar[s], 1);  // one multicast commit a use
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull_bar[a], 1);
            mbar_init(&tempty_bar[a], 2 * EW);  // the epilogue warps of both CTAs
        }
        for (int w = 0; w < EW; ++w) mbar_init(&kept_bar[w], 1);
        s_abort = 0;
        fence_mbar_init();
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
    }
    if (warp == 2) {
        tmem_alloc_pair(&s_tmem, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = s_tmem;

    if (warp == 0 || warp == 2 || warp == 3 || warp == 4 + EW) {
        // ----------------------------------------------------- producers --
        // Four issuing threads, one per (operand, k-block parity): one thread's
        // copies complete one after another.  B's bytes may land before the A
        // issuer arms the barrier; its transaction count goes below zero
        // meanwhile, and the phase cannot complete before the arrival.
        const bool loads_a = warp == 0 || warp == 2;
        const int par = (warp == 0 || warp == 3) ? 0 : 1;
        if (lane == 0) {
            int armed[NST] = {0};
            long long kc = 0;
            bool stop = false;
            for (int task = first_task; task < ntasks && !stop && !s_abort; task += task_stride) {
                int pm, tn, kb0, kb1;
                locate(task, pm, tn, kb0, kb1);
                const int arow = (pm * 2 + (int)rank) * 128;
                const int brow = EPI == P_UP ? tn * 128 : tn * 256 + (int)rank * 128;
                for (int kb = kb0; kb < kb1; ++kb, ++kc) {
                    if ((int)(kc & 1) != par) continue;
                    const int stage = (int)(kc % NST);
                    const uint32_t phase = (uint32_t)((kc / NST) & 1);
                    if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1u)) {
                        atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                        s_abort = 1;
                        stop = true;
                        break;
                    }
                    unsigned char* sa = smem + stage * P_STAGE;
                    const bool second = EPI == P_STORE && kb >= args.nkb1;
                    const int k = (second ? kb - args.nkb1 : kb) * P_BK;
                    if (loads_a) {
                        if (leader) {
                            mbar_arrive_expect_tx(&full_bar[stage], 2 * P_STAGE);
                            ++armed[stage];
                        }
                        const CUtensorMap* ma = second ? &tmA2 : &tmA;
                        if constexpr (!A_MN) {
                            tma_load_2d_pair(sa, ma, k, arow, &full_bar[stage]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                tma_load_2d_pair(sa + j * MN_LBO, ma, arow + j * 64, k, &full_bar[stage]);
                        }
                    } else {
                        unsigned char* sb = sa + P_OPERAND;
                        const CUtensorMap* mb = EPI == P_UP ? (leader ? &tmB : &tmB2) : second ? &tmB2 : &tmB;
                        if constexpr (!B_MN) {
                            tma_load_2d_pair(sb, mb, k, brow, &full_bar[stage]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 2; ++j)
                                tma_load_2d_pair(sb + j * MN_LBO, mb, brow + j * 64, k, &full_bar[stage]);
                        }
                    }
                }
            }
            // once the last phases armed here complete, no copy is still landing in either CTA
            if (leader && loads_a)
                for (int s = 0; s < NST; ++s)
                    if (armed[s]) (void)mbar_wait_bounded(&full_bar[s], (uint32_t)(armed[s] - 1) & 1u);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ----------------------------------------------------------- MMA --
        if (lane == 0 && leader) {
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            for (int task = first_task; task < ntasks && !s_abort; task += task_stride) {
                int pm, tn, kb0, kb1;
                locate(task, pm, tn, kb0, kb1);
                if (!mbar_wait_bounded(&tempty_bar[acc], acc_phase ^ 1u)) {
                    atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                    s_abort = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t d = tmem_base + (uint32_t)(acc * 256);
                bool ready = mbar_try_wait(&full_bar[stage], phase), fail = false;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!ready && !mbar_wait_bounded(&full_bar[stage], phase)) {
                        atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                        s_abort = 1;
                        fail = true;
                        break;
                    }
                    const uint32_t sa = smem_u32(smem + stage * P_STAGE), sb = sa + P_OPERAND;
#pragma unroll
                    for (int k = 0; k < P_BK / 16; ++k) {
                        const uint64_t ad = A_MN ? umma_desc_sw128(sa + k * 2048, MN_LBO, 1024)
                                                 : umma_desc_sw128(sa + k * 32, 16, 1024);
                        const uint64_t bd = B_MN ? umma_desc_sw128(sb + k * 2048, MN_LBO, 1024)
                                                 : umma_desc_sw128(sb + k * 32, 16, 1024);
                        tc_mma_f16_pair(d, ad, bd, IDESC, ((kb - kb0) | k) != 0 ? 1u : 0u);
                    }
                    tc_commit_pair_multicast(&empty_bar[stage], 0x3);
                    if (++stage == NST) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    ready = kb + 1 < kb1 && mbar_try_wait(&full_bar[stage], phase);
                }
                if (fail) break;
                tc_commit_pair_multicast(&tfull_bar[acc], 0x3);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------ epilogue --
        const int wg = (warp - 4) >> 2, ew = warp & 3;
        unsigned char* sbuf = smem + NST * P_STAGE + (warp - 4) * p_own<EPI>();
        StageRing<2> ring(sbuf);
        const uint32_t tempty_leader[2] = {leader_smem_addr(&tempty_bar[0]), leader_smem_addr(&tempty_bar[1])};
        // DGRAD: g and u as kept come by TMA, 32 bytes of the warp's 32 rows of each,
        // one such piece ahead, across tiles (each lane's own loads, of 32 rows an
        // instruction, took half of the kernel's time)
        unsigned char* kept = sbuf + 4096;
        uint64_t* kbar = &kept_bar[warp - 4];
        const int piece = args.keep == KEEP_8 ? 32 : 16;  // columns
        int f_task = first_task, f_col = 0;               // the next piece to fetch
        uint32_t k_phase = 0;
        bool k_due = false;           // a fetch is under way
        auto fetch_kept = [&] {       // what the place held is in registers
            __syncwarp();
            k_due = false;
            while (f_task < ntasks) {
                int pm, tn, kb0, kb1;
                locate(f_task, pm, tn, kb0, kb1);
                const int row0 = (pm * 2 + (int)rank) * 128 + ew * 32, col = tn * TILE_N + wg * WG_N + f_col;
                if (f_col < WG_N && row0 < args.M && col < args.N) {
                    if (lane == 0) {
                        mbar_arrive_expect_tx(kbar, 2048);
                        tma_load_2d(kept, &tmG, col, row0, kbar);
                        tma_load_2d(kept + 1024, &tmU, col, row0, kbar);
                    }
                    k_due = true;
                    f_col += piece;
                    return;
                }
                f_task += task_stride;
                f_col = 0;
            }
        };
        auto wait_kept = [&] {
            if (!__all_sync(FULL, mbar_wait_bounded(kbar, k_phase))) {
                if (lane == 0) atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                return false;
            }
            k_phase ^= 1u;
            k_due = false;
            return true;
        };
        if constexpr (EPI == P_DGRAD) fetch_kept();
        int acc = 0, it = 0;
        uint32_t acc_phase = 0;
        for (int task = first_task; task < ntasks; task += task_stride, ++it) {
            int pm, tn, kb0, kb1;
            const int sp = locate(task, pm, tn, kb0, kb1);
            const int row0 = (pm * 2 + (int)rank) * 128 + ew * 32;  // first row of this warp
            const int row = row0 + lane;
            const bool row_ok = row < args.M;
            const int gcol0 = tn * TILE_N + wg * WG_N;  // first column of this warpgroup
            float2 scales_ahead = make_float2(1.f, 1.f);
            if constexpr (EPI == P_DGRAD) {  // while the products still run
                if (args.keep == KEEP_8 && row_ok && gcol0 < args.N) {
                    const long long at = fp8_scale_at(row, gcol0 >> 7, args.bt);
                    scales_ahead = make_float2(fp8_scale(args.gs[at]), fp8_scale(args.us[at]));
                }
            }
            const bool ok = __all_sync(FULL, mbar_wait_bounded(&tfull_bar[acc], acc_phase));
            if (!ok && lane == 0) atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
            bool dead = !ok || __any_sync(FULL, s_abort != 0);
            if (dead && !(EPI == P_UP && args.keep == KEEP_8)) break;
            tc_fence_after();
            const uint32_t tbase = tmem_base + ((uint32_t)(ew * 32) << 16) + (uint32_t)(acc * 256 + wg * WG_N);

            if constexpr (EPI == P_STORE) {
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const int col = gcol0 + c * 32;
                    if (row0 >= args.M || col >= args.N) break;  // warp-uniform
                    uint32_t r[32];
                    tmem_ld32(tbase + c * 32, r);
                    tmem_wait_ld();
                    if (args.splits > 1) {
                        // float32 parts: each lane its row's 128 contiguous bytes
                        if (row_ok) {
                            float* p = args.part + ((long long)sp * args.M + row) * args.ldp + col;
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                if (col + 4 * q < args.ldp)  // ldp is a multiple of 4
                                    reinterpret_cast<uint4*>(p)[q] = make_uint4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
                        }
                        continue;
                    }
                    uint32_t w[16];
#pragma unroll
                    for (int q = 0; q < 16; ++q)
                        w[q] = pack16x2<DT>(__uint_as_float(r[2 * q]), __uint_as_float(r[2 * q + 1]));
                    if (args.vec_out) ring.store(&tmC, lane, w, col, row0);
                    else stage_store_plain(args.out, args.ldc, args.M, args.N, sbuf, lane, w, col, row0);
                }
            } else if constexpr (EPI == P_UP) {
                // 32 columns of h a warp, 16 at a time
                const bool live = !dead && row0 < args.M && gcol0 < args.N;
                float gtop = 0.f, utop = 0.f;
                if (live) {
                    if (lane == 0) bulk_wait_group_read0();
                    __syncwarp();
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t g[16], u[16], w[8];
                        tmem_ld16(tbase + half * 16, g);
                        tmem_ld16(tbase + 128 + half * 16, u);
                        tmem_wait_ld();
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            Float2 unused;
                            const Float2 gp = join2(__uint_as_float(g[2 * q]), __uint_as_float(g[2 * q + 1]));
                            const Float2 up = join2(__uint_as_float(u[2 * q]), __uint_as_float(u[2 * q + 1]));
                            const float2 h = split2(pair_mul(glu_act2<ACT, false>(gp, unused), up));
                            w[q] = pack16x2<DT>(h.x, h.y);
                        }
                        stage16(sbuf, lane, half, w);
                        if (args.keep == KEEP_16) {
#pragma unroll
                            for (int q = 0; q < 8; ++q) w[q] = pack16x2<DT>(__uint_as_float(g[2 * q]), __uint_as_float(g[2 * q + 1]));
                            stage16(sbuf + 2048, lane, half, w);
#pragma unroll
                            for (int q = 0; q < 8; ++q) w[q] = pack16x2<DT>(__uint_as_float(u[2 * q]), __uint_as_float(u[2 * q + 1]));
                            stage16(sbuf + 4096, lane, half, w);
                        } else if (args.keep == KEEP_8) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                gtop = fmaxf(gtop, fabsf(__uint_as_float(g[j])));  // NaN does not count
                                utop = fmaxf(utop, fabsf(__uint_as_float(u[j])));
                            }
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmC, sbuf, gcol0, row0);
                        if (args.keep == KEEP_16) {
                            tma_store_2d(&tmG, sbuf + 2048, gcol0, row0);
                            tma_store_2d(&tmU, sbuf + 4096, gcol0, row0);
                        }
                        bulk_commit_group();
                    }
                }
                if (args.keep == KEEP_8) {
                    uint32_t gmax = __float_as_uint(gtop), umax = __float_as_uint(utop);
                    // rare: infinities do not count either
                    const bool finite = !__any_sync(FULL, max(gmax, umax) >= 0x7F800000u);
                    if (!finite) {
                        gmax = umax = 0;
#pragma unroll 1
                        for (int half = 0; half < 2; ++half) {
                            uint32_t g[16], u[16];
                            tmem_ld16(tbase + half * 16, g);
                            tmem_ld16(tbase + 128 + half * 16, u);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                gmax = max(gmax, finite_mag(__uint_as_float(g[j])));
                                umax = max(umax, finite_mag(__uint_as_float(u[j])));
                            }
                        }
                    }
                    // The block of 128 columns spans the four warps of these rows (columns past
                    // N are zero).  A warp that gives up says so here, and all four leave: they
                    // meet once a tile or not at all.
                    const int slot = 4096 + (it & 1) * 256 + lane * 8;
                    *reinterpret_cast<uint2*>(sbuf + slot) = dead ? make_uint2(0xFFFFFFFFu, 0u) : make_uint2(gmax, umax);
                    named_bar_sync(1 + ew, 128);
#pragma unroll
                    for (int o = 1; o < 4; ++o) {
                        const uint2 v = *reinterpret_cast<const uint2*>(smem + NST * P_STAGE + ((wg ^ o) * 4 + ((warp - 4) & 3)) * p_own<EPI>() + slot);
                        gmax = max(gmax, v.x), umax = max(umax, v.y);
                    }
                    if (dead || gmax == 0xFFFFFFFFu) break;
                    const int ge = fp8_exponent(gmax), ue = fp8_exponent(umax);
                    if (row_ok && wg < 2) (wg ? args.us : args.gs)[fp8_scale_at(row, tn, args.bt)] = (uint8_t)((wg ? ue : ge) + 127);
                    if (live) {  // 32 bytes of g, then of u a row
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const float inv = two_to(m ? -ue : -ge);
                            const Float2 inv2 = join2(inv, inv);
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                uint32_t r[16], w[4];
                                tmem_ld16(tbase + m * 128 + half * 16, r);
                                tmem_wait_ld();
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    const float v0 = __uint_as_float(r[4 * q]), v1 = __uint_as_float(r[4 * q + 1]);
                                    const float v2 = __uint_as_float(r[4 * q + 2]), v3 = __uint_as_float(r[4 * q + 3]);
                                    w[q] = finite ? fp8_four(pair_mul(join2(v0, v1), inv2), pair_mul(join2(v2, v3), inv2))
                                                  : fp8_pack4<false>(v0, v1, v2, v3, inv);
                                }
                                *reinterpret_cast<uint4*>(sbuf + 2048 + m * 1024 + lane * 32 + half * 16) = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_2d(&tmG, sbuf + 2048, gcol0, row0);
                            tma_store_2d(&tmU, sbuf + 2048 + 1024, gcol0, row0);
                            bulk_commit_group();
                        }
                    }
                }
            } else {  // P_DGRAD
                const Float2 gs2 = join2(scales_ahead.x, scales_ahead.x), us2 = join2(scales_ahead.y, scales_ahead.y);
#pragma unroll 1
                for (int c = 0; c < WG_N / 32; ++c) {
                    const int col = gcol0 + c * 32;
                    if (row0 >= args.M || col >= args.N) break;
                    // dg and du go to the two buffers as they are formed, h to the first one
                    // once dg has left it
                    if (lane == 0) bulk_wait_group_read0();
                    __syncwarp();
                    uint32_t wh_[16];
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint32_t r[16], wg_[8], wu_[8], gw[8], uw[8];  // gw, uw: this row's 16-bit pairs, or four words of bytes
                        const bool some = args.keep == KEEP_8 ? half == 0 : col + half * 16 < args.N;  // a piece begins
                        if (some && !dead) dead = !wait_kept();
                        const unsigned char* at = kept + lane * 32;
                        if (args.keep == KEEP_8) {
                            const uint4 a = *reinterpret_cast<const uint4*>(at + 16 * half);
                            const uint4 b = *reinterpret_cast<const uint4*>(at + 1024 + 16 * half);
                            gw[0] = a.x, gw[1] = a.y, gw[2] = a.z, gw[3] = a.w;
                            uw[0] = b.x, uw[1] = b.y, uw[2] = b.z, uw[3] = b.w;
                        } else {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const uint4 a = *reinterpret_cast<const uint4*>(at + 16 * i);
                                const uint4 b = *reinterpret_cast<const uint4*>(at + 1024 + 16 * i);
                                gw[4 * i] = a.x, gw[4 * i + 1] = a.y, gw[4 * i + 2] = a.z, gw[4 * i + 3] = a.w;
                                uw[4 * i] = b.x, uw[4 * i + 1] = b.y, uw[4 * i + 2] = b.z, uw[4 * i + 3] = b.w;
                            }
                        }
                        if (!dead && (args.keep == KEEP_8 ? half == 1 : some)) fetch_kept();
                        tmem_ld16(tbase + c * 32 + half * 16, r);
                        tmem_wait_ld();
                        auto two = [&](int q, Float2 g, Float2 u) {  // elements 2q, 2q + 1
                            Float2 d;
                            const Float2 dh = join2(__uint_as_float(r[2 * q]), __uint_as_float(r[2 * q + 1]));
                            const Float2 a = glu_act2<ACT, true>(g, d);
                            const float2 dg = split2(pair_mul(pair_mul(dh, u), d)), du = split2(pair_mul(dh, a));
                            const float2 h = split2(pair_mul(a, u));
                            wg_[q] = pack16x2<DT>(dg.x, dg.y);
                            wu_[q] = pack16x2<DT>(du.x, du.y);
                            wh_[half * 8 + q] = pack16x2<DT>(h.x, h.y);
                        };
                        if (args.keep == KEEP_8) {
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                const uint32_t sh = 16 * (q & 1);
                                const float2 g = __half22float2(fp8_half2(gw[q >> 1] >> sh)), u = __half22float2(fp8_half2(uw[q >> 1] >> sh));
                                two(q, pair_mul(join2(g.x, g.y), gs2), pair_mul(join2(u.x, u.y), us2));
                            }
                        } else {
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                const float2 g = unpack16x2<DT>(gw[q]), u = unpack16x2<DT>(uw[q]);
                                two(q, join2(g.x, g.y), join2(u.x, u.y));
                            }
                        }
                        stage16(sbuf, lane, half, wg_);
                        stage16(sbuf + 2048, lane, half, wu_);
                    }
                    if (dead) break;
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmC, sbuf, col, row0);
                        bulk_commit_group();
                        tma_store_2d(&tmC2, sbuf + 2048, col, row0);
                        bulk_commit_group();
                        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                    }
                    __syncwarp();
                    stage32(sbuf, lane, wh_);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&tmC3, sbuf, col, row0);
                        bulk_commit_group();
                    }
                }
            }
            if (EPI == P_DGRAD && dead) break;
            // this accumulator back to the leader's MMA warp
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tempty_leader[acc]);
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        if constexpr (EPI == P_DGRAD)  // left early: what is under way lands first
            if (k_due) (void)mbar_wait_bounded(kbar, k_phase);
        if (lane == 0) bulk_wait_group0();
        __syncwarp();
    }
    // neither CTA leaves while the other can touch its shared or tensor memory
    tc_fence_before();
    cluster_sync();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// ------------------------------------------------------------------ host ----
struct Operand {
    const void* p;
    long long ld;
};

// Map of a 16-bit operand [rows][K] (K-major) or [K][rows] (MN-major): boxes of
// 64 k x 128 rows, or 64 rows x 64 k.
int operand_map(CUtensorMap* m, const Operand& o, bool mn, long long rows, long long K) {
    const auto t = CU_TENSOR_MAP_DATA_TYPE_UINT16;
    const auto sw = CU_TENSOR_MAP_SWIZZLE_128B;
    return mn ? tmap_2d(m, t, 2, o.p, rows, K, o.ld, 64, P_BK, sw) : tmap_2d(m, t, 2, o.p, K, rows, o.ld, P_BK, 128, sw);
}
int store_map(CUtensorMap* m, const void* p, long long rows, long long cols, long long ld) {
    return tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p, cols, rows, ld, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}

// Maps of g or u as kept: UP writes 32 columns of 32 rows, DGRAD reads 32 bytes of them.
int kept_map(CUtensorMap* m, int keep, const void* p, long long T, long long F, long long ldk, bool read) {
    if (keep == KEEP_8) return tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p, F, T, ldk, 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE);
    return read ? tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p, F, T, ldk, 16, 32, CU_TENSOR_MAP_SWIZZLE_NONE)
                : store_map(m, p, T, F, ldk);
}

bool operand_ok(const void* p, long long ld) { return aligned16(p) && ld % 8 == 0; }

template <int DT, bool A_MN, bool B_MN, int EPI, int ACT>
int launch_pair(const CUtensorMap (&m)[9], const PairArgs& args, cudaStream_t st) {
    auto k = pair_kernel<DT, A_MN, B_MN, EPI, ACT>;
    constexpr int smem = p_smem<EPI>();
    static SmemOnce once;
    SFFN_CUDA_TRY(once.set(k, smem));
    static const int pairs = resident_pairs(k, p_threads<EPI>(), smem);
    const long long tasks = (long long)((args.tiles_m + 1) / 2) * args.tiles_n * args.splits;
    const int clusters = (int)std::min<long long>(tasks, pairs);
    k<<<clusters * 2, p_threads<EPI>(), smem, st>>>(m[0], m[1], m[2], m[3], m[4], m[5], m[6], m[7], m[8], args);
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

// How many parts K is split into; a k-block of a pair takes about 0.27 us.
int split16(long long M, long long N, long long nkb) { return split_of(M, N, nkb, 1, 0.27); }
long long kblocks(long long K) { return (K + P_BK - 1) / P_BK; }

bool sizes_ok(long long M, long long N, long long K) {
    const long long most = 0x7FFFFF00;
    return M <= most && N <= most && K <= most && tiles_of(M, N) <= 0x1FFFFFF;
}

template <int DT>
int gemm16(const Operand& A, bool a_mn, const Operand& B, bool b_mn, const Operand& A2, const Operand& B2, long long K2,
           long long M, long long N, long long K, void* C, long long ldc, void* ws, size_t ws_bytes, uint32_t* status,
           cudaStream_t st) {
    PairArgs a{};
    a.M = (int)M;
    a.N = (int)N;
    a.tiles_m = (int)((M + 127) / 128);
    a.tiles_n = (int)((N + 255) / 256);
    a.nkb1 = (int)kblocks(K);
    a.nkb = a.nkb1 + (K2 ? (int)kblocks(K2) : 0);
    a.splits = split16(M, N, a.nkb);
    a.ldp = part_ld(N);
    if (a.splits > 1 && (!ws || ws_bytes < (size_t)a.splits * (size_t)M * (size_t)a.ldp * 4)) return SFFN_ERR_WORKSPACE;
    a.per_split = (a.nkb + a.splits - 1) / a.splits;
    a.part = static_cast<float*>(ws);
    a.out = static_cast<uint16_t*>(C);
    a.ldc = ldc;
    a.vec_out = aligned16(C) && ldc % 8 == 0;
    a.status = status;
    CUtensorMap m[9];
    memset(m, 0, sizeof(m));
    if (int rc = operand_map(&m[0], A, a_mn, M, K)) return rc;
    if (int rc = operand_map(&m[1], B, b_mn, N, K)) return rc;
    if (K2) {
        if (int rc = operand_map(&m[2], A2, a_mn, M, K2)) return rc;
        if (int rc = operand_map(&m[3], B2, b_mn, N, K2)) return rc;
    }
    if (a.vec_out && a.splits == 1)
        if (int rc = store_map(&m[4], C, M, N, ldc)) return rc;
    int rc = !a_mn && !b_mn ? launch_pair<DT, false, false, P_STORE, 0>(m, a, st)
             : !a_mn        ? launch_pair<DT, false, true, P_STORE, 0>(m, a, st)
             : b_mn         ? launch_pair<DT, true, true, P_STORE, 0>(m, a, st)
                            : launch_pair<DT, true, false, P_STORE, 0>(m, a, st);
    if (rc || a.splits == 1) return rc;
    return join_parts<DT>(a.part, a.splits, M, (int)N, C, ldc, st);
}

template <int DT, int EPI, bool B_MN>
int launch_act(int act, const CUtensorMap (&m)[9], const PairArgs& a, cudaStream_t st) {
    switch (act) {
        case GLU_RELU: return launch_pair<DT, false, B_MN, EPI, GLU_RELU>(m, a, st);
        case GLU_RELU2: return launch_pair<DT, false, B_MN, EPI, GLU_RELU2>(m, a, st);
        case GLU_SILU: return launch_pair<DT, false, B_MN, EPI, GLU_SILU>(m, a, st);
        default: return launch_pair<DT, false, B_MN, EPI, GLU_GELU>(m, a, st);
    }
}

// Arguments the two fused products share; F columns of h, D of x and y.
int check_glu(int dtype, int act, int keep, long long T, long long D, long long F, const void* g, const void* u, long long ldk,
              const void* gs, const void* us, const void* status) {
    if (dtype != SFFN_BF16 && dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (act < GLU_RELU || act > GLU_GELU || keep < KEEP_NONE || keep > KEEP_8 || T < 0 || D <= 0 || F <= 0 || !status)
        return SFFN_ERR_ARG;
    if (!sizes_ok(T, F, D) || T * fp8_block_tiles(F) > 0x7FFFFFFF) return SFFN_ERR_TOO_LARGE;
    if (keep == KEEP_NONE) return SFFN_OK;
    if (!g || !u || ldk < F || (keep == KEEP_8 && (!gs || !us))) return SFFN_ERR_ARG;
    if (!aligned16(g) || !aligned16(u) || ldk % (keep == KEEP_8 ? 16 : 8)) return SFFN_ERR_ALIGN;
    return SFFN_OK;
}

PairArgs glu_args(long long T, long long F, long long D, int tile_n, int keep, const void* gs, const void* us, uint32_t* status) {
    PairArgs a{};
    a.M = (int)T;
    a.N = (int)F;
    a.tiles_m = (int)((T + 127) / 128);
    a.tiles_n = (int)((F + tile_n - 1) / tile_n);
    a.nkb = a.nkb1 = a.per_split = (int)kblocks(D);
    a.splits = 1;
    a.keep = keep;
    a.gs = static_cast<uint8_t*>(const_cast<void*>(gs));
    a.us = static_cast<uint8_t*>(const_cast<void*>(us));
    a.bt = (int)fp8_block_tiles(F);
    a.status = status;
    return a;
}

}  // namespace
}  // namespace sffn

using namespace sffn;

extern "C" size_t sffn_gemm16_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t K2) {
    if (M <= 0 || N <= 0 || K <= 0 || K2 < 0 || !sizes_ok(M, N, K) || !sizes_ok(M, N, K2)) return 0;
    const int s = split16(M, N, kblocks(K) + (K2 ? kblocks(K2) : 0));
    return s > 1 ? (size_t)s * (size_t)M * (size_t)part_ld(N) * 4 : 0;
}

extern "C" int sffn_gemm16(int dtype, const void* A, int64_t lda, int a_mn, const void* B, int64_t ldb, int b_mn,
                           const void* A2, int64_t lda2, const void* B2, int64_t ldb2, int64_t K2, int64_t M, int64_t N,
                           int64_t K, void* C, int64_t ldc, void* workspace, size_t workspace_bytes, uint32_t* status_dev,
                           void* stream) {
    if (dtype != SFFN_BF16 && dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (M < 0 || N < 0 || K <= 0 || K2 < 0 || !status_dev) return SFFN_ERR_ARG;
    if (M == 0 || N == 0) return SFFN_OK;
    if (!sizes_ok(M, N, K) || !sizes_ok(M, N, K2)) return SFFN_ERR_TOO_LARGE;
    if (!A || !B || !C || ldc < N || lda < (a_mn ? M : K) || ldb < (b_mn ? N : K) ||
        (K2 && (!A2 || !B2 || lda2 < (a_mn ? M : K2) || ldb2 < (b_mn ? N : K2))))
        return SFFN_ERR_ARG;
    if (!operand_ok(A, lda) || !operand_ok(B, ldb) || (K2 && (!operand_ok(A2, lda2) || !operand_ok(B2, ldb2))) ||
        reinterpret_cast<uintptr_t>(C) % 2 || (workspace && !aligned16(workspace)))
        return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(A)) return rc;
    if (!sm100_sms()) return SFFN_ERR_DEVICE;
    const Operand a{A, lda}, b{B, ldb}, a2{A2, lda2}, b2{B2, ldb2};
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return dtype == SFFN_BF16
               ? gemm16<SFFN_BF16>(a, a_mn != 0, b, b_mn != 0, a2, b2, K2, M, N, K, C, ldc, workspace, workspace_bytes, status_dev, st)
               : gemm16<SFFN_F16>(a, a_mn != 0, b, b_mn != 0, a2, b2, K2, M, N, K, C, ldc, workspace, workspace_bytes, status_dev, st);
}

extern "C" int sffn_glu_up(int dtype, int act, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu,
                           int64_t ldwu, int64_t T, int64_t D, int64_t F, void* h, int64_t ldh, int keep, void* g, void* u,
                           int64_t ldk, void* g_scales, void* u_scales, uint32_t* status_dev, void* stream) {
    if (int rc = check_glu(dtype, act, keep, T, D, F, g, u, ldk, g_scales, u_scales, status_dev)) return rc;
    if (T == 0) return SFFN_OK;
    if (!x || !wg || !wu || !h || ldx < D || ldwg < D || ldwu < D || ldh < F) return SFFN_ERR_ARG;
    if (!operand_ok(x, ldx) || !operand_ok(wg, ldwg) || !operand_ok(wu, ldwu) || !operand_ok(h, ldh))
        return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(x)) return rc;
    if (!sm100_sms()) return SFFN_ERR_DEVICE;
    const PairArgs a = glu_args(T, F, D, 128, keep, g_scales, u_scales, status_dev);
    CUtensorMap m[9];
    memset(m, 0, sizeof(m));
    if (int rc = operand_map(&m[0], {x, ldx}, false, T, D)) return rc;
    if (int rc = operand_map(&m[1], {wg, ldwg}, false, F, D)) return rc;
    if (int rc = operand_map(&m[3], {wu, ldwu}, false, F, D)) return rc;
    if (int rc = store_map(&m[4], h, T, F, ldh)) return rc;
    if (keep != KEEP_NONE) {
        if (int rc = kept_map(&m[7], keep, g, T, F, ldk, false)) return rc;
        if (int rc = kept_map(&m[8], keep, u, T, F, ldk, false)) return rc;
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return dtype == SFFN_BF16 ? launch_act<SFFN_BF16, P_UP, false>(act, m, a, st)
                              : launch_act<SFFN_F16, P_UP, false>(act, m, a, st);
}

extern "C" int sffn_glu_dgrad(int dtype, int act, const void* dy, int64_t lddy, const void* w2, int64_t ldw2, int64_t T,
                              int64_t D, int64_t F, int keep, const void* g, const void* u, int64_t ldk,
                              const void* g_scales, const void* u_scales, void* dg, void* du, int64_t ldd, void* h,
                              int64_t ldh, uint32_t* status_dev, void* stream) {
    if (keep == KEEP_NONE) return SFFN_ERR_ARG;
    if (int rc = check_glu(dtype, act, keep, T, D, F, g, u, ldk, g_scales, u_scales, status_dev)) return rc;
    if (T == 0) return SFFN_OK;
    if (!dy || !w2 || !dg || !du || !h || lddy < D || ldw2 < F || ldd < F || ldh < F) return SFFN_ERR_ARG;
    if (!operand_ok(dy, lddy) || !operand_ok(w2, ldw2) || !operand_ok(dg, ldd) || !operand_ok(du, ldd) ||
        !operand_ok(h, ldh))
        return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(dy)) return rc;
    if (!sm100_sms()) return SFFN_ERR_DEVICE;
    const PairArgs a = glu_args(T, F, D, 256, keep, g_scales, u_scales, status_dev);
    CUtensorMap m[9];
    memset(m, 0, sizeof(m));
    if (int rc = operand_map(&m[0], {dy, lddy}, false, T, D)) return rc;
    if (int rc = operand_map(&m[1], {w2, ldw2}, true, F, D)) return rc;
    if (int rc = store_map(&m[4], dg, T, F, ldd)) return rc;
    if (int rc = store_map(&m[5], du, T, F, ldd)) return rc;
    if (int rc = store_map(&m[6], h, T, F, ldh)) return rc;
    if (int rc = kept_map(&m[7], keep, g, T, F, ldk, true)) return rc;
    if (int rc = kept_map(&m[8], keep, u, T, F, ldk, true)) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return dtype == SFFN_BF16 ? launch_act<SFFN_BF16, P_DGRAD, true>(act, m, a, st)
                              : launch_act<SFFN_F16, P_DGRAD, true>(act, m, a, st);
}
