// The gated feed-forward block h = act(x Wg^T) * (x Wu^T), y = h W2^T, and the
// products of its backward, in bfloat16 or float16 on the tcgen05 tensor cores.
//
// One kernel: CTA pairs (tcgen05.mma.cta_group::2, 256 x 256 tiles, float32
// accumulation in tensor memory, two accumulators), persistent over tiles;
// operands by TMA in a ring of 64-wide k-blocks, either major order, so no
// operand is transposed.
//   warps 0,2 / 3,12  issuers of A / B (even / odd k-blocks)
//   warp 1            MMA issuer (leader CTA)
//   warp 2            also tensor memory
//   warps 4-11        epilogue, two warpgroups; thread = accumulator row
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
constexpr int P_THREADS = 416;
constexpr int P_OPERAND = 128 * P_BK * 2;  // bytes of one operand a stage and CTA
constexpr int P_STAGE = 2 * P_OPERAND;
// The fused epilogues store three matrices instead of one and have more staging
// buffers a warp; their operand rings have four stages to make room.  Even
// counts: the issuers take alternate k-blocks.
template <int EPI>
constexpr int p_stages() { return EPI == P_STORE ? 6 : 4; }
template <int EPI>
constexpr int p_bufs() { return EPI == P_STORE ? 2 : EPI == P_UP ? 5 : 4; }
constexpr int P_KEPT = 4096;  // DGRAD: a warp's 32 x 32 of g and of u as kept
template <int EPI>
constexpr int p_smem() { return p_stages<EPI>() * P_STAGE + 8 * (p_bufs<EPI>() * 2048 + (EPI == P_DGRAD ? P_KEPT : 0)) + 1024; }
static_assert(p_smem<P_STORE>() <= 227 * 1024 - 1024 && p_smem<P_UP>() <= 227 * 1024 - 6144 &&
              p_smem<P_DGRAD>() <= 227 * 1024 - 1024, "shared memory");

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
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmA2, const __grid_constant__ CUtensorMap tmB2,
                const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmC2,
                const __grid_constant__ CUtensorMap tmC3, const __grid_constant__ CUtensorMap tmG,
                const __grid_constant__ CUtensorMap tmU, const PairArgs args) {
    constexpr int NST = p_stages<EPI>();
    constexpr uint32_t IDESC = idesc16<DT>(A_MN, B_MN);
    constexpr uint32_t MN_LBO = P_BK * 128;  // MN-major: 64-element blocks of 64 K rows x 128 bytes
    constexpr int TILE_N = EPI == P_UP ? 128 : 256;
    extern __shared__ __align__(1024) unsigned char p_smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p_smem_raw) + 1023) &
                                                           ~static_cast<uintptr_t>(1023));
    __shared__ __align__(8) uint64_t full_bar[NST], empty_bar[NST];
    __shared__ __align__(8) uint64_t tfull_bar[2], tempty_bar[2];
    __shared__ __align__(8) uint64_t kept_bar[8][2];  // DGRAD: each epilogue warp's g and u have come
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_dead;
    __shared__ uint2 s_amax[EPI == P_UP ? 2 : 1][2][128];  // UP: [tile parity][warpgroup][row], of g and u

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
            mbar_init(&tempty_bar[a], 16);  // the epilogue warps of both CTAs
        }
        for (int w = 0; w < 16; ++w) mbar_init(&kept_bar[w >> 1][w & 1], 1);
        s_abort = s_dead = 0;
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

    if (warp == 0 || warp == 2 || warp == 3 || warp == 12) {
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
    } else if (warp >= 4 && warp < 12) {
        // ------------------------------------------------------ epilogue --
        const int wg = (warp - 4) >> 2, ew = warp & 3;
        unsigned char* sbuf = smem + NST * P_STAGE + (warp - 4) * (p_bufs<EPI>() * 2048);
        StageRing<p_bufs<EPI>()> ring(sbuf);
        const uint32_t tempty_leader[2] = {leader_smem_addr(&tempty_bar[0]), leader_smem_addr(&tempty_bar[1])};
        // DGRAD: 32 columns of g and u as kept come by TMA, one such chunk ahead in 16
        // bits and two in 8, across tiles (each lane's own loads, of 32 rows an
        // instruction, took half of the kernel's time)
        unsigned char* kept = smem + NST * P_STAGE + 8 * (p_bufs<EPI>() * 2048) + (warp - 4) * P_KEPT;
        uint64_t* kbar = kept_bar[warp - 4];
        const int slots = args.keep == KEEP_8 ? 2 : 1;
        const uint32_t kept_bytes = args.keep == KEEP_8 ? 1024u : 2048u;  // of one matrix
        int f_task = first_task, f_chunk = 0, k_slot = 0;  // the next chunk to fetch; the slot of the next one to read
        uint32_t k_phase = 0, k_due = 0;                   // a bit a slot: its phase; a fetch is under way
        auto fetch_kept = [&](int slot) {                  // what the slot held is in registers
            __syncwarp();
            while (f_task < ntasks) {
                int pm, tn, kb0, kb1;
                locate(f_task, pm, tn, kb0, kb1);
                const int row0 = (pm * 2 + (int)rank) * 128 + ew * 32, col = tn * TILE_N + wg * (TILE_N / 2) + f_chunk * 32;
                if (f_chunk < 4 && row0 < args.M && col < args.N) {
                    if (lane == 0) {
                        unsigned char* to = kept + slot * 2048;
                        mbar_arrive_expect_tx(&kbar[slot], 2 * kept_bytes);
                        tma_load_2d(to, &tmG, col, row0, &kbar[slot]);
                        tma_load_2d(to + kept_bytes, &tmU, col, row0, &kbar[slot]);
                    }
                    k_due |= 1u << slot;
                    ++f_chunk;
                    return;
                }
                f_task += task_stride;
                f_chunk = 0;
            }
        };
        if constexpr (EPI == P_DGRAD)
            for (int i = 0; i < slots; ++i) fetch_kept(i);
        int acc = 0, it = 0;
        uint32_t acc_phase = 0;
        for (int task = first_task; task < ntasks; task += task_stride, ++it) {
            int pm, tn, kb0, kb1;
            const int sp = locate(task, pm, tn, kb0, kb1);
            const int row0 = (pm * 2 + (int)rank) * 128 + ew * 32;  // first row of this warp
            const int row = row0 + lane;
            const bool row_ok = row < args.M;
            const int gcol0 = tn * TILE_N + wg * (TILE_N / 2);  // first column of this warpgroup
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
            // The epilogue warps meet below (UP keeping 8 bits): all of them go on or
            // none.  s_dead is theirs alone, written before the first barrier and
            // read between the two.
            if constexpr (EPI == P_UP) {
                if (args.keep == KEEP_8) {
                    if (dead && lane == 0) s_dead = 1;
                    named_bar_sync(1, 256);
                    dead = *reinterpret_cast<volatile int*>(&s_dead) != 0;
                    named_bar_sync(1, 256);
                }
            }
            if (dead) break;
            tc_fence_after();
            const uint32_t tbase = tmem_base + ((uint32_t)(ew * 32) << 16) + (uint32_t)(acc * 256 + wg * (TILE_N / 2));

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
                float gtop = 0.f, utop = 0.f;
                const bool warp_live = row0 < args.M;
#pragma unroll 1
                for (int c = 0; c < 2; ++c) {
                    const int col = gcol0 + c * 32;
                    if (!warp_live || col >= args.N) break;
                    uint32_t g[32], u[32], w[16];
                    tmem_ld32(tbase + c * 32, g);
                    tmem_ld32(tbase + 128 + c * 32, u);
                    tmem_wait_ld();
#pragma unroll
                    for (int q = 0; q < 16; ++q) {
                        Float2 unused;
                        const Float2 gp = join2(__uint_as_float(g[2 * q]), __uint_as_float(g[2 * q + 1]));
                        const Float2 up = join2(__uint_as_float(u[2 * q]), __uint_as_float(u[2 * q + 1]));
                        const float2 h = split2(pair_mul(glu_act2<ACT, false>(gp, unused), up));
                        w[q] = pack16x2<DT>(h.x, h.y);
                    }
                    ring.store(&tmC, lane, w, col, row0);
                    if (args.keep == KEEP_16) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) w[q] = pack16x2<DT>(__uint_as_float(g[2 * q]), __uint_as_float(g[2 * q + 1]));
                        ring.store(&tmG, lane, w, col, row0);
#pragma unroll
                        for (int q = 0; q < 16; ++q) w[q] = pack16x2<DT>(__uint_as_float(u[2 * q]), __uint_as_float(u[2 * q + 1]));
                        ring.store(&tmU, lane, w, col, row0);
                    } else if (args.keep == KEEP_8) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            gtop = fmaxf(gtop, fabsf(__uint_as_float(g[j])));  // NaN does not count
                            utop = fmaxf(utop, fabsf(__uint_as_float(u[j])));
                        }
                    }
                }
                if (args.keep == KEEP_8) {
                    uint32_t gmax = __float_as_uint(gtop), umax = __float_as_uint(utop);
                    // rare: infinities do not count either
                    const bool finite = !__any_sync(FULL, max(gmax, umax) >= 0x7F800000u);
                    if (!finite) {
                        gmax = umax = 0;
#pragma unroll 1
                        for (int c = 0; c < 2; ++c) {
                            uint32_t g[32], u[32];
                            tmem_ld32(tbase + c * 32, g);
                            tmem_ld32(tbase + 128 + c * 32, u);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                gmax = max(gmax, finite_mag(__uint_as_float(g[j])));
                                umax = max(umax, finite_mag(__uint_as_float(u[j])));
                            }
                        }
                    }
                    // the block of 128 columns spans both warpgroups (columns past N are zero)
                    s_amax[it & 1][wg][ew * 32 + lane] = make_uint2(gmax, umax);
                    named_bar_sync(1, 256);
                    const uint2 other = s_amax[it & 1][wg ^ 1][ew * 32 + lane];
                    const int ge = fp8_exponent(max(gmax, other.x)), ue = fp8_exponent(max(umax, other.y));
                    if (row_ok) {
                        const long long at = fp8_scale_at(row, tn, args.bt);
                        if (wg == 0) args.gs[at] = (uint8_t)(ge + 127);
                        else args.us[at] = (uint8_t)(ue + 127);
                    }
                    // 64 columns of g, then of u, a lane's 64 bytes as 32 16-bit values are
#pragma unroll 1
                    for (int m = 0; m < 2; ++m) {
                        if (!warp_live || gcol0 >= args.N) break;
                        const float inv = two_to(m ? -ue : -ge);
                        uint32_t w[16];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            uint32_t r[32];
                            tmem_ld32(tbase + m * 128 + c * 32, r);
                            tmem_wait_ld();
#pragma unroll
                            for (int q = 0; q < 8; ++q) {
                                const float v0 = __uint_as_float(r[4 * q]), v1 = __uint_as_float(r[4 * q + 1]);
                                const float v2 = __uint_as_float(r[4 * q + 2]), v3 = __uint_as_float(r[4 * q + 3]);
                                if (finite) {
                                    const Float2 s2 = join2(inv, inv);
                                    w[c * 8 + q] = fp8_four(pair_mul(join2(v0, v1), s2), pair_mul(join2(v2, v3), s2));
                                } else {
                                    w[c * 8 + q] = fp8_pack4<false>(v0, v1, v2, v3, inv);
                                }
                            }
                        }
                        ring.store(m ? &tmU : &tmG, lane, w, gcol0, row0);
                    }
                }
            } else {  // P_DGRAD
                const float gscale = scales_ahead.x, uscale = scales_ahead.y;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const int col = gcol0 + c * 32;
                    if (row0 >= args.M || col >= args.N) break;
                    if (!__all_sync(FULL, mbar_wait_bounded(&kbar[k_slot], (k_phase >> k_slot) & 1u))) {
                        if (lane == 0) atomicOr(args.status, SFFN_STATUS_WAIT_TIMEOUT);
                        dead = true;
                        break;
                    }
                    k_phase ^= 1u << k_slot;
                    k_due &= ~(1u << k_slot);
                    uint32_t gw[16], uw[16];  // this row's: 16-bit pairs, or 8 words of four bytes
                    if (args.keep == KEEP_8) {
                        const unsigned char* at = kept + k_slot * 2048 + lane * 32;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint4 a = *reinterpret_cast<const uint4*>(at + 16 * i);
                            const uint4 b = *reinterpret_cast<const uint4*>(at + 1024 + 16 * i);
                            gw[4 * i] = a.x, gw[4 * i + 1] = a.y, gw[4 * i + 2] = a.z, gw[4 * i + 3] = a.w;
                            uw[4 * i] = b.x, uw[4 * i + 1] = b.y, uw[4 * i + 2] = b.z, uw[4 * i + 3] = b.w;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const unsigned char* at = kept + lane * 64 + 16 * (i ^ ((lane >> 1) & 3));
                            const uint4 a = *reinterpret_cast<const uint4*>(at);
                            const uint4 b = *reinterpret_cast<const uint4*>(at + 2048);
                            gw[4 * i] = a.x, gw[4 * i + 1] = a.y, gw[4 * i + 2] = a.z, gw[4 * i + 3] = a.w;
                            uw[4 * i] = b.x, uw[4 * i + 1] = b.y, uw[4 * i + 2] = b.z, uw[4 * i + 3] = b.w;
                        }
                    }
                    fetch_kept(k_slot);
                    k_slot = slots == 2 ? k_slot ^ 1 : 0;
                    uint32_t r[32], wg_[16], wu_[16], wh_[16];
                    tmem_ld32(tbase + c * 32, r);
                    tmem_wait_ld();
                    auto two = [&](int q, Float2 g, Float2 u) {  // elements 2q, 2q + 1
                        Float2 d;
                        const Float2 dh = join2(__uint_as_float(r[2 * q]), __uint_as_float(r[2 * q + 1]));
                        const Float2 a = glu_act2<ACT, true>(g, d);
                        const float2 dg = split2(pair_mul(pair_mul(dh, u), d)), du = split2(pair_mul(dh, a));
                        const float2 h = split2(pair_mul(a, u));
                        wg_[q] = pack16x2<DT>(dg.x, dg.y);
                        wu_[q] = pack16x2<DT>(du.x, du.y);
                        wh_[q] = pack16x2<DT>(h.x, h.y);
                    };
                    if (args.keep == KEEP_8) {
                        const Float2 gs2 = join2(gscale, gscale), us2 = join2(uscale, uscale);
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            const uint32_t sh = 16 * (q & 1);
                            const float2 g = __half22float2(fp8_half2(gw[q >> 1] >> sh)), u = __half22float2(fp8_half2(uw[q >> 1] >> sh));
                            two(q, pair_mul(join2(g.x, g.y), gs2), pair_mul(join2(u.x, u.y), us2));
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            const float2 g = unpack16x2<DT>(gw[q]), u = unpack16x2<DT>(uw[q]);
                            two(q, join2(g.x, g.y), join2(u.x, u.y));
                        }
                    }
                    ring.store(&tmC, lane, wg_, col, row0);
                    ring.store(&tmC2, lane, wu_, col, row0);
                    ring.store(&tmC3, lane, wh_, col, row0);
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
            for (int i = 0; i < 2; ++i)
                if ((k_due >> i) & 1u) (void)mbar_wait_bounded(&kbar[i], (k_phase >> i) & 1u);
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

// Maps of g or u as kept, to write (UP) and to read (DGRAD): 64 bytes of 32 rows,
// or 32 bytes in 8 bits where DGRAD reads 32 columns.
int kept_map(CUtensorMap* m, int keep, const void* p, long long T, long long F, long long ldk, bool read) {
    if (keep == KEEP_16) return store_map(m, p, T, F, ldk);
    return tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p, F, T, ldk, read ? 32 : 64, 32,
                   read ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_64B);
}

bool operand_ok(const void* p, long long ld) { return aligned16(p) && ld % 8 == 0; }

template <int DT, bool A_MN, bool B_MN, int EPI, int ACT>
int launch_pair(const CUtensorMap (&m)[9], const PairArgs& args, cudaStream_t st) {
    auto k = pair_kernel<DT, A_MN, B_MN, EPI, ACT>;
    constexpr int smem = p_smem<EPI>();
    static SmemOnce once;
    SFFN_CUDA_TRY(once.set(k, smem));
    static const int pairs = resident_pairs(k, P_THREADS, smem);
    const long long tasks = (long long)((args.tiles_m + 1) / 2) * args.tiles_n * args.splits;
    const int clusters = (int)std::min<long long>(tasks, pairs);
    k<<<clusters * 2, P_THREADS, smem, st>>>(m[0], m[1], m[2], m[3], m[4], m[5], m[6], m[7], m[8], args);
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
