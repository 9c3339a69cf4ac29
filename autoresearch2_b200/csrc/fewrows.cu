// Products of few rows (single tokens, small batches) with long weights:
// out[T, N] = x[T, K] W[N, K]^T for T <= 16, in 16 bits or in the 8-bit block
// format, and the gated pair act(x Wg^T) * (x Wu^T); and the entry points, which go
// on to narrow.cu for up to 64 rows.
//
// Bound by reading the weights once.  A tensor-core tile of 128 or 256 rows of
// x would leave most multiprocessors without a tile; here the weights are the
// rows of mma.sync (m16n8k16, float32 accumulation) and the tokens its columns.
// Measured: 1 row through 4096 x 14336 and back in bfloat16 57 us, 6.2 TB/s, 16 rows
// 64; 1 x 14336 x 4096 in 8 bits 18.7 us, 3.1 TB/s (8-bit operands are converted
// for mma.sync: two conversions for four elements of W and of x, and x's
// again for every 16 rows of W; the instruction for e4m3 itself takes as long).
// A block a multiprocessor, up to 16 rows of W (of Wg and Wu) at a time:
//   warp 16       copies 1 KB of each of these rows and of x a stage, by one TMA box
//                 a matrix
//   warps 0-15    multiply, 128 bytes of the stage's rows each, eight warps on a
//                 stage and eight on the next
//   warps 17-19   add the warps' sums in a fixed order and store, meanwhile
// Tried and slower on 16 rows x (14336 x 4096) x 2: a bulk copy for each row (1 KB
// each: the copy engine's rate, 94 us), weights by each warp's own loads and x from
// L2 (its latency, and warps that drift apart fetch scattered 128-byte pieces:
// 69 us).  Groups have equally many rows, so that the last ones end together.  The k index
// within a piece is permuted, alike for W and x, so that a lane's fragments are
// 16 contiguous bytes of a row.
#include <cuda.h>
#include <string.h>

#include "act.cuh"
#include "fp8.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace sffn {
namespace {

constexpr int S_MAX_ROWS = 16;
constexpr int S_WARPS = 16;                // that multiply
constexpr int S_ADDERS = 3;                // that add and store
constexpr int S_THREADS = (S_WARPS + 1 + S_ADDERS) * 32;
enum { S_PLAIN = 0, S_GATED = 1 };

struct FewArgs {
    int T, N, K;
    const void* x;
    long long ldx;  // elements
    const void* w[2];
    long long ldw[2];
    const uint8_t* xs;  // scale tiles (8-bit operands)
    const uint8_t* ws;
    int bt;
    int per;  // rows of W a group
    uint16_t* out;
    long long ldo;
    uint32_t* status;
    bool after;  // the kernel before on the stream wrote x and lets this one start early
};

template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (DT == SFFN_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row from byte k on, element by element (zeros past its `bytes`): rows
// that are not on 16 bytes, and a row's last bytes.  Not by __ldg: x may be written by
// the kernel before while this one is already resident, which the read-only path
// does not allow (for the weights alone it gains nothing).
template <int ESIZE>
__device__ __forceinline__ uint4 load_piece(const uint8_t* row, long long k, long long bytes) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16 / ESIZE; ++i) {
        if (k + i * ESIZE < bytes) {
            const uint32_t v = ESIZE == 2 ? (uint32_t)reinterpret_cast<const uint16_t*>(row + k)[i] : (uint32_t)row[k + i];
            w[i * ESIZE / 4] |= v << (8 * (i * ESIZE % 4));
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A stage in shared memory: rows of 1 KB, 16 of each matrix, then NT * 8 of x (rows
// and tokens past the last one hold anything: their sums are not stored); 8-bit
// operands' scale bytes of its eight blocks, 16 rows' of W and NT * 8 of x.
constexpr int S_ROW = 1024, S_PIECE = 128;
template <bool FP8, int MATS, int NT>
struct FewStage {
    static constexpr int SCALES = (MATS * 16 + NT * 8) * S_ROW;  // where these are
    static constexpr int BYTES = SCALES + (FP8 ? 512 : 0);
    static constexpr int SUMS = S_WARPS * NT * 8 * (MATS * 16 + 1) * 4;
    static constexpr int FIT = (232448 - 1024 - SUMS) / BYTES;
    // An even count: each stage then belongs to one half of the warps, and a warp
    // has waited for every earlier use of the stage it waits for.  (Were the halves
    // to take turns, one could find the phase before last complete and take it for
    // its own, when copies land out of order.)
    static constexpr int DEPTH = FIT >= 8 ? 8 : FIT & ~1;
    static_assert(DEPTH >= 2, "stages");
};

// A lane's two vectors of a row's piece, from each half of 64 bytes.  Rows are 1 KB
// apart, so lanes of odd rows read the halves in the other order: a
// quarter-warp's eight then meet different banks.
__device__ __forceinline__ void load_halves(const unsigned char* row, int gid, uint4 (&v)[2]) {
    const int odd = gid & 1;
    const uint4 a = *reinterpret_cast<const uint4*>(row + odd * 64), b = *reinterpret_cast<const uint4*>(row + (odd ^ 1) * 64);
    v[0] = odd ? b : a;
    v[1] = odd ? a : b;
}

// DT: type of x and W (FP8: both in 8 bits) and OT of the output; NT tiles of 8
// tokens.
template <int DT, int OT, bool FP8, int MODE, int ACT, int NT, bool VEC>
__global__ void __launch_bounds__(S_THREADS, 1)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmW2,
                    const __grid_constant__ CUtensorMap tmX, const FewArgs a) {
    constexpr int MATS = MODE == S_GATED ? 2 : 1;
    constexpr int ROWS = MATS * 16;  // rows of sums
    constexpr int ESIZE = FP8 ? 1 : 2;
    using St = FewStage<FP8, MATS, NT>;
    constexpr int STAGE = St::BYTES, DEPTH = St::DEPTH;
    extern __shared__ __align__(128) unsigned char few_smem[];
    float* red = reinterpret_cast<float*>(few_smem + (VEC ? DEPTH * STAGE : 0));  // [S_WARPS][NT * 8][ROWS + 1]
    __shared__ __align__(8) uint64_t full_bar[DEPTH], empty_bar[DEPTH];  // a stage's rows have come; are read
    __shared__ __align__(8) uint64_t sums_bar, free_bar;                 // the warps' sums are written; are read
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gid = lane >> 2, tig = lane & 3;
    const long long bytes = (long long)a.K * ESIZE;
    const long long whole = bytes & ~15LL;  // copied; a row's last few bytes are read where they are multiplied
    const int chunks = (int)((bytes + S_ROW - 1) / S_ROW);
    const int groups = (a.N + a.per - 1) / a.per;
    if (threadIdx.x == 0) {
        for (int s = 0; s < DEPTH; ++s) {
            mbar_init(&full_bar[s], VEC && FP8 ? 1 + 32 : 1);  // the boxes' bytes; each lane's scales
            mbar_init(&empty_bar[s], S_WARPS / 2);
        }
        mbar_init(&sums_bar, S_WARPS);
        mbar_init(&free_bar, S_ADDERS);
        fence_mbar_init();
    }
    __syncthreads();
    grid_dependents_start();

    if (warp == S_WARPS) {
        // -------------------------------------------------------- copies --
        if constexpr (VEC) {
            const uint32_t count = (uint32_t)(a.per * MATS + a.T) * S_ROW;  // whole boxes: zeros past the edges
            // the scales of a stage's eight blocks: lane = half of them of a row of W or of x
            auto copy_scales = [&](const uint8_t* tiles, long long row, int c, int stage, int place) {
                const int block = c * 8 + (lane & 1) * 4;
                if (block < (int)fp8_blocks(a.K))
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(few_smem + stage * STAGE + St::SCALES) + place * 8 + (lane & 1) * 4),
                                 "l"(tiles + fp8_scale_at(row, block, a.bt))
                                 : "memory");
            };
            auto copy_w = [&](int group, int c, int stage) {
                if (lane == 0) {
                    unsigned char* to = few_smem + stage * STAGE;
                    mbar_arrive_expect_tx(&full_bar[stage], count);
                    tma_load_2d(to, &tmW, c * (S_ROW / 4), group * a.per, &full_bar[stage]);
                    if constexpr (MATS == 2) tma_load_2d(to + 16 * S_ROW, &tmW2, c * (S_ROW / 4), group * a.per, &full_bar[stage]);
                }
                if constexpr (FP8) copy_scales(a.ws, min(group * a.per + (lane >> 1), a.N - 1), c, stage, lane >> 1);
            };
            auto copy_x = [&](int c, int stage) {
                if (lane == 0) tma_load_2d(few_smem + stage * STAGE + ROWS * S_ROW, &tmX, c * (S_ROW / 4), 0, &full_bar[stage]);
                if constexpr (FP8) {
#pragma unroll
                    for (int i = 0; i < (NT + 1) / 2; ++i) {
                        const int t = i * 16 + (lane >> 1);
                        if (t < NT * 8) copy_scales(a.xs, min(t, a.T - 1), c, stage, 16 + t);
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full_bar[stage])) : "memory");
                }
            };
            // W into all stages while the kernel before may still be writing x
            int ahead = 0;
            for (int group = blockIdx.x; a.after && group < groups && ahead < DEPTH; group += gridDim.x)
                for (int c = 0; c < chunks && ahead < DEPTH; ++c) copy_w(group, c, ahead++);
            grid_dependency_wait();
            int stage = 0;
            uint32_t phase = 1;
            for (int group = blockIdx.x; group < groups; group += gridDim.x)
                for (int c = 0; c < chunks; ++c) {
                    if (ahead > 0) {
                        --ahead;
                    } else {
                        if (!__all_sync(FULL, mbar_wait_bounded(&empty_bar[stage], phase))) {
                            if (lane == 0) atomicOr(a.status, SFFN_STATUS_WAIT_TIMEOUT);
                            // no copy lands after the block has left
                            for (int s = 0; s < DEPTH; ++s) (void)mbar_wait_bounded(&full_bar[s], (s < stage ? phase : phase ^ 1u) ^ 1u);
                            return;
                        }
                        copy_w(group, c, stage);
                    }
                    copy_x(c, stage);
                    if constexpr (FP8) __syncwarp();
                    if (++stage == DEPTH) stage = 0, phase ^= 1u;
                }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
        return;
    }
    if (warp > S_WARPS) {
        // -------------------------------------------------------- adders --
        grid_dependency_wait();
        uint32_t phase = 0;
        for (int group = blockIdx.x; group < groups; group += gridDim.x, phase ^= 1u) {
            if (!__all_sync(FULL, mbar_wait_bounded(&sums_bar, phase))) {
                if (lane == 0) atomicOr(a.status, SFFN_STATUS_WAIT_TIMEOUT);
                return;
            }
            const int n0 = group * a.per, rows = min(a.per, a.N - n0);
            for (int i = (warp - S_WARPS - 1) * 32 + lane; i < 16 * a.T; i += S_ADDERS * 32) {
                const int t = i >> 4, r = i & 15;
                float sum[MATS];
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    float v[S_WARPS];
#pragma unroll
                    for (int w = 0; w < S_WARPS; ++w) v[w] = red[(w * (NT * 8) + t) * (ROWS + 1) + m * 16 + r];
#pragma unroll
                    for (int o = S_WARPS / 2; o > 0; o >>= 1)
#pragma unroll
                        for (int w = 0; w < o; ++w) v[w] += v[w + o];
                    sum[m] = v[0];
                }
                if (r < rows) {
                    float v = sum[0];
                    if constexpr (MODE == S_GATED) v = glu_act<ACT>(sum[0]) * sum[1];
                    a.out[(long long)t * a.ldo + n0 + r] = Elt<OT>::from_f(v);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&free_bar);
        }
        return;
    }

    // ------------------------------------------------------------ products --
    grid_dependency_wait();
    const uint8_t* xrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) xrow[t] = static_cast<const uint8_t*>(a.x) + (long long)min(t * 8 + gid, a.T - 1) * a.ldx * ESIZE;
    // row h * 8 + gid of a group (past the group's end: any, its sums are not stored)
    auto row_of = [&](int group, int h) { return (long long)min(group * a.per + h * 8 + gid, a.N - 1); };
    // this warp's stages: every other one of the block's, from warp / 8 on
    int it = 0;
    uint32_t free_phase = 1;  // the first use finds the sums' place free
    for (int group = blockIdx.x; group < groups; group += gridDim.x) {
        float acc[MATS][NT][4];
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][t][j] = 0.f;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c, ++it) {
            if ((it & 1) != (warp >> 3)) continue;
            const int stage = it % DEPTH;
            if constexpr (VEC) {
                if (!__all_sync(FULL, mbar_wait_bounded(&full_bar[stage], (uint32_t)(it / DEPTH) & 1u))) {
                    if (lane == 0) atomicOr(a.status, SFFN_STATUS_WAIT_TIMEOUT);
                    return;
                }
            }
            const int off = (warp & 7) * S_PIECE + tig * 16;  // of this lane's first vector in the rows
            const long long k = (long long)c * S_ROW + off;
            const unsigned char* slot = few_smem + stage * STAGE + gid * S_ROW + off;
            if ((long long)c * S_ROW + (warp & 7) * S_PIECE < bytes) {
                float part[FP8 ? NT : 1][4];
                if constexpr (FP8) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) part[t][j] = 0.f;
                }
                uint4 w[MATS][2][2], x[NT][2];  // [][half of the rows][half of the piece]
                auto direct = [&](const uint8_t* row, uint4(&v)[2]) {
                    v[0] = load_piece<ESIZE>(row, k, bytes);
                    v[1] = load_piece<ESIZE>(row, k + 64, bytes);
                };
                const bool ring = VEC && k + 80 <= whole;
#pragma unroll
                for (int m = 0; m < MATS; ++m)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (ring) load_halves(slot + (m * 16 + h * 8) * S_ROW, gid, w[m][h]);
                        else direct(static_cast<const uint8_t*>(a.w[m]) + row_of(group, h) * a.ldw[m] * ESIZE, w[m][h]);
                    }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (ring) load_halves(slot + (ROWS + t * 8) * S_ROW, gid, x[t]);
                    else direct(xrow[t], x[t]);
                }
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    if constexpr (!FP8) {
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int m = 0; m < MATS; ++m) {
                                const uint4 w0 = w[m][0][q], w1 = w[m][1][q], xv = x[t][q];
                                mma16816<DT>(acc[m][t], w0.x, w1.x, w0.y, w1.y, xv.x, xv.y);
                                mma16816<DT>(acc[m][t], w0.z, w1.z, w0.w, w1.w, xv.z, xv.w);
                            }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            auto halves = [&](const uint4& u, uint32_t& lo, uint32_t& hi) {
                                const uint32_t v = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
                                const __half2 l = fp8_half2(v), h = fp8_half2(v >> 16);
                                lo = *reinterpret_cast<const uint32_t*>(&l);
                                hi = *reinterpret_cast<const uint32_t*>(&h);
                            };
                            uint32_t w0l, w0h, w1l, w1h;
                            halves(w[0][0][q], w0l, w0h);
                            halves(w[0][1][q], w1l, w1h);
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                uint32_t xl, xh;
                                halves(x[t][q], xl, xh);
                                mma16816<SFFN_F16>(part[t], w0l, w1l, w0h, w1h, xl, xh);
                            }
                        }
                    }
                }
                if constexpr (FP8) {
                    // one block of 128: the sum of its products times its two scales
                    int we[2], xe[NT][2];
                    if constexpr (VEC) {
                        const unsigned char* at = few_smem + stage * STAGE + St::SCALES + (warp & 7);
#pragma unroll
                        for (int h = 0; h < 2; ++h) we[h] = at[(h * 8 + gid) * 8];
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int h = 0; h < 2; ++h) xe[t][h] = at[(16 + t * 8 + tig * 2 + h) * 8];
                    } else {
                        const int block = c * (S_WARPS / 2) + (warp & 7);
                        auto byte = [&](const uint8_t* p, long long row) { return (int)p[fp8_scale_at(row, block, a.bt)]; };
#pragma unroll
                        for (int h = 0; h < 2; ++h) we[h] = byte(a.ws, row_of(group, h));
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int h = 0; h < 2; ++h) xe[t][h] = byte(a.xs, min(t * 8 + tig * 2 + h, a.T - 1));
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int wb = we[j >> 1], xb = xe[t][j & 1], e = wb + xb - 127;  // 2^(e - 127)
                            if (e >= 1 && e <= 254 && max(wb, xb) < 255) {
                                acc[0][t][j] = fmaf(part[t][j], __uint_as_float((uint32_t)e << 23), acc[0][t][j]);
                            } else {  // in two factors: the product may be in a float's range all the same
                                const int f = e - 127, f1 = f >> 1;
                                const float s1 = max(wb, xb) == 255 ? __uint_as_float(0x7FFFFFFFu) : two_to(max(f1, -126));
                                acc[0][t][j] += part[t][j] * s1 * two_to(max(f - f1, -126));
                            }
                        }
                }
            }
            if constexpr (VEC) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty_bar[stage]);
            }
        }
        // this warp's sums, token x row of W, once the last ones are read
        if (!__all_sync(FULL, mbar_wait_bounded(&free_bar, free_phase))) {
            if (lane == 0) atomicOr(a.status, SFFN_STATUS_WAIT_TIMEOUT);
            return;
        }
        free_phase ^= 1u;
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    red[(warp * (NT * 8) + t * 8 + tig * 2 + (j & 1)) * (ROWS + 1) + m * 16 + (j >> 1) * 8 + gid] = acc[m][t][j];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sums_bar);
    }
}

template <int DT, int OT, bool FP8, int MODE, int ACT, int NT, bool VEC>
int launch_few_nt(FewArgs a, cudaStream_t st) {
    auto k = few_rows_kernel<DT, OT, FP8, MODE, ACT, NT, VEC>;
    constexpr int MATS = MODE == S_GATED ? 2 : 1;
    using St = FewStage<FP8, MATS, NT>;
    constexpr int smem = (VEC ? St::DEPTH * St::BYTES : 0) + St::SUMS;
    static_assert(smem <= 232448 - 1024, "shared memory");
    static SmemOnce once;
    SFFN_CUDA_TRY(once.set(k, smem));
    const int sms = sm100_sms();
    if (!sms) return SFFN_ERR_DEVICE;
    const long long rounds = ((a.N + 15) / 16 + sms - 1) / sms;
    a.per = (int)((a.N + sms * rounds - 1) / (sms * rounds));
    CUtensorMap m[3];
    memset(m, 0, sizeof(m));
    if constexpr (VEC) {  // rows as 4-byte elements, whole 16-byte vectors of them
        constexpr int ES = FP8 ? 1 : 2;
        const auto u32 = CU_TENSOR_MAP_DATA_TYPE_UINT32;
        const auto none = CU_TENSOR_MAP_SWIZZLE_NONE;
        const long long inner = (long long)a.K * ES / 16 * 4;
        if (inner) {
            for (int i = 0; i < MATS; ++i)
                if (int rc = tmap_2d(&m[i], u32, 4, a.w[i], inner, a.N, a.ldw[i] * ES / 4, S_ROW / 4, a.per, none)) return rc;
            if (int rc = tmap_2d(&m[2], u32, 4, a.x, inner, a.T, a.ldx * ES / 4, S_ROW / 4, a.T, none)) return rc;
        } else {
            return launch_few_nt<DT, OT, FP8, MODE, ACT, NT, false>(a, st);  // rows of less than 16 bytes
        }
    }
    const int groups = (a.N + a.per - 1) / a.per;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(groups < sms ? groups : sms);
    config.blockDim = dim3(S_THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = a.after ? 1 : 0;
    SFFN_CUDA_TRY(cudaLaunchKernelEx(&config, k, m[0], m[1], m[2], a));
    return SFFN_OK;
}

template <int DT, int OT, bool FP8, int MODE, int ACT, bool VEC>
int launch_few(const FewArgs& a, cudaStream_t st) {
    return a.T <= 8 ? launch_few_nt<DT, OT, FP8, MODE, ACT, 1, VEC>(a, st) : launch_few_nt<DT, OT, FP8, MODE, ACT, 2, VEC>(a, st);
}

template <int DT, bool VEC>
int launch_gated(int act, const FewArgs& a, cudaStream_t st) {
    switch (act) {
        case GLU_RELU: return launch_few<DT, DT, false, S_GATED, GLU_RELU, VEC>(a, st);
        case GLU_RELU2: return launch_few<DT, DT, false, S_GATED, GLU_RELU2, VEC>(a, st);
        case GLU_SILU: return launch_few<DT, DT, false, S_GATED, GLU_SILU, VEC>(a, st);
        default: return launch_few<DT, DT, false, S_GATED, GLU_GELU, VEC>(a, st);
    }
}

bool rows16(const void* p, long long ld, int esize) { return aligned16(p) && ld * esize % 16 == 0; }

int check_few(long long T, long long N, long long K) {
    if (T < 0 || N < 0 || K <= 0 || T > NARROW_MAX_ROWS) return SFFN_ERR_ARG;
    return N > 0x7FFFFF00 || K > 0x7FFFFF00 ? SFFN_ERR_TOO_LARGE : SFFN_OK;
}

}  // namespace
}  // namespace sffn

using namespace sffn;

namespace sffn {
namespace {
int few_mm(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t T, int64_t N, int64_t K, void* out,
           int64_t ldo, bool after, uint32_t* status_dev, cudaStream_t st, DeviceScope& scope) {
    if (dtype != SFFN_BF16 && dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (int rc = check_few(T, N, K)) return rc;
    if (T == 0 || N == 0) return SFFN_OK;
    if (!x || !w || !out || !status_dev || ldx < K || ldw < K || ldo < N) return SFFN_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 1) return SFFN_ERR_ALIGN;
    const bool vec = rows16(x, ldx, 2) && rows16(w, ldw, 2);
    if (T > S_MAX_ROWS && !vec) return SFFN_ERR_ALIGN;
    if (scope.device() < 0)
        if (int rc = scope.bind(x)) return rc;
    if (T > S_MAX_ROWS) return narrow_mm(dtype, x, ldx, w, ldw, T, N, K, out, ldo, after, status_dev, st);
    FewArgs a{};
    a.status = status_dev;
    a.T = (int)T, a.N = (int)N, a.K = (int)K;
    a.x = x, a.ldx = ldx;
    a.w[0] = w, a.ldw[0] = ldw;
    a.out = static_cast<uint16_t*>(out), a.ldo = ldo;
    a.after = after;
    if (dtype == SFFN_BF16)
        return vec ? launch_few<SFFN_BF16, SFFN_BF16, false, S_PLAIN, 0, true>(a, st)
                   : launch_few<SFFN_BF16, SFFN_BF16, false, S_PLAIN, 0, false>(a, st);
    return vec ? launch_few<SFFN_F16, SFFN_F16, false, S_PLAIN, 0, true>(a, st)
               : launch_few<SFFN_F16, SFFN_F16, false, S_PLAIN, 0, false>(a, st);
}

int few_glu(int dtype, int act, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
            int64_t T, int64_t D, int64_t F, void* h, int64_t ldh, uint32_t* status_dev, cudaStream_t st, DeviceScope& scope) {
    if (dtype != SFFN_BF16 && dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (int rc = check_few(T, F, D)) return rc;
    if (act < GLU_RELU || act > GLU_GELU) return SFFN_ERR_ARG;
    if (T == 0 || F == 0) return SFFN_OK;
    if (!x || !wg || !wu || !h || !status_dev || ldx < D || ldwg < D || ldwu < D || ldh < F) return SFFN_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(wg) | reinterpret_cast<uintptr_t>(wu) |
         reinterpret_cast<uintptr_t>(h)) & 1)
        return SFFN_ERR_ALIGN;
    const bool vec = rows16(x, ldx, 2) && rows16(wg, ldwg, 2) && rows16(wu, ldwu, 2);
    if (T > S_MAX_ROWS && !vec) return SFFN_ERR_ALIGN;
    if (scope.device() < 0)
        if (int rc = scope.bind(x)) return rc;
    if (T > S_MAX_ROWS) return narrow_glu(dtype, act, x, ldx, wg, ldwg, wu, ldwu, T, D, F, h, ldh, status_dev, st);
    FewArgs a{};
    a.status = status_dev;
    a.T = (int)T, a.N = (int)F, a.K = (int)D;
    a.x = x, a.ldx = ldx;
    a.w[0] = wg, a.ldw[0] = ldwg;
    a.w[1] = wu, a.ldw[1] = ldwu;
    a.out = static_cast<uint16_t*>(h), a.ldo = ldh;
    if (dtype == SFFN_BF16) return vec ? launch_gated<SFFN_BF16, true>(act, a, st) : launch_gated<SFFN_BF16, false>(act, a, st);
    return vec ? launch_gated<SFFN_F16, true>(act, a, st) : launch_gated<SFFN_F16, false>(act, a, st);
}
}  // namespace
}  // namespace sffn

extern "C" int sffn_few_rows_mm(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t T, int64_t N,
                                int64_t K, void* out, int64_t ldo, uint32_t* status_dev, void* stream) {
    DeviceScope scope;
    return few_mm(dtype, x, ldx, w, ldw, T, N, K, out, ldo, false, status_dev, reinterpret_cast<cudaStream_t>(stream), scope);
}

extern "C" int sffn_few_rows_ffn(int dtype, int act, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu,
                                 int64_t ldwu, const void* w2, int64_t ldw2, int64_t T, int64_t D, int64_t F, void* h,
                                 int64_t ldh, void* y, int64_t ldy, uint32_t* status_dev, void* stream) {
    if (T > S_MAX_ROWS && !(rows16(h, ldh, 2) && rows16(w2, ldw2, 2))) return SFFN_ERR_ALIGN;
    DeviceScope scope;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (int rc = few_glu(dtype, act, x, ldx, wg, ldwg, wu, ldwu, T, D, F, h, ldh, status_dev, st, scope)) return rc;
    return few_mm(dtype, h, ldh, w2, ldw2, T, D, F, y, ldy, T > 0 && F > 0, status_dev, st, scope);
}

extern "C" int sffn_few_rows_fp8(const void* x, int64_t ldx, const void* x_scales, const void* w, int64_t ldw,
                                 const void* w_scales, int64_t T, int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo,
                                 uint32_t* status_dev, void* stream) {
    return few_rows_fp8(x, ldx, x_scales, w, ldw, w_scales, T, N, K, out, out_dtype, ldo, false, status_dev, stream);
}

int sffn::few_rows_fp8(const void* x, int64_t ldx, const void* x_scales, const void* w, int64_t ldw, const void* w_scales,
                       int64_t T, int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo, bool after,
                       uint32_t* status_dev, void* stream) {
    if (out_dtype != SFFN_BF16 && out_dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (int rc = check_few(T, N, K)) return rc;
    if (T == 0 || N == 0) return SFFN_OK;
    if (!x || !x_scales || !w || !w_scales || !out || !status_dev || ldx < K || ldw < K || ldo < N) return SFFN_ERR_ARG;
    if (!rows16(x, ldx, 1) || !rows16(w, ldw, 1) || !aligned16(x_scales) || !aligned16(w_scales) ||
        reinterpret_cast<uintptr_t>(out) % 2)
        return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(x)) return rc;
    FewArgs a{};
    a.status = status_dev;
    a.T = (int)T, a.N = (int)N, a.K = (int)K;
    a.x = x, a.ldx = ldx;
    a.w[0] = w, a.ldw[0] = ldw;
    a.xs = static_cast<const uint8_t*>(x_scales), a.ws = static_cast<const uint8_t*>(w_scales);
    a.bt = (int)fp8_block_tiles(K);
    a.after = after;
    a.out = static_cast<uint16_t*>(out), a.ldo = ldo;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    // Nine rows and more of long weights, too: the second tile of 8 tokens costs conversions
    // (16 rows, us, here and there: 14336 x 4096 23.3 and 16.7, 8192 x 4096 14.6 and 12.7,
    // 65536 x 512 34.0 and 11.6, 1024 x 32768 24.6 and 18.6, but 4096 x 4096 8.8 and 9.1, 8192 x
    // 2048 9.5 and 10.1; of the 13 shapes timed the rule is wrong for 2048 x 16384, 13.8 and 15.7;
    // 8 rows of 14336 x 4096 18.8).
    if (T > S_MAX_ROWS || (T > 8 && N >= (1LL << 25) / K)) return narrow_fp8(x, ldx, x_scales, w, ldw, w_scales, T, N, K, out, out_dtype, ldo, after, status_dev, st);
    return out_dtype == SFFN_BF16 ? launch_few<SFFN_F16, SFFN_BF16, true, S_PLAIN, 0, true>(a, st)
                                  : launch_few<SFFN_F16, SFFN_F16, true, S_PLAIN, 0, true>(a, st);
}
