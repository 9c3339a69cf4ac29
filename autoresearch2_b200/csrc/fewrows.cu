// Products of few rows (single tokens, small batches) with long weights:
// out[T, N] = x[T, K] W[N, K]^T for T <= 32, in 16 bits or in the 8-bit block
// format, and the gated pair act(x Wg^T) * (x Wu^T).
//
// Bound by reading the weights once.  A tensor-core tile of 128 or 256 rows of
// x would leave most multiprocessors without a tile; here the weights are the
// rows of mma.sync (m16n8k16, float32 accumulation) and the tokens its columns.
// One block a multiprocessor takes 16 rows of W at a time (of Wg and Wu each),
// all its 16 warps on them in alternate 128-byte pieces, and adds their sums in
// shared memory in a fixed order.  The whole multiprocessor on one group of rows
// keeps the groups short, so that the last ones end together.  Weights come by
// cp.async, 192 KB of them under way on a multiprocessor, across the ends of
// groups; a thread copies the very bytes it multiplies, so that only its own
// copies need waiting for.  The k index within a piece is permuted, alike for W
// and x, so that these are 16 contiguous bytes of a row.
#include "act.cuh"
#include "fp8.cuh"
#include "tmap.cuh"

namespace sffn {
namespace {

constexpr int S_MAX_ROWS = 32;
constexpr int S_WARPS = 16;
constexpr int S_PIECE = 128;  // bytes of a row a warp takes at a time: one block of 8-bit values, 64 16-bit ones
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
    uint16_t* out;
    long long ldo;
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

// 16 bytes of a row from byte k on (zeros past its `bytes`), aligned for VEC.
template <bool VEC, int ESIZE, bool STREAM>
__device__ __forceinline__ uint4 load_piece(const uint8_t* row, long long k, long long bytes) {
    if (VEC && k + 16 <= bytes) {
        const uint4* p = reinterpret_cast<const uint4*>(row + k);
        return STREAM ? __ldcs(p) : __ldg(p);
    }
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16 / ESIZE; ++i) {
        if (k + i * ESIZE < bytes) {
            const uint32_t v = ESIZE == 2 ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(row + k) + i) : (uint32_t)__ldg(row + k + i);
            w[i * ESIZE / 4] |= v << (8 * (i * ESIZE % 4));
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Byte of the scale tiles of one row, for every block.
__device__ __forceinline__ uint32_t scale_byte(const uint8_t* s, long long row, int block, int bt) {
    return __ldg(s + fp8_scale_at(row, block, bt));
}

// Pieces of the weights under way: 64 bytes a thread and matrix each.
template <int MATS, int NT>
constexpr int few_depth() { return MATS == 1 ? 6 : NT == 4 ? 2 : 3; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {  // zeros after `bytes`
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// DT: type of x and W (FP8: both in 8 bits) and OT of the output; NT tiles of 8
// tokens.
template <int DT, int OT, bool FP8, int MODE, int ACT, int NT, bool VEC>
__global__ void __launch_bounds__(S_WARPS * 32, 1) few_rows_kernel(const FewArgs a) {
    constexpr int MATS = MODE == S_GATED ? 2 : 1;
    constexpr int ROWS = MATS * 16;  // rows of sums
    constexpr int ESIZE = FP8 ? 1 : 2;
    constexpr int DEPTH = few_depth<MATS, NT>();
    constexpr int VECS = MATS * 4;  // 16-byte vectors of weights a thread takes of a piece
    extern __shared__ __align__(16) unsigned char few_smem[];
    // [DEPTH][VECS][threads] vectors, then [S_WARPS][NT * 8][ROWS + 1] sums
    uint4* ring = reinterpret_cast<uint4*>(few_smem);
    float* red = reinterpret_cast<float*>(few_smem + DEPTH * VECS * S_WARPS * 32 * 16);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gid = lane >> 2, tig = lane & 3;
    const long long bytes = (long long)a.K * ESIZE;
    const int pieces = (int)((bytes + S_PIECE - 1) / S_PIECE);
    const int mine = pieces > warp ? (pieces - warp + S_WARPS - 1) / S_WARPS : 0;
    const int groups = (a.N + 15) / 16;

    const uint8_t* xrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) xrow[t] = static_cast<const uint8_t*>(a.x) + (long long)min(t * 8 + gid, a.T - 1) * a.ldx * ESIZE;

    // the copies run DEPTH - 1 pieces ahead: of piece ci of group cg, into slot cs
    int cg = mine ? (int)blockIdx.x : groups, ci = 0, cs = 0;
    auto copy = [&] {
        if (cg < groups) {
            const long long k0 = ((long long)warp + (long long)ci * S_WARPS) * S_PIECE + tig * 16;
            uint4* slot = ring + (cs * VECS) * (S_WARPS * 32) + threadIdx.x;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // rows past the end read the last one; their sums are not stored
                const long long n = min(cg * 16 + h * 8 + gid, a.N - 1);
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    const uint8_t* row = static_cast<const uint8_t*>(a.w[m]) + n * a.ldw[m] * ESIZE;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint4* to = slot + ((m * 2 + h) * 2 + q) * (S_WARPS * 32);
                        const long long k = k0 + q * 64, left = bytes - k;
                        if constexpr (VEC)
                            cp_async16((uint32_t)__cvta_generic_to_shared(to), left > 0 ? row + k : row,
                                       left >= 16 ? 16u : left > 0 ? (uint32_t)left : 0u);
                        else
                            *to = load_piece<false, ESIZE, true>(row, k, bytes);
                    }
                }
            }
            if (++ci == mine) ci = 0, cg += gridDim.x;
            cs = cs + 1 == DEPTH ? 0 : cs + 1;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int slot_at = 0;

#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) copy();
    for (int group = blockIdx.x; group < groups; group += gridDim.x) {
        const int n0 = group * 16;
        float acc[MATS][NT][4];
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][t][j] = 0.f;
#pragma unroll 1
        for (int i = 0; i < mine; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 2) : "memory");
            uint4 w[MATS][2][2], x[2][NT];
            const long long xk = ((long long)warp + (long long)i * S_WARPS) * S_PIECE + tig * 16;
            if constexpr (FP8 || NT <= 2) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int t = 0; t < NT; ++t) x[q][t] = load_piece<VEC, ESIZE, false>(xrow[t], xk + q * 64, bytes);
            }
#pragma unroll
            for (int v = 0; v < VECS; ++v) w[v >> 2][(v >> 1) & 1][v & 1] = ring[(slot_at * VECS + v) * (S_WARPS * 32) + threadIdx.x];
            slot_at = slot_at + 1 == DEPTH ? 0 : slot_at + 1;
            copy();  // into the slot read in the last step
            if constexpr (!FP8) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if constexpr (NT > 2) x[q][t] = load_piece<VEC, ESIZE, false>(xrow[t], xk + q * 64, bytes);
#pragma unroll
                        for (int m = 0; m < MATS; ++m) {
                            const uint4 w0 = w[m][0][q], w1 = w[m][1][q], xb = x[q][t];
                            mma16816<DT>(acc[m][t], w0.x, w1.x, w0.y, w1.y, xb.x, xb.y);
                            mma16816<DT>(acc[m][t], w0.z, w1.z, w0.w, w1.w, xb.z, xb.w);
                        }
                    }
            } else {
                // one block of 128: the sum of its products, then its two scales
                const int block = warp + i * S_WARPS;
                int we[2], xe[NT][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) we[h] = (int)scale_byte(a.ws, min(n0 + h * 8 + gid, a.N - 1), block, a.bt);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) xe[t][h] = (int)scale_byte(a.xs, min(t * 8 + tig * 2 + h, a.T - 1), block, a.bt);
                float part[NT][4];
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) part[t][j] = 0.f;
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        auto halves = [&](const uint4& u, uint32_t& lo, uint32_t& hi) {
                            const uint32_t v = c == 0 ? u.x : c == 1 ? u.y : c == 2 ? u.z : u.w;
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
                            halves(x[q][t], xl, xh);
                            mma16816<SFFN_F16>(part[t], w0l, w1l, w0h, w1h, xl, xh);
                        }
                    }
                // 2^(ew + ex) in two factors: one of the scales may leave the range
                // of a float where the product of both does not
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int wb = we[j >> 1], xb = xe[t][j & 1];
                        const int e = wb + xb - 254, e1 = e >> 1;
                        float s1 = two_to(max(e1, -126));
                        const float s2 = two_to(max(e - e1, -126));
                        if (wb == 255 || xb == 255) s1 = __uint_as_float(0x7FFFFFFFu);
                        acc[0][t][j] += part[t][j] * s1 * s2;
                    }
            }
        }
        // the warps' sums, token x row of W
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    red[(warp * (NT * 8) + t * 8 + tig * 2 + (j & 1)) * (ROWS + 1) + m * 16 + (j >> 1) * 8 + gid] = acc[m][t][j];
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * a.T; i += S_WARPS * 32) {
            const int t = i >> 4, r = i & 15;
            float sum[MATS];
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                sum[m] = 0.f;
#pragma unroll
                for (int w = 0; w < S_WARPS; ++w) sum[m] += red[(w * (NT * 8) + t) * (ROWS + 1) + m * 16 + r];
            }
            if (n0 + r < a.N) {
                float v = sum[0], unused;
                if constexpr (MODE == S_GATED) v = glu_act<ACT, false>(sum[0], unused) * sum[1];
                a.out[(long long)t * a.ldo + n0 + r] = Elt<OT>::from_f(v);
            }
        }
        __syncthreads();
    }
}

template <int DT, int OT, bool FP8, int MODE, int ACT, int NT, bool VEC>
int launch_few_nt(const FewArgs& a, cudaStream_t st) {
    auto k = few_rows_kernel<DT, OT, FP8, MODE, ACT, NT, VEC>;
    constexpr int MATS = MODE == S_GATED ? 2 : 1;
    constexpr int smem = few_depth<MATS, NT>() * MATS * 4 * S_WARPS * 32 * 16 + S_WARPS * NT * 8 * (MATS * 16 + 1) * 4;
    static_assert(smem <= 232448, "shared memory");
    SFFN_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const int sms = sm100_sms();
    if (!sms) return SFFN_ERR_DEVICE;
    k<<<min((a.N + 15) / 16, sms), S_WARPS * 32, smem, st>>>(a);
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

template <int DT, int OT, bool FP8, int MODE, int ACT, bool VEC>
int launch_few(const FewArgs& a, cudaStream_t st) {
    return a.T <= 8    ? launch_few_nt<DT, OT, FP8, MODE, ACT, 1, VEC>(a, st)
           : a.T <= 16 ? launch_few_nt<DT, OT, FP8, MODE, ACT, 2, VEC>(a, st)
                       : launch_few_nt<DT, OT, FP8, MODE, ACT, 4, VEC>(a, st);
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
    if (T < 0 || N < 0 || K <= 0 || T > S_MAX_ROWS) return SFFN_ERR_ARG;
    return N > 0x7FFFFF00 || K > 0x7FFFFF00 ? SFFN_ERR_TOO_LARGE : SFFN_OK;
}

}  // namespace
}  // namespace sffn

using namespace sffn;

extern "C" int sffn_few_rows_mm(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t T, int64_t N,
                                int64_t K, void* out, int64_t ldo, void* stream) {
    if (dtype != SFFN_BF16 && dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (int rc = check_few(T, N, K)) return rc;
    if (T == 0 || N == 0) return SFFN_OK;
    if (!x || !w || !out || ldx < K || ldw < K || ldo < N) return SFFN_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(out)) & 1) return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(x)) return rc;
    FewArgs a{};
    a.T = (int)T, a.N = (int)N, a.K = (int)K;
    a.x = x, a.ldx = ldx;
    a.w[0] = w, a.ldw[0] = ldw;
    a.out = static_cast<uint16_t*>(out), a.ldo = ldo;
    const bool vec = rows16(x, ldx, 2) && rows16(w, ldw, 2);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == SFFN_BF16)
        return vec ? launch_few<SFFN_BF16, SFFN_BF16, false, S_PLAIN, 0, true>(a, st)
                   : launch_few<SFFN_BF16, SFFN_BF16, false, S_PLAIN, 0, false>(a, st);
    return vec ? launch_few<SFFN_F16, SFFN_F16, false, S_PLAIN, 0, true>(a, st)
               : launch_few<SFFN_F16, SFFN_F16, false, S_PLAIN, 0, false>(a, st);
}

extern "C" int sffn_few_rows_glu(int dtype, int act, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu,
                                 int64_t ldwu, int64_t T, int64_t D, int64_t F, void* h, int64_t ldh, void* stream) {
    if (dtype != SFFN_BF16 && dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (int rc = check_few(T, F, D)) return rc;
    if (act < GLU_RELU || act > GLU_GELU) return SFFN_ERR_ARG;
    if (T == 0 || F == 0) return SFFN_OK;
    if (!x || !wg || !wu || !h || ldx < D || ldwg < D || ldwu < D || ldh < F) return SFFN_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(wg) | reinterpret_cast<uintptr_t>(wu) |
         reinterpret_cast<uintptr_t>(h)) & 1)
        return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(x)) return rc;
    FewArgs a{};
    a.T = (int)T, a.N = (int)F, a.K = (int)D;
    a.x = x, a.ldx = ldx;
    a.w[0] = wg, a.ldw[0] = ldwg;
    a.w[1] = wu, a.ldw[1] = ldwu;
    a.out = static_cast<uint16_t*>(h), a.ldo = ldh;
    const bool vec = rows16(x, ldx, 2) && rows16(wg, ldwg, 2) && rows16(wu, ldwu, 2);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == SFFN_BF16) return vec ? launch_gated<SFFN_BF16, true>(act, a, st) : launch_gated<SFFN_BF16, false>(act, a, st);
    return vec ? launch_gated<SFFN_F16, true>(act, a, st) : launch_gated<SFFN_F16, false>(act, a, st);
}

extern "C" int sffn_few_rows_ffn(int dtype, int act, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu,
                                 int64_t ldwu, const void* w2, int64_t ldw2, int64_t T, int64_t D, int64_t F, void* h,
                                 int64_t ldh, void* y, int64_t ldy, void* stream) {
    if (int rc = sffn_few_rows_glu(dtype, act, x, ldx, wg, ldwg, wu, ldwu, T, D, F, h, ldh, stream)) return rc;
    return sffn_few_rows_mm(dtype, h, ldh, w2, ldw2, T, D, F, y, ldy, stream);
}

extern "C" int sffn_few_rows_fp8(const void* x, int64_t ldx, const void* x_scales, const void* w, int64_t ldw,
                                 const void* w_scales, int64_t T, int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo,
                                 void* stream) {
    if (out_dtype != SFFN_BF16 && out_dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (int rc = check_few(T, N, K)) return rc;
    if (T == 0 || N == 0) return SFFN_OK;
    if (!x || !x_scales || !w || !w_scales || !out || ldx < K || ldw < K || ldo < N) return SFFN_ERR_ARG;
    if (!rows16(x, ldx, 1) || !rows16(w, ldw, 1) || reinterpret_cast<uintptr_t>(out) % 2) return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(x)) return rc;
    FewArgs a{};
    a.T = (int)T, a.N = (int)N, a.K = (int)K;
    a.x = x, a.ldx = ldx;
    a.w[0] = w, a.ldw[0] = ldw;
    a.xs = static_cast<const uint8_t*>(x_scales), a.ws = static_cast<const uint8_t*>(w_scales);
    a.bt = (int)fp8_block_tiles(K);
    a.out = static_cast<uint16_t*>(out), a.ldo = ldo;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    return out_dtype == SFFN_BF16 ? launch_few<SFFN_F16, SFFN_BF16, true, S_PLAIN, 0, true>(a, st)
                                  : launch_few<SFFN_F16, SFFN_F16, true, S_PLAIN, 0, true>(a, st);
}
