// Products of few rows (single tokens, small batches) with long weights:
// out[T, N] = x[T, K] W[N, K]^T for T <= 32, in 16 bits or in the 8-bit block
// format, and the gated pair act(x Wg^T) * (x Wu^T).
//
// Bound by reading the weights once.  A tensor-core tile of 128 or 256 rows of
// x would leave most multiprocessors without a tile; here the weights are the
// rows of mma.sync (m16n8k16, float32 accumulation) and the tokens its columns:
// a block takes 16 or 32 rows of W, its eight warps alternate 128-byte pieces
// of them, and add their sums in shared memory, in a fixed order.  The k index
// within a piece is permuted, alike for W and x, so that a lane's fragments are
// 16 contiguous bytes of its row and both are read straight into registers.
#include "act.cuh"
#include "fp8.cuh"

namespace sffn {
namespace {

constexpr int S_MAX_ROWS = 32;
constexpr int S_WARPS = 8;
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

// DT: type of x and W (FP8: both in 8 bits) and OT of the output; MT tiles of
// 16 weight rows (of each matrix), NT of 8 tokens.
template <int DT, int OT, bool FP8, int MODE, int ACT, int MT, int NT, bool VEC>
__global__ void __launch_bounds__(S_WARPS * 32) few_rows_kernel(const FewArgs a) {
    constexpr int MATS = MODE == S_GATED ? 2 : 1;
    constexpr int ROWS = MATS * MT * 16;  // rows of sums a block holds
    constexpr int ESIZE = FP8 ? 1 : 2;
    constexpr int PIECE = 128;  // bytes of a row a warp takes at a time: one block of 8-bit values, 64 16-bit ones
    __shared__ float red[S_WARPS][NT * 8][ROWS + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gid = lane >> 2, tig = lane & 3;
    const int n0 = blockIdx.x * (MT * 16);
    const long long bytes = (long long)a.K * ESIZE;
    float acc[MATS][MT][NT][4];
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[m][i][t][j] = 0.f;

    // rows past the end read the last one; their sums are not stored
    const uint8_t* wrow[MATS][MT][2];
    int wn[MT][2];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wn[i][h] = min(n0 + i * 16 + h * 8 + gid, a.N - 1);
#pragma unroll
            for (int m = 0; m < MATS; ++m)
                wrow[m][i][h] = static_cast<const uint8_t*>(a.w[m]) + (long long)wn[i][h] * a.ldw[m] * ESIZE;
        }
    const uint8_t* xrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) xrow[t] = static_cast<const uint8_t*>(a.x) + (long long)min(t * 8 + gid, a.T - 1) * a.ldx * ESIZE;

#pragma unroll(MATS * MT * NT <= 2 ? 4 : 2)
    for (long long k0 = (long long)warp * PIECE; k0 < bytes; k0 += S_WARPS * PIECE) {
        uint4 wv[MATS][MT][2][2], xv[NT][2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const long long k = k0 + p * 64 + tig * 16;
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) wv[m][i][h][p] = load_piece<VEC, ESIZE, true>(wrow[m][i][h], k, bytes);
#pragma unroll
            for (int t = 0; t < NT; ++t) xv[t][p] = load_piece<VEC, ESIZE, false>(xrow[t], k, bytes);
        }
        if constexpr (!FP8) {
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int m = 0; m < MATS; ++m)
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            const uint4 w0 = wv[m][i][0][p], w1 = wv[m][i][1][p], xb = xv[t][p];
                            mma16816<DT>(acc[m][i][t], w0.x, w1.x, w0.y, w1.y, xb.x, xb.y);
                            mma16816<DT>(acc[m][i][t], w0.z, w1.z, w0.w, w1.w, xb.z, xb.w);
                        }
        } else {
            // one block of 128: the sum of its products, then its two scales
            const int block = (int)(k0 >> 7);
            float part[MATS][MT][NT][4];
#pragma unroll
            for (int m = 0; m < MATS; ++m)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int j = 0; j < 4; ++j) part[m][i][t][j] = 0.f;
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t xb[NT][2];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const uint32_t v = q == 0 ? xv[t][p].x : q == 1 ? xv[t][p].y : q == 2 ? xv[t][p].z : xv[t][p].w;
                        const __half2 lo = fp8_half2(v), hi = fp8_half2(v >> 16);
                        xb[t][0] = *reinterpret_cast<const uint32_t*>(&lo);
                        xb[t][1] = *reinterpret_cast<const uint32_t*>(&hi);
                    }
#pragma unroll
                    for (int m = 0; m < MATS; ++m)
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            uint32_t wa[2][2];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint4 u = wv[m][i][h][p];
                                const uint32_t v = q == 0 ? u.x : q == 1 ? u.y : q == 2 ? u.z : u.w;
                                const __half2 lo = fp8_half2(v), hi = fp8_half2(v >> 16);
                                wa[h][0] = *reinterpret_cast<const uint32_t*>(&lo);
                                wa[h][1] = *reinterpret_cast<const uint32_t*>(&hi);
                            }
#pragma unroll
                            for (int t = 0; t < NT; ++t)
                                mma16816<SFFN_F16>(part[m][i][t], wa[0][0], wa[1][0], wa[0][1], wa[1][1], xb[t][0], xb[t][1]);
                        }
                }
            int we[MT][2], xe[NT][2];
            bool nan = false;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    we[i][h] = (int)scale_byte(a.ws, wn[i][h], block, a.bt);
                    nan |= we[i][h] == 255;
                }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    xe[t][h] = (int)scale_byte(a.xs, min(t * 8 + tig * 2 + h, a.T - 1), block, a.bt);
                    nan |= xe[t][h] == 255;
                }
            // 2^(ew + ex) in two factors: the exponent alone may leave the range
            // of a float where the product does not
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int wb = we[i][j >> 1], xb = xe[t][j & 1];
                        const int e = wb + xb - 254, e1 = e >> 1;
                        float s1 = two_to(max(e1, -126)), s2 = two_to(max(e - e1, -126));
                        if (nan && (wb == 255 || xb == 255)) s1 = __uint_as_float(0x7FFFFFFFu);
#pragma unroll
                        for (int m = 0; m < MATS; ++m) acc[m][i][t][j] += part[m][i][t][j] * s1 * s2;
                    }
        }
    }
    // sums of the warps: row of W x token
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    red[warp][t * 8 + tig * 2 + (j & 1)][(m * MT + i) * 16 + (j >> 1) * 8 + gid] = acc[m][i][t][j];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 16 * a.T; i += S_WARPS * 32) {
        const int t = i / (MT * 16), r = i % (MT * 16);
        float s[MATS];
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            s[m] = 0.f;
#pragma unroll
            for (int w = 0; w < S_WARPS; ++w) s[m] += red[w][t][m * MT * 16 + r];
        }
        if (n0 + r < a.N) {
            float v = s[0], unused;
            if constexpr (MODE == S_GATED) v = glu_act<ACT, false>(s[0], unused) * s[1];
            a.out[(long long)t * a.ldo + n0 + r] = Elt<OT>::from_f(v);
        }
    }
}

template <int DT, int OT, bool FP8, int MODE, int ACT, bool VEC>
int launch_few(const FewArgs& a, cudaStream_t st) {
    const int nt = a.T <= 8 ? 1 : a.T <= 16 ? 2 : 4;
    const int grid = (a.N + 15) / 16;
    constexpr int threads = S_WARPS * 32;
    if (nt == 1) few_rows_kernel<DT, OT, FP8, MODE, ACT, 1, 1, VEC><<<grid, threads, 0, st>>>(a);
    else if (nt == 2) few_rows_kernel<DT, OT, FP8, MODE, ACT, 1, 2, VEC><<<grid, threads, 0, st>>>(a);
    else few_rows_kernel<DT, OT, FP8, MODE, ACT, 1, 4, VEC><<<grid, threads, 0, st>>>(a);
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
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
    if (int rc = scope.bind_same(x, {w, out})) return rc;
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
    if (int rc = scope.bind_same(x, {wg, wu, h})) return rc;
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

extern "C" int sffn_few_rows_fp8(const void* x, int64_t ldx, const void* x_scales, const void* w, int64_t ldw,
                                 const void* w_scales, int64_t T, int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo,
                                 void* stream) {
    if (out_dtype != SFFN_BF16 && out_dtype != SFFN_F16) return SFFN_ERR_DTYPE;
    if (int rc = check_few(T, N, K)) return rc;
    if (T == 0 || N == 0) return SFFN_OK;
    if (!x || !x_scales || !w || !w_scales || !out || ldx < K || ldw < K || ldo < N) return SFFN_ERR_ARG;
    if (!rows16(x, ldx, 1) || !rows16(w, ldw, 1) || reinterpret_cast<uintptr_t>(out) % 2) return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind_same(x, {x_scales, w, w_scales, out})) return rc;
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
