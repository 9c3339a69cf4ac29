// Activations in the 8-bit block format (fp8.cuh): pack and unpack.
//
// Both are bound by memory: per element of a 16-bit tensor the pack reads two
// bytes and writes one (and 1/128), the unpack the reverse.  Eight lanes share
// a block of 128, 16 contiguous elements each: whole 16-byte loads and stores,
// the amax by three shuffles.  65536 x 4096 bfloat16: 129 us to pack and 133 to
// unpack, 6.3 and 6.1 TB/s, 96% and 93% of the copy rate.
#include "fp8.cuh"

namespace sffn {
namespace {

constexpr int Q_THREADS = 256;
constexpr int Q_GROUPS = Q_THREADS / 8;  // blocks of 128 a thread block takes

// 16 elements of a row, as they are stored.
template <int DT>
struct Sixteen {
    uint32_t w[DT == SFFN_F32 ? 16 : 8];

    // from column c on, zeros past the row's end
    template <bool VEC>
    __device__ __forceinline__ void load(const void* row, long long c, long long width) {
        using bits = typename Elt<DT>::bits;
        const bits* p = static_cast<const bits*>(row) + c;
        constexpr int N = sizeof(w) / 16;
        if (VEC && c + 16 <= width) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else if constexpr (DT == SFFN_F32) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = c + i < width ? p[i] : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                w[i] = (c + 2 * i < width ? (uint32_t)p[2 * i] : 0u) | (c + 2 * i + 1 < width ? (uint32_t)p[2 * i + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (DT == SFFN_F32) return __uint_as_float(w[i]);
        else return (i & 1) ? unpack16x2<DT>(w[i >> 1]).y : unpack16x2<DT>(w[i >> 1]).x;
    }
    // bits, as float32, of the largest magnitude, infinities and NaN included
    __device__ __forceinline__ uint32_t amax() const {
        uint32_t m = 0;
        if constexpr (DT == SFFN_F32) {
#pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
            return m;
        } else {  // magnitudes order as their bits do
#pragma unroll
            for (int i = 0; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
            return __float_as_uint(Elt<DT>::to_f((uint16_t)max(m & 0xFFFFu, m >> 16)));
        }
    }
    __device__ __forceinline__ uint32_t finite_amax() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, finite_mag(get(i)));
        return m;
    }
};

constexpr int Q_PER = 2;  // blocks a group of eight lanes takes

// Eight lanes a block; the groups run over padded rows x padded blocks (whole
// scale tiles), those of the padding write their scale byte, zero.  Each takes
// two blocks, whose loads are under way together.
template <int DT, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
    fp8_pack_kernel(const void* __restrict__ x, long long rows, long long width, long long ld, uint8_t* __restrict__ values,
                    long long ldv, uint8_t* __restrict__ scales, uint32_t blocks4, uint32_t groups) {
    grid_dependents_start();
    const int sub = threadIdx.x & 7;
    const unsigned lanes = 0xFFu << (threadIdx.x & 24);
    uint32_t row[Q_PER];
    int block[Q_PER];
    bool live[Q_PER], some[Q_PER];
    Sixteen<DT> v[Q_PER];
#pragma unroll
    for (int k = 0; k < Q_PER; ++k) {
        const uint32_t id = (blockIdx.x * (uint32_t)Q_PER + k) * Q_GROUPS + (threadIdx.x >> 3);
        row[k] = id / blocks4;
        block[k] = (int)(id - row[k] * blocks4);
        some[k] = id < groups;
        live[k] = some[k] && row[k] < rows && (long long)block[k] * FP8_BLOCK < width;
        if (live[k])
            v[k].template load<VEC>(static_cast<const typename Elt<DT>::bits*>(x) + (long long)row[k] * ld,
                                    (long long)block[k] * FP8_BLOCK + sub * 16, width);
    }
#pragma unroll
    for (int k = 0; k < Q_PER; ++k) {  // each branch is one of the eight lanes
        if (!some[k]) continue;
        uint8_t* scale = scales + fp8_scale_at(row[k], block[k], blocks4 >> 2);
        if (!live[k]) {
            if (sub == 0) *scale = 0;
            continue;
        }
        uint32_t amax = v[k].amax();
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(lanes, amax, o));
        const bool finite = amax < 0x7F800000u;
        if (!finite) {
            amax = v[k].finite_amax();
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(lanes, amax, o));
        }
        const int e = fp8_exponent(amax);
        if (sub == 0) *scale = (uint8_t)(e + 127);
        const long long c = (long long)block[k] * FP8_BLOCK + sub * 16;
        if (c >= width) continue;
        const float inv = two_to(-e);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[k].get(4 * i), b = v[k].get(4 * i + 1), d = v[k].get(4 * i + 2), f = v[k].get(4 * i + 3);
            w[i] = finite ? fp8_pack4<true>(a, b, d, f, inv) : fp8_pack4<false>(a, b, d, f, inv);
        }
        __stcs(reinterpret_cast<uint4*>(values + (long long)row[k] * ldv + c), make_uint4(w[0], w[1], w[2], w[3]));
    }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
    fp8_unpack_kernel(const uint8_t* __restrict__ values, long long ldv, const uint8_t* __restrict__ scales, long long rows,
                      long long width, void* __restrict__ out, long long ldo, uint32_t blocks, uint32_t groups) {
    using bits = typename Elt<DT>::bits;
    const uint32_t id = blockIdx.x * (uint32_t)Q_GROUPS + (threadIdx.x >> 3);
    const uint32_t row = id / blocks;
    const int block = (int)(id - row * blocks);
    const long long c = (long long)block * FP8_BLOCK + (threadIdx.x & 7) * 16;
    const bool live = id < groups && c < width;
    if (VEC && !live) return;
    uint4 v = make_uint4(0, 0, 0, 0);
    float s = 0.f;
    if (live) {
        v = __ldcs(reinterpret_cast<const uint4*>(values + (long long)row * ldv + c));
        s = fp8_scale(scales[fp8_scale_at(row, block, (blocks + 3) >> 2)]);
    }
    // A value beyond the type's largest finite one (its rounding to 8 bits may
    // have crossed that) becomes the largest; the last step of 8 bits is far
    // wider than the difference.
    const float most = DT == SFFN_F16 ? 65504.f : DT == SFFN_BF16 ? __uint_as_float(0x7F7F0000u) : __uint_as_float(0x7F7FFFFFu);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float q[4];
        fp8_unpack4(w[i], q);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float y = q[j] * s;
            f[4 * i + j] = y != y ? y : fminf(fmaxf(y, -most), most);
        }
    }
    bits* p = static_cast<bits*>(out) + (long long)row * ldo + c;
    if (VEC && c + 16 <= width) {
        uint4* q = reinterpret_cast<uint4*>(p);
        if constexpr (DT == SFFN_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                q[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                                  __float_as_uint(f[4 * i + 3]));
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                q[i] = make_uint4(pack16x2<DT>(f[8 * i], f[8 * i + 1]), pack16x2<DT>(f[8 * i + 2], f[8 * i + 3]),
                                  pack16x2<DT>(f[8 * i + 4], f[8 * i + 5]), pack16x2<DT>(f[8 * i + 6], f[8 * i + 7]));
        }
    } else if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (c + i < width) p[i] = Elt<DT>::from_f(f[i]);
    } else {
        // a warp's four blocks through shared memory: whole runs of 32 elements a store
        __shared__ bits buf[Q_THREADS / 32][4][FP8_BLOCK + 16 / sizeof(bits)];
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 16; ++i) buf[warp][lane >> 3][(lane & 7) * 16 + i] = Elt<DT>::from_f(f[i]);
        __syncwarp();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint32_t gid = blockIdx.x * (uint32_t)Q_GROUPS + warp * 4 + g;
            if (gid >= groups) break;
            const uint32_t r = gid / blocks;
            const long long c0 = (long long)(gid - r * blocks) * FP8_BLOCK;
            bits* q = static_cast<bits*>(out) + (long long)r * ldo + c0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c0 + j * 32 + lane < width) q[j * 32 + lane] = buf[warp][g][j * 32 + lane];
        }
    }
}

template <int DT>
int pack(const void* x, long long rows, long long width, long long ld, uint8_t* values, long long ldv, uint8_t* scales,
         cudaStream_t st) {
    const long long blocks4 = 4 * fp8_block_tiles(width), groups = ((rows + 127) & ~127LL) * blocks4;
    if (groups > 0xFFFFFFFFll - Q_PER * Q_GROUPS) return SFFN_ERR_TOO_LARGE;
    const bool vec = aligned16(x) && ld * esize_of(DT) % 16 == 0;
    const unsigned grid = (unsigned)((groups + Q_PER * Q_GROUPS - 1) / (Q_PER * Q_GROUPS));
    if (vec)
        fp8_pack_kernel<DT, true><<<grid, Q_THREADS, 0, st>>>(x, rows, width, ld, values, ldv, scales, (uint32_t)blocks4, (uint32_t)groups);
    else
        fp8_pack_kernel<DT, false><<<grid, Q_THREADS, 0, st>>>(x, rows, width, ld, values, ldv, scales, (uint32_t)blocks4, (uint32_t)groups);
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

template <int DT>
int unpack(const uint8_t* values, long long ldv, const uint8_t* scales, long long rows, long long width, void* out,
           long long ldo, cudaStream_t st) {
    const long long blocks = fp8_blocks(width), groups = rows * blocks;
    if (groups > 0xFFFFFFFFll - Q_GROUPS) return SFFN_ERR_TOO_LARGE;
    const bool vec = aligned16(out) && ldo * esize_of(DT) % 16 == 0;
    const unsigned grid = (unsigned)((groups + Q_GROUPS - 1) / Q_GROUPS);
    if (vec)
        fp8_unpack_kernel<DT, true><<<grid, Q_THREADS, 0, st>>>(values, ldv, scales, rows, width, out, ldo, (uint32_t)blocks, (uint32_t)groups);
    else
        fp8_unpack_kernel<DT, false><<<grid, Q_THREADS, 0, st>>>(values, ldv, scales, rows, width, out, ldo, (uint32_t)blocks, (uint32_t)groups);
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}

// Rows of 16-bit matrices copied to rows on 16 bytes, as TMA reads them; up to
// four matrices a launch.  A thread takes 8 elements of a destination row.
struct PadArgs {
    const uint16_t* src[4];
    uint16_t* dst[4];
    long long cols[4], ld[4], ldd[4];
    long long first[5];  // first 8-element vector of each matrix, in order
    int count;
};
__global__ void __launch_bounds__(256) pad_rows_kernel(const PadArgs a) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.first[a.count]; i += (long long)gridDim.x * 256) {
        int m = 0;
#pragma unroll
        for (int k = 1; k < 4; ++k)
            if (k < a.count && i >= a.first[k]) m = k;
        const long long per = (a.cols[m] + 7) / 8, at = i - a.first[m], row = at / per, c = (at - row * per) * 8;
        const uint16_t* p = a.src[m] + row * a.ld[m] + c;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            w[j] = (c + 2 * j < a.cols[m] ? (uint32_t)__ldg(p + 2 * j) : 0u) | (c + 2 * j + 1 < a.cols[m] ? (uint32_t)__ldg(p + 2 * j + 1) << 16 : 0u);
        *reinterpret_cast<uint4*>(a.dst[m] + row * a.ldd[m] + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

bool fp8_matrix_ok(const void* values, long long ldv, const void* scales, long long width) {
    return values && scales && ldv >= width;
}

}  // namespace
}  // namespace sffn

using namespace sffn;

extern "C" int sffn_fp8_pack(const void* x, int dtype, int64_t rows, int64_t width, int64_t ld, void* values, int64_t ldv,
                             void* scales, void* stream) {
    if (!dtype_ok(dtype)) return SFFN_ERR_DTYPE;
    if (rows < 0 || width < 0) return SFFN_ERR_ARG;
    if (rows == 0 || width == 0) return SFFN_OK;
    if (!x || !fp8_matrix_ok(values, ldv, scales, width) || ld < 0 || (rows > 1 && ld < width)) return SFFN_ERR_ARG;
    if (!aligned16(values) || ldv % 16 || reinterpret_cast<uintptr_t>(x) % esize_of(dtype)) return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(x)) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    uint8_t *v = static_cast<uint8_t*>(values), *s = static_cast<uint8_t*>(scales);
    return dtype == SFFN_F32 ? pack<SFFN_F32>(x, rows, width, ld, v, ldv, s, st)
         : dtype == SFFN_BF16 ? pack<SFFN_BF16>(x, rows, width, ld, v, ldv, s, st)
                              : pack<SFFN_F16>(x, rows, width, ld, v, ldv, s, st);
}

extern "C" int sffn_fp8_unpack(const void* values, int64_t ldv, const void* scales, int64_t rows, int64_t width, int dtype,
                               void* out, int64_t ldo, void* stream) {
    if (!dtype_ok(dtype)) return SFFN_ERR_DTYPE;
    if (rows < 0 || width < 0) return SFFN_ERR_ARG;
    if (rows == 0 || width == 0) return SFFN_OK;
    if (!out || !fp8_matrix_ok(values, ldv, scales, width) || ldo < width) return SFFN_ERR_ARG;
    if (!aligned16(values) || ldv % 16 || reinterpret_cast<uintptr_t>(out) % esize_of(dtype)) return SFFN_ERR_ALIGN;
    DeviceScope scope;
    if (int rc = scope.bind(values)) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const uint8_t *v = static_cast<const uint8_t*>(values), *s = static_cast<const uint8_t*>(scales);
    return dtype == SFFN_F32 ? unpack<SFFN_F32>(v, ldv, s, rows, width, out, ldo, st)
         : dtype == SFFN_BF16 ? unpack<SFFN_BF16>(v, ldv, s, rows, width, out, ldo, st)
                              : unpack<SFFN_F16>(v, ldv, s, rows, width, out, ldo, st);
}

extern "C" int sffn_pad_rows16(int count, const int64_t* desc, void* stream) {
    if (count < 0 || count > 4 || (count && !desc)) return SFFN_ERR_ARG;
    PadArgs a{};
    const void* some = nullptr;
    for (int i = 0; i < count; ++i, desc += 6) {
        const long long rows = desc[1], cols = desc[2];
        a.src[i] = reinterpret_cast<const uint16_t*>(desc[0]);
        a.dst[i] = reinterpret_cast<uint16_t*>(desc[4]);
        a.cols[i] = cols, a.ld[i] = desc[3], a.ldd[i] = desc[5];
        if (rows < 0 || cols < 0 || a.ldd[i] < cols) return SFFN_ERR_ARG;
        if (rows && cols) {
            if (!a.src[i] || !a.dst[i]) return SFFN_ERR_ARG;
            if (!aligned16(a.dst[i]) || a.ldd[i] % 8 || desc[0] % 2) return SFFN_ERR_ALIGN;
            some = a.src[i];
        }
        a.first[i + 1] = a.first[i] + rows * ((cols + 7) / 8);
    }
    a.count = count;
    if (!some) return SFFN_OK;
    DeviceScope scope;
    if (int rc = scope.bind(some)) return rc;
    const long long n = a.first[count], grid = (n + 255) / 256;
    pad_rows_kernel<<<(unsigned)(grid < 148 * 16 ? grid : 148 * 16), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
    SFFN_CHECK_LAUNCH();
    return SFFN_OK;
}
