// Activations in the 8-bit block format (fp8.cuh): pack and unpack.
//
// Both are bound by memory: per element of a 16-bit tensor the pack reads two
// bytes and writes one (and 1/128), the unpack the reverse.  Eight lanes share
// a block of 128, 16 contiguous elements each: whole 16-byte loads and stores,
// the amax by three shuffles.
#include "fp8.cuh"

namespace sffn {
namespace {

constexpr int Q_THREADS = 256;
constexpr int Q_GROUPS = Q_THREADS / 8;  // blocks of 128 a thread block takes

// 16 elements from column c on, zeros past the row's end.
template <int DT, bool VEC>
__device__ __forceinline__ void load16(const void* row, long long c, long long width, float (&f)[16]) {
    using bits = typename Elt<DT>::bits;
    const bits* p = static_cast<const bits*>(row) + c;
    if (VEC && c + 16 <= width) {
        const uint4* q = reinterpret_cast<const uint4*>(p);
        if constexpr (DT == SFFN_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 v = __ldcs(q + i);
                f[4 * i] = __uint_as_float(v.x);
                f[4 * i + 1] = __uint_as_float(v.y);
                f[4 * i + 2] = __uint_as_float(v.z);
                f[4 * i + 3] = __uint_as_float(v.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 v = __ldcs(q + i);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 a = unpack16x2<DT>(w[j]);
                    f[8 * i + 2 * j] = a.x;
                    f[8 * i + 2 * j + 1] = a.y;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = c + i < width ? Elt<DT>::to_f(p[i]) : 0.f;
    }
}

// Eight lanes a block; the groups run over padded rows x padded blocks (whole
// scale tiles), those of the padding write their scale byte, zero.
template <int DT, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
    fp8_pack_kernel(const void* __restrict__ x, long long rows, long long width, long long ld, uint8_t* __restrict__ values,
                    long long ldv, uint8_t* __restrict__ scales, uint32_t blocks4, uint32_t groups) {
    const uint32_t id = blockIdx.x * (uint32_t)Q_GROUPS + (threadIdx.x >> 3);
    const int sub = threadIdx.x & 7;
    const uint32_t row = id / blocks4;
    const int block = (int)(id - row * blocks4);
    const bool in_grid = id < groups;
    const long long c = (long long)block * FP8_BLOCK + sub * 16;
    const bool live = in_grid && row < rows && (long long)block * FP8_BLOCK < width;
    float f[16];
    uint32_t amax = 0;
    if (live) {
        load16<DT, VEC>(static_cast<const typename Elt<DT>::bits*>(x) + (long long)row * ld, c, width, f);
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = max(amax, finite_mag(f[i]));
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(FULL, amax, o));
    if (!in_grid) return;
    const int e = fp8_exponent(amax);
    if (sub == 0) scales[fp8_scale_at(row, block, blocks4 >> 2)] = live ? (uint8_t)(e + 127) : 0;
    if (!live || c >= width) return;
    const float inv = two_to(-e);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = fp8_pack4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3], inv);
    *reinterpret_cast<uint4*>(values + (long long)row * ldv + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
    fp8_unpack_kernel(const uint8_t* __restrict__ values, long long ldv, const uint8_t* __restrict__ scales, long long rows,
                      long long width, void* __restrict__ out, long long ldo, uint32_t blocks, uint32_t groups) {
    using bits = typename Elt<DT>::bits;
    const uint32_t id = blockIdx.x * (uint32_t)Q_GROUPS + (threadIdx.x >> 3);
    if (id >= groups) return;
    const uint32_t row = id / blocks;
    const int block = (int)(id - row * blocks);
    const long long c = (long long)block * FP8_BLOCK + (threadIdx.x & 7) * 16;
    if (c >= width) return;
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(values + (long long)row * ldv + c));
    const float s = fp8_scale(scales[fp8_scale_at(row, block, (blocks + 3) >> 2)]);
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
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (c + i < width) p[i] = Elt<DT>::from_f(f[i]);
    }
}

template <int DT>
int pack(const void* x, long long rows, long long width, long long ld, uint8_t* values, long long ldv, uint8_t* scales,
         cudaStream_t st) {
    const long long blocks4 = 4 * fp8_block_tiles(width), groups = ((rows + 127) & ~127LL) * blocks4;
    if (groups > 0xFFFFFFFFll - Q_GROUPS) return SFFN_ERR_TOO_LARGE;
    const bool vec = aligned16(x) && ld * esize_of(DT) % 16 == 0;
    const unsigned grid = (unsigned)((groups + Q_GROUPS - 1) / Q_GROUPS);
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
    if (int rc = scope.bind_same(x, {values, scales})) return rc;
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
    if (int rc = scope.bind_same(values, {scales, out})) return rc;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const uint8_t *v = static_cast<const uint8_t*>(values), *s = static_cast<const uint8_t*>(scales);
    return dtype == SFFN_F32 ? unpack<SFFN_F32>(v, ldv, s, rows, width, out, ldo, st)
         : dtype == SFFN_BF16 ? unpack<SFFN_BF16>(v, ldv, s, rows, width, out, ldo, st)
                              : unpack<SFFN_F16>(v, ldv, s, rows, width, out, ldo, st);
}
