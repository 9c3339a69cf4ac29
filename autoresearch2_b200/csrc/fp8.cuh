// The 8-bit block format: e4m3 values, one power-of-two scale for each 128
// elements of a row.
//
//   amax = largest finite magnitude of the block
//   e    = smallest integer with amax <= 448 * 2^e, at least -118 (0 for a
//          block of zeros)
//   v    = e4m3(x * 2^-e), to nearest, ties to even; infinities and NaN -> NaN
//
// A power of two scales without rounding, so each element is rounded once, and
// dequantised values are exact in bfloat16 and float32.  e >= -118 keeps the
// smallest step, 2^(e - 9), and 2^-e representable.  Scales are stored as bytes
// e + 127 (the tensor cores' ue8m0) in tiles of 128 rows x 4 blocks, 512
// contiguous bytes as the block-scaled tcgen05.mma reads them:
// [rows / 128][blocks / 4][row % 32][row % 128 / 32][block % 4].
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace sffn {

// sffn_few_rows_fp8; `after`: right behind the pack of x on the stream.
int few_rows_fp8(const void* x, int64_t ldx, const void* x_scales, const void* w, int64_t ldw, const void* w_scales, int64_t T,
                 int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo, bool after, uint32_t* status_dev, void* stream);

// The same products of up to 64 rows, of operands whose rows are on 16 bytes.
constexpr int NARROW_MAX_ROWS = 64;
int narrow_mm(int dtype, const void* x, long long ldx, const void* w, long long ldw, long long T, long long N, long long K, void* out,
              long long ldo, bool after, uint32_t* status, cudaStream_t st);
int narrow_glu(int dtype, int act, const void* x, long long ldx, const void* wg, long long ldwg, const void* wu, long long ldwu, long long T,
               long long D, long long F, void* h, long long ldh, uint32_t* status, cudaStream_t st);
int narrow_fp8(const void* x, long long ldx, const void* x_scales, const void* w, long long ldw, const void* w_scales, long long T, long long N,
               long long K, void* out, int out_dtype, long long ldo, bool after, uint32_t* status, cudaStream_t st);

constexpr int FP8_BLOCK = 128;
constexpr int FP8_LOWEST = -118;

__host__ __device__ inline long long fp8_blocks(long long width) { return (width + FP8_BLOCK - 1) / FP8_BLOCK; }
// Tiles of four blocks across a row.
__host__ __device__ inline long long fp8_block_tiles(long long width) { return (fp8_blocks(width) + 3) / 4; }

// Byte of (row, block) in the scale tiles, bt = fp8_block_tiles(width).
__device__ __forceinline__ long long fp8_scale_at(long long row, int block, long long bt) {
    return ((row >> 7) * bt + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

// |v| as bits where finite, else 0: what enters a block's amax.
__device__ __forceinline__ uint32_t finite_mag(float v) {
    const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
    return b < 0x7F800000u ? b : 0u;
}

// e of a block whose amax has these bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ int fp8_exponent(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return amax_bits == 0 ? 0 : max(e, FP8_LOWEST);
}

// 2^e, -126 <= e <= 127.
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The scale a byte stands for: 2^(byte - 127), 255 is NaN.
__device__ __forceinline__ float fp8_scale(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7FFFFFFFu) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// Four values scaled by 2^-e as four e4m3 bytes.  No finite value saturates
// (the scale sees to that), an infinity becomes a NaN; FINITE: there is none.
template <bool FINITE>
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float inv) {
    const float inf = __uint_as_float(0x7F800000u), nan = __uint_as_float(0x7FFFFFFFu);
    a = FINITE || fabsf(a) < inf ? a * inv : nan;
    b = FINITE || fabsf(b) < inf ? b * inv : nan;
    c = FINITE || fabsf(c) < inf ? c * inv : nan;
    d = FINITE || fabsf(d) < inf ? d * inv : nan;
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// Two e4m3 bytes (low half of w) as two float16 values, exact.
__device__ __forceinline__ __half2 fp8_half2(uint32_t w) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
    return __half2(h);
}

// Four e4m3 bytes as floats.
__device__ __forceinline__ void fp8_unpack4(uint32_t w, float (&f)[4]) {
    const float2 a = __half22float2(fp8_half2(w)), b = __half22float2(fp8_half2(w >> 16));
    f[0] = a.x;
    f[1] = a.y;
    f[2] = b.x;
    f[3] = b.y;
}

// Two floats as two 16-bit values of type DT (nearest, ties to even).
template <int DT>
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi) {
    if constexpr (DT == SFFN_F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <int DT>
__device__ __forceinline__ float2 unpack16x2(uint32_t w) {
    if constexpr (DT == SFFN_F16) {
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    } else {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
}

}  // namespace sffn
