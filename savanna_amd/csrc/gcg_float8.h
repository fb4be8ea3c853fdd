// Tensors in 8-bit floating point with a scale for each block of 128 elements along a row: the format, shared by the norm that
// writes it (gcg_rmsnorm.hip), the quantisers (gcg_float8.hip) and the products (gcg_product8.hip).
//
// (rows, D) is kept as codes (rows, Dp), Dp = D to the next multiple of 128, and scales (rows, S), S = 4 ceil(D / 512), so that a
// product reads whole blocks and whole words of four scales.  A scale is a byte b that stands for 2^(b - 127), the smallest power of
// two that brings the block's largest magnitude to at most the format's largest number (448, or 57344 with 5 bits of exponent); a block of
// zeros has 127.  Codes beyond D are zero, scales beyond the last block 127.
//
// Powers of two make scaling exact: a code is its element rounded once, to 4 (3) significant bits, the matrix instructions apply the
// bytes by themselves, and what is already in 8 bits is quantised again along its other dimension without another rounding (only
// numbers 2^15 times smaller than the largest of the new block lose bits).  A block that holds an infinity or a NaN takes the scale of fp32's
// largest numbers, 2^120 (5 bits of exponent: 2^113): these become NaN (an infinity stays one with 5 bits) and numbers below 2^110 (2^96) zero.
#pragma once
#include "gcg_row.h"

namespace gcg {

constexpr int kBlockF8 = 128;
inline __host__ __device__ int64_t f8_cols(int64_t D) { return (D + 127) / 128 * 128; }
inline __host__ __device__ int64_t f8_scales(int64_t D) { return (D + 511) / 512 * 4; }

// the byte of a block whose largest magnitude has the bits `top`.  (Adding 0x1fffff carries into the exponent where the fraction is beyond
// 1.75, that of the largest number of either format.)
template <bool E5M2> __device__ __forceinline__ uint32_t f8_scale(uint32_t top)
{
    const uint32_t t = top < 0x7f7fffffu ? top : 0x7f7fffffu;
    const int b = (int)((t + 0x1fffffu) >> 23) - (E5M2 ? 15 : 8);
    return top == 0 ? 127u : b > 0 ? (uint32_t)b : 0u;
}
// 2^(127 - b), which brings the block into range
__device__ __forceinline__ float f8_down(uint32_t b) { return __uint_as_float((254u - b) << 23); }
// 2^(b - 127), whose lowest is subnormal; the byte 255, which no quantiser here writes, is no number, whatever it multiplies.  (Both are the shifted
// byte with the fraction's first bit set.)
__device__ __forceinline__ float f8_up(uint32_t b) { return __uint_as_float(b << 23 | (b - 1u >= 254u ? 1u << 22 : 0u)); }

// four codes in a word, rounded to nearest even; what is beyond the range is NaN (5 bits of exponent: infinity)
template <bool E5M2> __device__ __forceinline__ uint32_t f8_codes(float a, float b, float c, float d, float down)
{
    int w;
    if constexpr (E5M2) {
        w = __builtin_amdgcn_cvt_pk_bf8_f32(a * down, b * down, 0, false);
        w = __builtin_amdgcn_cvt_pk_bf8_f32(c * down, d * down, w, true);
    } else {
        w = __builtin_amdgcn_cvt_pk_fp8_f32(a * down, b * down, 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c * down, d * down, w, true);
    }
    return (uint32_t)w;
}
template <bool E5M2> __device__ __forceinline__ void f8_values(uint32_t w, float up, float *v)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    f2 lo, hi;
    if constexpr (E5M2) {
        lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false);
        hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
    } else {
        lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
        hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    }
    v[0] = lo[0] * up; v[1] = lo[1] * up; v[2] = hi[0] * up; v[3] = hi[1] * up;
}

// One vector a lane, at row elements c ..; the 128 / V lanes of a block hold it side by side (absent elements zero).  Dp: codes of a row.
template <int V, bool E5M2, bool STREAM>
__device__ __forceinline__ void store_f8(uint8_t *codes, uint8_t *scales, int c, int Dp, const float (&v)[V])
{
    const uint32_t b = f8_scale<E5M2>(lanes_max<kBlockF8 / V>(top_of<V>(v)));
    const float down = f8_down(b);
    if (c >= Dp) return;
    if constexpr (V == 8) {
        put<STREAM>((u32x2 *)(codes + c), u32x2{f8_codes<E5M2>(v[0], v[1], v[2], v[3], down), f8_codes<E5M2>(v[4], v[5], v[6], v[7], down)});
    } else {
        put<STREAM>((uint32_t *)(codes + c), f8_codes<E5M2>(v[0], v[1], v[2], v[3], down));
    }
    if ((c & (kBlockF8 - 1)) == 0) scales[c / kBlockF8] = (uint8_t)b;
}

} // namespace gcg
