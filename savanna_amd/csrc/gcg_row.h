// Rows of any width and element alignment in 16-byte vectors, sums and maxima over lanes, and the 8-bit checkpoint format:
// what the norms (gcg_norm.hip, gcg_rmsnorm.hip), the checkpoint
// kernels (gcg_act8.hip) and those of the 8-bit floating-point tensors (gcg_float8.hip) share.
#pragma once
#include "gcg_common.h"

namespace gcg {

// 16-byte (8-byte) vectors that start at any element: the unaligned forms of the global loads and stores
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));

template <typename T> constexpr int kVec = 16 / (int)sizeof(T);          // elements of a vector

// Accesses with the streaming hint, for tensors that the last-level cache (256 MB) does not hold from one kernel to the next
// anyway: 16384 x 12288 bf16 into 8 bits and back 128 + 124 us without, 104 + 103 with; norm of 32768 x 8192 203 and 192, its
// backward 295 and 273, from 8 bits 320 and 312.  Smaller ones gain nothing, and the next kernel finds them in the cache.
constexpr int64_t kStreamBytes = 256ll << 20;
template <bool STREAM, typename P> __device__ __forceinline__ P fetch(const P *p)
{
    if constexpr (STREAM) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool STREAM, typename P, typename X> __device__ __forceinline__ void put(P *p, const X &v)
{
    if constexpr (STREAM) __builtin_nontemporal_store((P)v, p);
    else *p = v;
}

__device__ __forceinline__ void unpack_vec(const u32x4 &r, float (&v)[4], float)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void unpack_vec(const u32x4 &r, float (&v)[8], bf16_t)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(r[i] << 16); v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u); }
}
__device__ __forceinline__ void unpack_vec(const u32x4 &r, float (&v)[8], f16_t)
{
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    h8 h;
    __builtin_memcpy(&h, &r, 16);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
}
__device__ __forceinline__ u32x4 pack_vec(const float (&v)[4], float)
{
    return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
__device__ __forceinline__ u32x4 pack_vec(const float (&v)[8], bf16_t)
{
    return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ u32x4 pack_vec(const float (&v)[8], f16_t)
{
    return u32x4{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7])};
}

// The vector of row elements c .. c + kVec - 1, of which those at D and beyond are absent (zeros).  TAIL: D is not a multiple
// of the vector, so one lane of a row has a vector that ends inside it and goes element by element.
// STREAM: with the streaming hint.
template <typename T, bool TAIL, bool STREAM> __device__ __forceinline__ u32x4 load_row_vec(const T *row, int c, int D)
{
    constexpr int V = kVec<T>;
    u32x4 r = {0, 0, 0, 0};
    if (c + V <= D) r = fetch<STREAM>((const u32x4_any *)(row + c));
    else if (TAIL && c < D) {
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = c + i < D ? Elem<T>::load(row + c + i) : 0.f;
        r = pack_vec(v, T{});
    }
    return r;
}
// The same for a lane that goes from row to row and requests the next one while it works: element by element in a branch, the vector that ends
// inside the row would be waited for there.  So where a vector would reach beyond the row, its last kVec elements are loaded, and put
// in their place (in_place) when they are needed.  Rows shorter than a vector take the branch.
template <typename T, bool TAIL, bool STREAM> __device__ __forceinline__ u32x4 request_row_vec(const T *row, int c, int D)
{
    constexpr int V = kVec<T>;
    if constexpr (TAIL) {
        if (D < V) return load_row_vec<T, true, STREAM>(row, c, D);
        return fetch<STREAM>((const u32x4_any *)(row + (c < D - V ? c : D - V)));
    } else {
        return load_row_vec<T, false, STREAM>(row, c, D);
    }
}
template <typename T, bool TAIL> __device__ __forceinline__ u32x4 in_place(u32x4 r, int c, int D)
{
    constexpr int V = kVec<T>;
    if constexpr (TAIL) {
        const int left = D - c;
        if (D >= V && __any(left < V)) {
            const int s = (V - D % V) * (int)sizeof(T);                     // bytes
            u32x4 t = r;
            if (s & 8) t = u32x4{t[2], t[3], 0, 0};
            if (s & 4) t = u32x4{t[1], t[2], t[3], 0};
            if (s & 2) t = u32x4{t[0] >> 16 | t[1] << 16, t[1] >> 16 | t[2] << 16, t[2] >> 16 | t[3] << 16, t[3] >> 16};
            if (left < V) r = left > 0 ? t : u32x4{0, 0, 0, 0};
        }
    }
    return r;
}
template <typename T, bool TAIL, bool STREAM>
__device__ __forceinline__ void store_row_vec(T *row, int c, int D, const float (&v)[kVec<T>])
{
    constexpr int V = kVec<T>;
    if (c + V <= D) put<STREAM>((u32x4_any *)(row + c), pack_vec(v, T{}));
    else if (TAIL && c < D) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < D) Elem<T>::store(row + c + i, v[i]);
    }
}

// ---- sums and maxima over lanes ---------------------------------------------------------------------------
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_add(float x)
{
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROWS, 0xf, false));
}
// the wave's sum, the same in every lane: inside rows of 16 lanes (pairs, fours, mirrored eights, mirrored sixteens), then
// from row to row
__device__ __forceinline__ float wave_sum(float x)
{
    x = dpp_add<0xb1, 0xf>(x);
    x = dpp_add<0x4e, 0xf>(x);
    x = dpp_add<0x141, 0xf>(x);
    x = dpp_add<0x140, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);
    x = dpp_add<0x143, 0xc>(x);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t x)
{
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false);
    return x > y ? x : y;
}
// largest of the N = 16 or 32 lanes that this lane belongs to
template <int N> __device__ __forceinline__ uint32_t lanes_max(uint32_t x)
{
    x = dpp_max<0xb1>(x);
    x = dpp_max<0x4e>(x);
    x = dpp_max<0x141>(x);
    x = dpp_max<0x140>(x);
    if constexpr (N == 32) {
        const uint32_t y = (uint32_t)__builtin_amdgcn_ds_swizzle((int)x, 0x401f);       // lane ^ 16
        x = x > y ? x : y;
    }
    return x;
}

// weight or bias of a norm, elements c .. c + V - 1: of the tensors' type, or fp32
template <typename T, bool TAIL>
__device__ __forceinline__ void load_param(const void *p, bool f32, int c, int D, float absent, float (&v)[kVec<T>])
{
    constexpr int V = kVec<T>;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = absent;
    if (!p || c >= D) return;
    if (f32 && sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (!TAIL || c + i < D) v[i] = ((const float *)p)[c + i];
    } else {
        unpack_vec(load_row_vec<T, TAIL, false>((const T *)p, c, D), v, T{});
    }
}

// sums of N numbers over the TPR lanes of a row.  More than one wave: through `slots`, of which the caller gives another set
// every time, so that one barrier is enough.
template <int TPR, int N> __device__ __forceinline__ void row_sum(float (&s)[N], float *slots)
{
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = wave_sum(s[n]);
    if constexpr (TPR > kWave) {
        constexpr int W = TPR / kWave;
        const int wave = threadIdx.x / kWave, first = threadIdx.x / TPR * W;
        if (threadIdx.x % kWave == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) slots[wave * N + n] = s[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            s[n] = slots[first * N + n];
#pragma unroll
            for (int i = 1; i < W; ++i) s[n] += slots[(first + i) * N + n];
        }
    }
}

// ---- the 8-bit checkpoint format ----------------------------------------------------------------------------
// Blocks of 128 elements along a row share an fp32 scale; the last block of a row may be shorter.  top = the largest
// magnitude; scale = top * fp32(1 / 127), code = rint(x * (127 / top)), value = code * scale: one step is 1 / 127 of the
// block's largest, so a value is at most half of that off (0.4 % of the largest).  Magnitudes are compared as integers,
// which orders infinities and NaN above everything: a block that holds one gets the scale NaN and comes back as NaN
// throughout, so that an overflow is still seen in the gradients.  Below 2^-100 the quotient would leave fp32: zeros.
constexpr int kBlock8 = 128;

struct Scale8 { float scale, inv; };
__device__ __forceinline__ Scale8 scale8(uint32_t top_bits)
{
    const float top = __uint_as_float(top_bits);
    if (top_bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
    if (top < 0x1p-100f) return {0.f, 0.f};
    return {top * (1.0f / 127.0f), 127.0f / top};
}
// Four codes in a word.  fl(x * inv) + 1.5 * 2^23 is rounded to a whole number (to even, as rint), whose lowest byte is the
// code; the product is rounded by itself first, as in the format's definition.  A NaN or infinity has inv = 0 and a scale that
// makes every code count as NaN.
__device__ __forceinline__ uint32_t codes8(float a, float b, float c, float d, float inv)
{
#pragma clang fp contract(off)
    const float magic = 12582912.f;
    const uint32_t i = __float_as_uint(a * inv + magic), j = __float_as_uint(b * inv + magic);
    const uint32_t k = __float_as_uint(c * inv + magic), l = __float_as_uint(d * inv + magic);
    const uint32_t lo = __builtin_amdgcn_perm(j, i, 0x0c0c0400u), hi = __builtin_amdgcn_perm(l, k, 0x04000c0cu);
    return lo | hi;
}
__device__ __forceinline__ void values8(uint32_t w, float scale, float *v)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> (8 * i)) * scale;
}

// the magnitude's bits of the largest of a lane's elements
template <int V> __device__ __forceinline__ uint32_t top_of(const float (&v)[V])
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
        m = b > m ? b : m;
    }
    return m;
}
// Codes of one vector a lane, at row elements c ..; the 128 / V lanes of a block hold it side by side (absent elements zero).
template <int V, bool TAIL, bool STREAM>
__device__ __forceinline__ void store_codes8(int8_t *codes, float *scales, int c, int D, const float (&v)[V])
{
    const Scale8 s = scale8(lanes_max<kBlock8 / V>(top_of<V>(v)));
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) w[i] = codes8(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], s.inv);
    if (c + V <= D) {
        if constexpr (V == 8) put<STREAM>((u32x2_any *)(codes + c), u32x2{w[0], w[1]});
        else put<STREAM>((u32_any *)(codes + c), w[0]);
    } else if (TAIL) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < D) codes[c + i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
    }
    if (c < D && (c & (kBlock8 - 1)) == 0) scales[c / kBlock8] = s.scale;
}
// The words of a vector's codes, absent ones zero.
template <int V, bool TAIL, bool STREAM> __device__ __forceinline__ u32x2 load_codes8(const int8_t *codes, int c, int D)
{
    u32x2 w = {0, 0};
    if (c + V <= D) {
        if constexpr (V == 8) w = fetch<STREAM>((const u32x2_any *)(codes + c));
        else w[0] = fetch<STREAM>((const u32_any *)(codes + c));
    } else if (TAIL && c < D) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c + i < D) w[i / 4] |= (uint32_t)(uint8_t)codes[c + i] << (8 * (i % 4));
    }
    return w;
}

} // namespace gcg
