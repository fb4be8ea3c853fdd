// Tensors into 8-bit floating point with a scale for each block of 128 (format: gcg_float8.h), along their rows, along their columns
// (the result transposed, as a product over the rows reads it) or both from one reading, and back.
//
// Bound by memory: s + 1 bytes an element for one direction (s the element's size), s + 2 for both, against a dozen vector instructions.
//
// Measured, bf16: 16384 x 4096 along the rows 34 us (5.9 TB/s), 16384 x 8192 back 69 (5.8); 8192 x 4096 along both from one reading 29 (4.6; a pass each
// way 22 + 29), 4096 x 4096 along the columns 14 (3.5: a tile's two barriers, four workgroups a CU), 8192 x 4096 from 8 bits along the columns 17 (4.0).
#include "gcg_float8.h"

namespace gcg {
namespace {

// ---- along the rows, and back ----------------------------------------------------------------------------------
// A lane holds one 16-byte vector of a block, so a block is 16 lanes (32 in fp32) and its maximum a few lane exchanges.  The lanes take
// the vectors of the rows, filled to whole blocks, one after the other, UNROLL of them each, a fixed step apart.
constexpr int UNROLL = 2;
struct WalkF8 {
    int64_t rows, D, Dp, S;
    int64_t per_row, step_row, step_vec;
};

template <typename T, bool E5M2, bool TAIL, bool STREAM>
__global__ __launch_bounds__(256) void to_float8_kernel(const T *__restrict__ x, uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                        WalkF8 w)
{
    constexpr int V = kVec<T>;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t row = id / w.per_row, vec = id % w.per_row;
    while (row < w.rows) {
        int64_t r[UNROLL], c[UNROLL];
        u32x4 raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            r[u] = row; c[u] = vec * V;
            row += w.step_row; vec += w.step_vec;
            if (vec >= w.per_row) { vec -= w.per_row; ++row; }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            raw[u] = u32x4{0, 0, 0, 0};
            const int64_t left = w.D - c[u];
            if (r[u] < w.rows && left > 0) raw[u] = load_row_vec<T, TAIL, STREAM>(x + r[u] * w.D + c[u], 0, (int)(left < V ? left : V));
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float v[V];
            unpack_vec(raw[u], v, T{});
            // (the lanes of a block are in one row and one wave, so all of them are here or none)
            const int at = (int)(c[u] & (kBlockF8 - 1));
            const int64_t block = c[u] / kBlockF8;
            const bool here = r[u] < w.rows;
            store_f8<V, E5M2, STREAM>(codes + r[u] * w.Dp + block * kBlockF8, scales + r[u] * w.S + block, at, here ? kBlockF8 : 0, v);
            if (here && at == 0 && block == w.Dp / kBlockF8 - 1) {
                for (int64_t i = block + 1; i < w.S; ++i) scales[r[u] * w.S + i] = 127;
            }
        }
    }
}

template <typename T, bool E5M2, bool TAIL, bool STREAM>
__global__ __launch_bounds__(256) void from_float8_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                          T *__restrict__ x, WalkF8 w)
{
    constexpr int V = kVec<T>;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t row = id / w.per_row, vec = id % w.per_row;
    while (row < w.rows) {
        int64_t r[UNROLL], c[UNROLL];
        uint32_t raw[UNROLL][V / 4], b[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            r[u] = row; c[u] = vec * V;
            row += w.step_row; vec += w.step_vec;
            if (vec >= w.per_row) { vec -= w.per_row; ++row; }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            b[u] = 127;
#pragma unroll
            for (int i = 0; i < V / 4; ++i) raw[u][i] = 0;
            if (r[u] < w.rows) {
                const uint8_t *from = codes + r[u] * w.Dp + c[u];
                if constexpr (V == 8) {
                    const u32x2 q = fetch<STREAM>((const u32x2 *)from);
                    raw[u][0] = q[0]; raw[u][1] = q[1];
                } else {
                    raw[u][0] = fetch<STREAM>((const uint32_t *)from);
                }
                b[u] = scales[r[u] * w.S + c[u] / kBlockF8];
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float v[V];
#pragma unroll
            for (int i = 0; i < V / 4; ++i) f8_values<E5M2>(raw[u][i], f8_up(b[u]), v + 4 * i);
            const int64_t left = w.D - c[u];
            if (r[u] < w.rows && left > 0) store_row_vec<T, TAIL, STREAM>(x + r[u] * w.D + c[u], 0, (int)(left < V ? left : V), v);
        }
    }
}

template <typename T> WalkF8 make_walk(int64_t rows, int64_t D, int64_t *blocks)
{
    constexpr int V = kVec<T>;
    WalkF8 w;
    w.rows = rows;
    w.D = D;
    w.Dp = f8_cols(D);
    w.S = f8_scales(D);
    w.per_row = w.Dp / V;
    const int64_t total = rows * w.per_row, most = 1 << 23;         // (a launch holds 2^32 threads)
    *blocks = (total + 256 * UNROLL - 1) / (256 * UNROLL);
    if (*blocks > most) *blocks = most;
    const int64_t step = *blocks * 256;
    w.step_row = step / w.per_row;
    w.step_vec = step % w.per_row;
    return w;
}
template <typename T> bool streams(int64_t rows, int64_t D) { return rows * D * (int64_t)sizeof(T) > kStreamBytes; }

template <typename T, bool E5M2> int to_t(const void *x, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t D, hipStream_t st)
{
    int64_t blocks;
    const WalkF8 w = make_walk<T>(rows, D, &blocks);
    const auto go = [&](auto kernel) { return launch_main(kernel, dim3((unsigned)blocks), dim3(256), st, (const T *)x, codes, scales, w); };
    if (D % kVec<T>) return go(to_float8_kernel<T, E5M2, true, false>);
    return streams<T>(rows, D) ? go(to_float8_kernel<T, E5M2, false, true>) : go(to_float8_kernel<T, E5M2, false, false>);
}
template <typename T, bool E5M2>
int from_t(const uint8_t *codes, const uint8_t *scales, void *x, int64_t rows, int64_t D, hipStream_t st)
{
    int64_t blocks;
    const WalkF8 w = make_walk<T>(rows, D, &blocks);
    const auto go = [&](auto kernel) { return launch_main(kernel, dim3((unsigned)blocks), dim3(256), st, codes, scales, (T *)x, w); };
    if (D % kVec<T>) return go(from_float8_kernel<T, E5M2, true, false>);
    return streams<T>(rows, D) ? go(from_float8_kernel<T, E5M2, false, true>) : go(from_float8_kernel<T, E5M2, false, false>);
}

// ---- along the columns, transposed, and along the rows from the same reading --------------------------------------
// A workgroup takes a tile of 128 x 128, a thread 8 x 8 of it in registers: a row's largest is over 16 lanes, a column's over four lanes of
// four waves.  The transposed codes, eight of a column in a thread, change places in shared memory (8-byte pieces at
// exchanged places, so that those of 16 columns lie in different banks) and leave in whole lines of 128 bytes.
struct Codes8 { };              // an operand in 8-bit floating point, 4 bits of exponent
struct Codes5 { };              // ... 5 bits

struct ColumnsF8 {
    const void *x;
    const uint8_t *x_scales;            // of an operand in 8 bits
    uint8_t *codes, *scales;            // along the rows, or null
    uint8_t *codes_t, *scales_t;        // along the columns
    int64_t R, D, Dp, S, Rp, St;
    uint32_t col_tiles;
};

template <typename T, bool TAIL> __device__ __forceinline__ void load8(const ColumnsF8 &a, int64_t row, int64_t c, float (&v)[8])
{
    constexpr int V = kVec<T>;
#pragma unroll
    for (int h = 0; h < 8 / V; ++h) {
        const int64_t at = c + h * V, left = a.D - at;
        u32x4 raw = {0, 0, 0, 0};
        if (row < a.R && left > 0) raw = load_row_vec<T, TAIL, false>((const T *)a.x + row * a.D + at, 0, (int)(left < V ? left : V));
        float q[V];
        unpack_vec(raw, q, T{});
#pragma unroll
        for (int i = 0; i < V; ++i) v[h * V + i] = q[i];
    }
}

template <typename T, bool E5M2, bool ROWS, bool TAIL> __global__ __launch_bounds__(256) void to_float8_columns_kernel(ColumnsF8 a)
{
    __shared__ __attribute__((aligned(16))) uint8_t tile[128 * 128];
    __shared__ uint32_t tops[4][128];
    const int cg = threadIdx.x & 15, rg = threadIdx.x >> 4, wave = threadIdx.x / kWave;
    const int64_t rt = blockIdx.x / a.col_tiles, ct = blockIdx.x % a.col_tiles;
    const int64_t row0 = rt * 128 + rg * 8, col0 = ct * 128 + cg * 8;
    float v[8][8];
    if constexpr (std::is_same_v<T, Codes8> || std::is_same_v<T, Codes5>) {
        u32x2 raw[8];
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            raw[i] = u32x2{0, 0};
            b[i] = 127;
            if (row0 + i < a.R) {
                raw[i] = *(const u32x2 *)((const uint8_t *)a.x + (row0 + i) * a.Dp + col0);
                b[i] = a.x_scales[(row0 + i) * a.S + ct];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) f8_values<std::is_same_v<T, Codes5>>(raw[i][h], f8_up(b[i]), v[i] + 4 * h);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) load8<T, TAIL>(a, row0 + i, col0, v[i]);
    }

    uint32_t top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        top[j] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t u = __float_as_uint(v[i][j]) & 0x7fffffffu;
            top[j] = u > top[j] ? u : top[j];
        }
        // the wave's four groups of rows
        uint32_t other = __shfl_xor(top[j], 16);
        top[j] = other > top[j] ? other : top[j];
        other = __shfl_xor(top[j], 32);
        top[j] = other > top[j] ? other : top[j];
    }
    if ((threadIdx.x & 63) < 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) tops[wave][cg * 8 + j] = top[j];
    }
    if constexpr (ROWS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool here = row0 + i < a.R;
            store_f8<8, E5M2, false>(a.codes + (row0 + i) * a.Dp + ct * 128, a.scales + (row0 + i) * a.S + ct, cg * 8, here ? 128 : 0, v[i]);
            if (here && cg == 0 && ct == a.col_tiles - 1) {
                for (int64_t k = ct + 1; k < a.S; ++k) a.scales[(row0 + i) * a.S + k] = 127;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int col = cg * 8 + j;
        uint32_t t = tops[0][col];
#pragma unroll
        for (int w = 1; w < 4; ++w) t = tops[w][col] > t ? tops[w][col] : t;
        const uint32_t b = f8_scale<E5M2>(t);
        const float down = f8_down(b);
        const u32x2 word = {f8_codes<E5M2>(v[0][j], v[1][j], v[2][j], v[3][j], down), f8_codes<E5M2>(v[4][j], v[5][j], v[6][j], v[7][j], down)};
        *(u32x2 *)(tile + col * 128 + ((rg ^ cg) * 8)) = word;
        if (rg == 0 && col0 + j < a.D) {
            uint8_t *to = a.scales_t + (col0 + j) * a.St + rt;
            *to = (uint8_t)b;
            if (rt == a.Rp / 128 - 1) {
                for (int64_t k = 1; k < a.St - rt; ++k) to[k] = 127;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int col = p * 32 + (threadIdx.x >> 3), seg = threadIdx.x & 7, f = col >> 3;
        const u32x2 lo = *(const u32x2 *)(tile + col * 128 + ((2 * seg) ^ f) * 8), hi = *(const u32x2 *)(tile + col * 128 + ((2 * seg + 1) ^ f) * 8);
        if (ct * 128 + col < a.D) *(u32x4 *)(a.codes_t + (ct * 128 + col) * a.Rp + rt * 128 + seg * 16) = u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
}

template <typename T, bool E5M2> int columns_t(const ColumnsF8 &a, hipStream_t st)
{
    const dim3 grid((unsigned)(a.Rp / 128 * a.col_tiles)), block(256);
    if constexpr (std::is_same_v<T, Codes8> || std::is_same_v<T, Codes5>) {
        return launch_main(to_float8_columns_kernel<T, E5M2, false, false>, grid, block, st, a);
    } else {
        if (a.D % kVec<T>) return a.codes ? launch_main(to_float8_columns_kernel<T, E5M2, true, true>, grid, block, st, a)
                                          : launch_main(to_float8_columns_kernel<T, E5M2, false, true>, grid, block, st, a);
        return a.codes ? launch_main(to_float8_columns_kernel<T, E5M2, true, false>, grid, block, st, a)
                       : launch_main(to_float8_columns_kernel<T, E5M2, false, false>, grid, block, st, a);
    }
}

} // namespace

int to_float8_launch(int dtype, int e5m2, const void *x, uint8_t *codes, uint8_t *scales, int64_t rows, int64_t D, hipStream_t st)
{
    switch (dtype) {
    case GCG_F32: return e5m2 ? to_t<float, true>(x, codes, scales, rows, D, st) : to_t<float, false>(x, codes, scales, rows, D, st);
    case GCG_BF16: return e5m2 ? to_t<bf16_t, true>(x, codes, scales, rows, D, st) : to_t<bf16_t, false>(x, codes, scales, rows, D, st);
    default: return e5m2 ? to_t<f16_t, true>(x, codes, scales, rows, D, st) : to_t<f16_t, false>(x, codes, scales, rows, D, st);
    }
}

int from_float8_launch(int dtype, int e5m2, const uint8_t *codes, const uint8_t *scales, void *x, int64_t rows, int64_t D, hipStream_t st)
{
    switch (dtype) {
    case GCG_F32: return e5m2 ? from_t<float, true>(codes, scales, x, rows, D, st) : from_t<float, false>(codes, scales, x, rows, D, st);
    case GCG_BF16: return e5m2 ? from_t<bf16_t, true>(codes, scales, x, rows, D, st) : from_t<bf16_t, false>(codes, scales, x, rows, D, st);
    default: return e5m2 ? from_t<f16_t, true>(codes, scales, x, rows, D, st) : from_t<f16_t, false>(codes, scales, x, rows, D, st);
    }
}

// x: of type dtype, or, with x_scales, in 8 bits of the format from5
int to_float8_columns_launch(int dtype, int e5m2, int from5, const void *x, const uint8_t *x_scales, uint8_t *codes, uint8_t *scales,
                             uint8_t *codes_t, uint8_t *scales_t, int64_t rows, int64_t D, hipStream_t st)
{
    const ColumnsF8 a = {x, x_scales, codes, scales, codes_t, scales_t, rows, D, f8_cols(D), f8_scales(D), f8_cols(rows), f8_scales(rows),
                         (uint32_t)(f8_cols(D) / 128)};
    if (x_scales) {
        if (from5) return e5m2 ? columns_t<Codes5, true>(a, st) : columns_t<Codes5, false>(a, st);
        return e5m2 ? columns_t<Codes8, true>(a, st) : columns_t<Codes8, false>(a, st);
    }
    switch (dtype) {
    case GCG_F32: return e5m2 ? columns_t<float, true>(a, st) : columns_t<float, false>(a, st);
    case GCG_BF16: return e5m2 ? columns_t<bf16_t, true>(a, st) : columns_t<bf16_t, false>(a, st);
    default: return e5m2 ? columns_t<f16_t, true>(a, st) : columns_t<f16_t, false>(a, st);
    }
}

} // namespace gcg
