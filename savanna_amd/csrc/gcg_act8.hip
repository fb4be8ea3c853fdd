// Activation checkpoints in 8 bits: a (rows, D) tensor into codes and block scales (the format is in gcg_row.h) and back.
//
// Bound by memory: s + 1 + 1/32 bytes an element each way, against a dozen vector instructions.  A lane holds one 16-byte
// vector of a block, so a block is 16 lanes (32 in fp32) and its maximum a few lane exchanges; no shared memory, no barrier.
// Measured, 16384 x 12288 bf16: 98 us each way, 6.2 TB/s, more than a copy of that size reaches (5.2); small tensors (701 x 1001
// fp32: 3.6 and 3.4 us) are bound by the launch.
#include "gcg_row.h"

namespace gcg {
namespace {

// A wave's vectors lie wave * 64 .. + 63 in the row-major list of a row's vectors; rows of whole blocks are one long row.
// Each lane takes UNROLL of them, a fixed step apart, whose parts in rows and vectors the host divides (a loop over more of them in
// fewer workgroups is slower: 16384 x 12288 bf16 110 us, 98 this way).
constexpr int UNROLL = 2;
struct Walk { int64_t rows; int64_t D; int64_t per_row; int64_t step_row, step_vec; };

template <typename T, bool TAIL, bool STREAM>
__global__ __launch_bounds__(256) void pack8_kernel(const T *__restrict__ x, int8_t *__restrict__ codes, float *__restrict__ scales,
                                                    Walk w)
{
    constexpr int V = kVec<T>;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t row = id / w.per_row, vec = id % w.per_row;
    const int64_t nb = (w.D + kBlock8 - 1) / kBlock8;
    while (row < w.rows) {
        int64_t r[UNROLL], c[UNROLL];
        u32x4 raw[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            r[u] = row; c[u] = vec;
            row += w.step_row; vec += w.step_vec;
            if (vec >= w.per_row) { vec -= w.per_row; ++row; }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            raw[u] = u32x4{0, 0, 0, 0};
            if (r[u] < w.rows) raw[u] = load_row_vec<T, TAIL, STREAM>(x + r[u] * w.D + c[u] * V, 0, (int)(w.D - c[u] * V < V ? w.D - c[u] * V : V));
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float v[V];
            unpack_vec(raw[u], v, T{});
            const int64_t at = c[u] * V, left = w.D - at;
            // (a row's vectors are padded to whole blocks, so the lanes of a block are in one row and one wave)
            const int D = r[u] < w.rows && left > 0 ? (int)(left < V ? left : V) : 0;
            const Scale8 s = scale8(lanes_max<kBlock8 / V>(top_of<V>(v)));
            uint32_t word[V / 4];
#pragma unroll
            for (int i = 0; i < V / 4; ++i) word[i] = codes8(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], s.inv);
            if (D > 0) {
                int8_t *to = codes + r[u] * w.D + at;
                if (D == V) {
                    if constexpr (V == 8) put<STREAM>((u32x2_any *)to, u32x2{word[0], word[1]});
                    else put<STREAM>((u32_any *)to, word[0]);
                } else if (TAIL) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (i < D) to[i] = (int8_t)(word[i / 4] >> (8 * (i % 4)));
                }
                if ((at & (kBlock8 - 1)) == 0) scales[r[u] * nb + at / kBlock8] = s.scale;
            }
        }
    }
}

template <typename T, bool TAIL, bool STREAM>
__global__ __launch_bounds__(256) void unpack8_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scales,
                                                      T *__restrict__ x, Walk w)
{
    constexpr int V = kVec<T>;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t row = id / w.per_row, vec = id % w.per_row;
    const int64_t nb = (w.D + kBlock8 - 1) / kBlock8;
    while (row < w.rows) {
        int64_t r[UNROLL], c[UNROLL];
        u32x2 raw[UNROLL];
        float scale[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            r[u] = row; c[u] = vec * V;
            row += w.step_row; vec += w.step_vec;
            if (vec >= w.per_row) { vec -= w.per_row; ++row; }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            raw[u] = u32x2{0, 0};
            scale[u] = 0.f;
            if (r[u] < w.rows && c[u] < w.D) {
                const int64_t left = w.D - c[u];
                raw[u] = load_codes8<V, TAIL, STREAM>(codes + r[u] * w.D + c[u], 0, (int)(left < V ? left : V));
                scale[u] = scales[r[u] * nb + c[u] / kBlock8];
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float v[V];
#pragma unroll
            for (int i = 0; i < V / 4; ++i) values8(raw[u][i], scale[u], v + 4 * i);
            const int64_t left = w.D - c[u];
            if (r[u] < w.rows && left > 0) store_row_vec<T, TAIL, STREAM>(x + r[u] * w.D + c[u], 0, (int)(left < V ? left : V), v);
        }
    }
}

template <typename T> Walk make_walk(int64_t rows, int64_t D, int64_t *blocks)
{
    constexpr int V = kVec<T>;
    Walk w;
    if (D % kBlock8 == 0) { D *= rows; rows = 1; }
    w.rows = rows;
    w.D = D;
    w.per_row = (D + kBlock8 - 1) / kBlock8 * (kBlock8 / V);
    const int64_t total = rows * w.per_row, most = 1 << 23;         // (a launch holds 2^32 threads)
    *blocks = (total + 256 * UNROLL - 1) / (256 * UNROLL);
    if (*blocks > most) *blocks = most;
    const int64_t step = *blocks * 256;
    w.step_row = step / w.per_row;
    w.step_vec = step % w.per_row;
    return w;
}

template <typename T> bool streams(int64_t rows, int64_t D) { return rows * D * (int64_t)sizeof(T) > kStreamBytes; }

template <typename T> int pack_t(const void *x, int8_t *codes, float *scales, int64_t rows, int64_t D, hipStream_t st)
{
    int64_t blocks;
    const Walk w = make_walk<T>(rows, D, &blocks);
    const auto go = [&](auto kernel) { return launch_main(kernel, dim3((unsigned)blocks), dim3(256), st, (const T *)x, codes, scales, w); };
    if (D % kVec<T>) return streams<T>(rows, D) ? go(pack8_kernel<T, true, true>) : go(pack8_kernel<T, true, false>);
    return streams<T>(rows, D) ? go(pack8_kernel<T, false, true>) : go(pack8_kernel<T, false, false>);
}
template <typename T> int unpack_t(const int8_t *codes, const float *scales, void *x, int64_t rows, int64_t D, hipStream_t st)
{
    int64_t blocks;
    const Walk w = make_walk<T>(rows, D, &blocks);
    const auto go = [&](auto kernel) { return launch_main(kernel, dim3((unsigned)blocks), dim3(256), st, codes, scales, (T *)x, w); };
    if (D % kVec<T>) return streams<T>(rows, D) ? go(unpack8_kernel<T, true, true>) : go(unpack8_kernel<T, true, false>);
    return streams<T>(rows, D) ? go(unpack8_kernel<T, false, true>) : go(unpack8_kernel<T, false, false>);
}

} // namespace

int pack8_launch(int dtype, const void *x, int8_t *codes, float *scales, int64_t rows, int64_t D, hipStream_t st)
{
    switch (dtype) {
    case GCG_F32: return pack_t<float>(x, codes, scales, rows, D, st);
    case GCG_BF16: return pack_t<bf16_t>(x, codes, scales, rows, D, st);
    default: return pack_t<f16_t>(x, codes, scales, rows, D, st);
    }
}
int unpack8_launch(int dtype, const int8_t *codes, const float *scales, void *x, int64_t rows, int64_t D, hipStream_t st)
{
    switch (dtype) {
    case GCG_F32: return unpack_t<float>(codes, scales, x, rows, D, st);
    case GCG_BF16: return unpack_t<bf16_t>(codes, scales, x, rows, D, st);
    default: return unpack_t<f16_t>(codes, scales, x, rows, D, st);
    }
}

} // namespace gcg
