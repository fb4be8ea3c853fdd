// Layer norm, forward and backward, with the weight's and bias's gradient, and its 8-bit form.
//
//   mean = sum x / D, rstd = (sum (x - mean)^2 / D + eps)^-1/2, xh = (x - mean) rstd, y = xh w + b
//   g = dy w;  dx = rstd (g - mean(g) - xh mean(g xh));  dw = sum over rows of dy xh, db of dy
//
// Bound by memory: 2 s bytes an element forward, 3 s backward (s the element's size), for some ten and twenty vector
// instructions.  A row is held in the registers of TPR lanes, so it is read once and the variance is summed about the mean; a
// row of one wave needs no barrier.  All sums are fp32.  With `codes` the forward writes the row's 8-bit checkpoint (gcg_row.h)
// from the same registers, and the backward reads that in the row's place, about the exact row's mean and rstd.
//
// Measured: 16384 x 4096 bf16 forward 46 us (5.8 TB/s), backward 81 + 4 (5.0); 15009 x 2560 f16 29 and 50 + 4; 32768 x 8192 bf16 with
// the 8-bit form 247 (5.4 TB/s) and 326 + 5 (4.1: twice the lanes a row, and codes to convert); 2048 x 256 fp32 forward 3.2, a launch.
#include "gcg_row.h"

namespace gcg {
namespace {

// weight or bias elements c .. c + V - 1: of the tensors' type, or fp32
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

struct NormFwd {
    const void *x, *w, *b;
    void *y;
    float *stats;               // (rows, 2): mean, rstd; or null
    int8_t *codes;              // the 8-bit checkpoint of x, or null
    float *scales;
    int64_t rows;
    int32_t D;
    float inv_d, eps;
    int32_t param_f32;
};

// TPR lanes hold a row, K vectors each; a workgroup of max(TPR, 256) threads walks over rows, the next row's loads in flight
// while one is worked on.
template <typename T, int TPR, int K, bool BITS8, bool TAIL, bool STREAM>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_fwd_kernel(NormFwd a)
{
    constexpr int V = kVec<T>, THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
    __shared__ float slots[2][2][THREADS / kWave];
    const int t = threadIdx.x % TPR, D = a.D;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / TPR;
    const int64_t nb = (D + kBlock8 - 1) / kBlock8;

    u32x4 next[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        next[k] = u32x4{0, 0, 0, 0};
        if (row < a.rows) next[k] = load_row_vec<T, TAIL, STREAM>((const T *)a.x + row * D, (k * TPR + t) * V, D);
    }
    float w[K][V], b[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        load_param<T, TAIL>(a.w, a.param_f32, (k * TPR + t) * V, D, 1.f, w[k]);
        load_param<T, TAIL>(a.b, a.param_f32, (k * TPR + t) * V, D, 0.f, b[k]);
    }
    // every group of the workgroup goes through the same number of turns, so that all meet at the barriers
    for (int64_t base = (int64_t)blockIdx.x * GROUPS, turn = 0; base < a.rows; base += step, row += step, ++turn) {
        float v[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k) unpack_vec(next[k], v[k], T{});
        if (row + step < a.rows) {
#pragma unroll
            for (int k = 0; k < K; ++k) next[k] = load_row_vec<T, TAIL, STREAM>((const T *)a.x + (row + step) * D, (k * TPR + t) * V, D);
        }
        float s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] += v[k][i];
        row_sum<TPR, 1>(s, slots[turn & 1][0]);
        const float mean = s[0] * a.inv_d;
        float q[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = v[k][i] - mean;
                if ((k * TPR + t) * V + (TAIL ? i : 0) < D) q[0] = fmaf(d, d, q[0]);
            }
        row_sum<TPR, 1>(q, slots[turn & 1][1]);
        const float rstd = 1.0f / sqrtf(q[0] * a.inv_d + a.eps);
        if (row < a.rows) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * TPR + t) * V;
                float y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = fmaf((v[k][i] - mean) * rstd, w[k][i], b[k][i]);
                store_row_vec<T, TAIL, STREAM>((T *)a.y + row * D, c, D, y);
                if constexpr (BITS8) store_codes8<V, TAIL, STREAM>(a.codes + row * D, a.scales + row * nb, c, D, v[k]);
            }
            if (a.stats && t == 0) *(float2 *)(a.stats + 2 * row) = float2{mean, rstd};
        }
    }
}

struct NormBwd {
    const void *dy, *x;
    const int8_t *codes;
    const float *scales, *stats;
    const void *w;
    void *dx;
    float *partial;             // (workgroups, 2, D): dw, db over a workgroup's rows
    int64_t rows;
    int32_t D;
    float inv_d;
    int32_t param_f32;
};

// A lane keeps 8 columns (K vectors) of its row and, over all rows it walks, of dw and db, and requests the next row while one
// is worked on: 16 waves a CU with two rows each in flight.  (16 columns a lane leave room for 8 waves: 15009 x 2560 f16 51 us
// instead of 49, 32768 x 8192 from 8 bits 382 instead of 328, 16384 x 4096 bf16 80 and 79.)  Above 8192 columns it has 32, and registers for neither the
// next row nor w.
template <typename T, int TPR, int K, bool BITS8, bool TAIL, bool STREAM>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void layer_norm_bwd_kernel(NormBwd a)
{
    constexpr int V = kVec<T>, THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
    constexpr bool AHEAD = K * V <= 8;
    __shared__ float slots[2][2 * THREADS / kWave];
    __shared__ float sums[GROUPS > 1 ? 2 * TPR * K * V : 1];
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, D = a.D;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + group;
    const int64_t nb = (D + kBlock8 - 1) / kBlock8;

    u32x4 next_dy[K], next_x[BITS8 ? 1 : K];
    u32x2 next_codes[BITS8 ? K : 1];
    float next_scale[BITS8 ? K : 1];
    float2 next_stats = {0.f, 0.f};
    const auto request = [&](int64_t r) {
        next_stats = *(const float2 *)(a.stats + 2 * r);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * TPR + t) * V;
            next_dy[k] = load_row_vec<T, TAIL, STREAM>((const T *)a.dy + r * D, c, D);
            if constexpr (BITS8) {
                next_codes[k] = load_codes8<V, TAIL, STREAM>(a.codes + r * D, c, D);
                next_scale[k] = c < D ? a.scales[r * nb + c / kBlock8] : 0.f;
            } else {
                next_x[k] = load_row_vec<T, TAIL, STREAM>((const T *)a.x + r * D, c, D);
            }
        }
    };
    // the row's dy and xh of vector k (absent columns: dy = 0, which makes them count for nothing)
    const auto values = [&](int k, float (&dy)[V], float (&xh)[V], float mean, float rstd) {
        unpack_vec(next_dy[k], dy, T{});
        if constexpr (BITS8) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) values8(next_codes[k][i], next_scale[k], xh + 4 * i);
        } else {
            unpack_vec(next_x[k], xh, T{});
        }
#pragma unroll
        for (int i = 0; i < V; ++i) xh[i] = (xh[i] - mean) * rstd;
    };
    const auto weights = [&](int k, float (&w)[V]) { load_param<T, TAIL>(a.w, a.param_f32, (k * TPR + t) * V, D, 1.f, w); };
    float w[AHEAD ? K : 1][V], dw[K][V], db[K][V];
    if constexpr (AHEAD) {
        if (row < a.rows) request(row);
#pragma unroll
        for (int k = 0; k < K; ++k) weights(k, w[k]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
    for (int64_t base = (int64_t)blockIdx.x * GROUPS, turn = 0; base < a.rows; base += step, row += step, ++turn) {
        const bool here = row < a.rows;
        if (!AHEAD && here) request(row);
        float dy[AHEAD ? K : 1][V], xh[AHEAD ? K : 1][V];
        const float mean = next_stats.x, rstd = next_stats.y;
        if constexpr (AHEAD) {
#pragma unroll
            for (int k = 0; k < K; ++k) values(k, dy[k], xh[k], mean, rstd);
            if (row + step < a.rows) request(row + step);
        }
        float s[2] = {0.f, 0.f};
        if (here) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int at = AHEAD ? k : 0;
                if constexpr (!AHEAD) {
                    values(k, dy[0], xh[0], mean, rstd);
                    weights(k, w[0]);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float g = dy[at][i] * w[at][i];
                    s[0] += g;
                    s[1] = fmaf(g, xh[at][i], s[1]);
                    dw[k][i] = fmaf(dy[at][i], xh[at][i], dw[k][i]);
                    db[k][i] += dy[at][i];
                }
            }
        }
        row_sum<TPR, 2>(s, slots[turn & 1]);
        if (here) {
            const float c1 = s[0] * a.inv_d, c2 = s[1] * a.inv_d;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int at = AHEAD ? k : 0;
                if constexpr (!AHEAD) {
                    asm volatile("" : "+v"(next_dy[k]));        // converted again here, not kept in fp32 over the barrier
                    if constexpr (BITS8) asm volatile("" : "+v"(next_codes[k]));
                    else asm volatile("" : "+v"(next_x[k]));
                    values(k, dy[0], xh[0], mean, rstd);
                    weights(k, w[0]);
                }
                float dx[V];
#pragma unroll
                for (int i = 0; i < V; ++i) dx[i] = rstd * (fmaf(dy[at][i], w[at][i], -c1) - xh[at][i] * c2);
                store_row_vec<T, TAIL, STREAM>((T *)a.dx + row * D, (k * TPR + t) * V, D, dx);
            }
        }
    }
    if (!a.partial) return;
    // groups after the first hand their sums over, one group after the other
    if constexpr (GROUPS > 1) {
#pragma unroll 1
        for (int g = 1; g < GROUPS; ++g) {
            __syncthreads();
            if (group == g) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        sums[(k * V + i) * TPR + t] = dw[k][i];
                        sums[(K * V + k * V + i) * TPR + t] = db[k][i];
                    }
            }
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        dw[k][i] += sums[(k * V + i) * TPR + t];
                        db[k][i] += sums[(K * V + k * V + i) * TPR + t];
                    }
            }
        }
    }
    if (group == 0) {
        float *to = a.partial + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = (k * TPR + t) * V + i;
                if (c < D) {
                    to[c] = dw[k][i];
                    to[D + c] = db[k][i];
                }
            }
    }
}

// dw and db from the workgroups' partial sums, in a fixed order: 32 columns a workgroup, 32 threads a column.  (A few megabytes, so
// what counts is that all of them are on the way at once: 512 sets of 4096 columns 9.3 us with 64 columns and 16 threads, 4.0 now.)
template <typename P> __global__ __launch_bounds__(1024) void layer_norm_reduce_kernel(const float *partial, int n, int D, P *dw, P *db)
{
    __shared__ float part[32][33];
    const int lane = threadIdx.x % 32, slice = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < 2 * D) {
#pragma unroll 8
        for (int i = slice; i < n; i += 32) s += partial[(int64_t)i * 2 * D + c];
    }
    part[slice][lane] = s;
    __syncthreads();
    s = part[lane][slice];
#pragma unroll
    for (int d = 16; d > 0; d /= 2) s += __shfl_xor(s, d);
    const int out = blockIdx.x * 32 + slice;
    if (lane == 0 && out < 2 * D) {
        P *to = out < D ? dw : db;
        if (to) Elem<P>::store(to + (out < D ? out : out - D), s);
    }
}

// Lanes of a row and vectors of a lane: forward up to 32 (fp32: 16) columns a lane, backward 8 (32 above 8192
// columns), whose sums dw and db it keeps too.
template <typename T, int TPR, int K, bool BITS8> int fwd_launch(const NormFwd &a, hipStream_t st)
{
    constexpr int THREADS = TPR > 256 ? TPR : 256;
    const int64_t need = (a.rows + THREADS / TPR - 1) / (THREADS / TPR), most = 256 * 2048 / THREADS;
    const dim3 grid((unsigned)(need < most ? need : most)), block(THREADS);
    const bool tail = a.D % kVec<T>, stream = a.rows * a.D * (int64_t)sizeof(T) > kStreamBytes;
    if (tail) {
        return stream ? launch_main(layer_norm_fwd_kernel<T, TPR, K, BITS8, true, true>, grid, block, st, a)
                      : launch_main(layer_norm_fwd_kernel<T, TPR, K, BITS8, true, false>, grid, block, st, a);
    }
    return stream ? launch_main(layer_norm_fwd_kernel<T, TPR, K, BITS8, false, true>, grid, block, st, a)
                  : launch_main(layer_norm_fwd_kernel<T, TPR, K, BITS8, false, false>, grid, block, st, a);
}
template <typename T, bool BITS8> int fwd_width(const NormFwd &a, hipStream_t st)
{
    const int vecs = (a.D + kVec<T> - 1) / kVec<T>;
    if (vecs <= 64) return fwd_launch<T, 64, 1, BITS8>(a, st);
    if (vecs <= 128) return fwd_launch<T, 64, 2, BITS8>(a, st);
    if (vecs <= 256) return fwd_launch<T, 64, 4, BITS8>(a, st);
    if (vecs <= 512) return fwd_launch<T, 256, 2, BITS8>(a, st);
    if (vecs <= 1024) return fwd_launch<T, 256, 4, BITS8>(a, st);
    // at most 16384 columns
    return fwd_launch<T, 1024, 16 / kVec<T>, BITS8>(a, st);
}
template <typename T> int fwd_t(const NormFwd &a, hipStream_t st) { return a.codes ? fwd_width<T, true>(a, st) : fwd_width<T, false>(a, st); }

// lanes that hold a row of the backward
int bwd_lanes(int D)
{
    int tpr = 64;
    while (tpr * 8 < D && tpr < 1024) tpr *= 2;
    return D > 8192 ? 512 : tpr;
}
// Workgroups of the backward, each of which writes a set of partial sums: two a CU, one of 1024 threads.
int bwd_blocks(int64_t rows, int D)
{
    const int tpr = bwd_lanes(D), threads = tpr > 256 ? tpr : 256;
    const int64_t need = (rows + threads / tpr - 1) / (threads / tpr), most = threads >= 1024 || D > 8192 ? 256 : 512;
    return (int)(need < most ? need : most);
}
template <typename T, int TPR, bool BITS8, int COLUMNS = 8> int bwd_launch(const NormBwd &a, hipStream_t st)
{
    constexpr int K = COLUMNS / kVec<T>;
    const dim3 grid((unsigned)bwd_blocks(a.rows, a.D)), block(TPR > 256 ? TPR : 256);
    const bool tail = a.D % kVec<T>, stream = a.rows * a.D * (int64_t)sizeof(T) > kStreamBytes;
    if (tail) {
        return stream ? launch_main(layer_norm_bwd_kernel<T, TPR, K, BITS8, true, true>, grid, block, st, a)
                      : launch_main(layer_norm_bwd_kernel<T, TPR, K, BITS8, true, false>, grid, block, st, a);
    }
    return stream ? launch_main(layer_norm_bwd_kernel<T, TPR, K, BITS8, false, true>, grid, block, st, a)
                  : launch_main(layer_norm_bwd_kernel<T, TPR, K, BITS8, false, false>, grid, block, st, a);
}
template <typename T, bool BITS8> int bwd_width(const NormBwd &a, hipStream_t st)
{
    switch (bwd_lanes(a.D)) {
    case 64: return bwd_launch<T, 64, BITS8>(a, st);
    case 128: return bwd_launch<T, 128, BITS8>(a, st);
    case 256: return bwd_launch<T, 256, BITS8>(a, st);
    case 512: return a.D <= 8192 ? bwd_launch<T, 512, BITS8>(a, st) : bwd_launch<T, 512, BITS8, 32>(a, st);
    default: return bwd_launch<T, 1024, BITS8>(a, st);
    }
}
template <typename T> int bwd_t(const NormBwd &a, hipStream_t st) { return a.codes ? bwd_width<T, true>(a, st) : bwd_width<T, false>(a, st); }

int tensor_code(int dtype) { return dtype == GCG_BF16_F32 ? GCG_BF16 : dtype == GCG_F16_F32 ? GCG_F16 : dtype; }

} // namespace

size_t layer_norm_bwd_workspace(int64_t rows, int D) { return (size_t)bwd_blocks(rows, D) * 2 * D * sizeof(float); }

int layer_norm_fwd_launch(int dtype, const void *x, const void *w, const void *b, void *y, float *stats, int8_t *codes, float *scales,
                          int64_t rows, int D, float eps, hipStream_t st)
{
    const NormFwd a = {x, w, b, y, stats, codes, scales, rows, D, 1.0f / (float)D, eps, tensor_code(dtype) != dtype};
    switch (tensor_code(dtype)) {
    case GCG_F32: return fwd_t<float>(a, st);
    case GCG_BF16: return fwd_t<bf16_t>(a, st);
    default: return fwd_t<f16_t>(a, st);
    }
}

int layer_norm_bwd_launch(int dtype, const void *dy, const void *x, const int8_t *codes, const float *scales, const float *stats,
                          const void *w, void *dx, void *dw, void *db, void *ws, int64_t rows, int D, hipStream_t st)
{
    const NormBwd a = {dy, x, codes, scales, stats, w, dx, dw || db ? (float *)ws : nullptr, rows, D, 1.0f / (float)D,
                       tensor_code(dtype) != dtype};
    int rc;
    switch (tensor_code(dtype)) {
    case GCG_F32: rc = bwd_t<float>(a, st); break;
    case GCG_BF16: rc = bwd_t<bf16_t>(a, st); break;
    default: rc = bwd_t<f16_t>(a, st); break;
    }
    if (rc || !a.partial) return rc;
    const dim3 grid((unsigned)((2 * D + 31) / 32)), block(1024);
    const int n = bwd_blocks(rows, D);
    switch (dtype) {
    case GCG_BF16: return launch_plain(layer_norm_reduce_kernel<bf16_t>, grid, block, st, (const float *)ws, n, D, (bf16_t *)dw, (bf16_t *)db);
    case GCG_F16: return launch_plain(layer_norm_reduce_kernel<f16_t>, grid, block, st, (const float *)ws, n, D, (f16_t *)dw, (f16_t *)db);
    default: return launch_plain(layer_norm_reduce_kernel<float>, grid, block, st, (const float *)ws, n, D, (float *)dw, (float *)db);
    }
}

} // namespace gcg
