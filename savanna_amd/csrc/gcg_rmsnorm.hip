// Root-mean-square norm of a residual sum, forward and backward, with its output in the tensors' type or in 8-bit floating point.
//
//   r = x + residual (rounded to the type), rstd = (sum r^2 / D + eps)^-1/2, y = r rstd w
//   g = dy w, xh = r rstd;  dr' = rstd (g - xh mean(g xh)) + dr;  dw = sum over rows of dy xh
//
// where dr is the gradient that reaches r along the residual stream, and dr' that of x and of residual.  Bound by memory: with the
// residual 4 s bytes an element forward (s the element's size; 3 s + 1 into 8 bits) and 4 s backward, for some ten vector
// instructions.  A row is held in the registers of TPR lanes, so that it is read once, and the next row's loads are in flight while one is
// worked on; a row of one wave needs no barrier.  All sums are fp32; r is rounded before it is normed, since it is what the
// backward and the next layer read.  The 8-bit output is formed of y in fp32, each block's largest by lane exchanges.
//
// Measured: 16384 x 4096 bf16 with the residual forward 87 us (6.0 TB/s), backward 112 + 4 (4.7); 16384 x 8192 into 8 bits 169 (5.5); 15325 x 2358, whose
// rows end inside a vector, 56 (5.1) and 59 + 4 (4.9; with that vector loaded in a branch, which keeps the next row from being under way, 96 and 152);
// 8 x 4096 3.3, a launch.
#include "gcg_float8.h"

namespace gcg {
namespace {

struct RmsFwd {
    const void *x, *residual, *w;
    void *y, *r;
    uint8_t *codes, *scales;    // the output in 8 bits, in y's place
    float *rstd;                // (rows), or null
    int64_t rows;
    int32_t D, Dp, S;
    float inv_d, eps;
    int32_t param_f32;
};

template <typename T, int TPR, int K, bool RES, bool OUT8, bool TAIL, bool STREAM>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_norm_fwd_kernel(RmsFwd a)
{
    constexpr int V = kVec<T>, THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
    __shared__ float slots[2][THREADS / kWave];
    const int t = threadIdx.x % TPR, D = a.D;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / TPR;

    u32x4 next[K], next_res[RES ? K : 1];
    const auto request = [&](int64_t r) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            next[k] = request_row_vec<T, TAIL, STREAM>((const T *)a.x + r * D, (k * TPR + t) * V, D);
            if constexpr (RES) next_res[k] = request_row_vec<T, TAIL, STREAM>((const T *)a.residual + r * D, (k * TPR + t) * V, D);
        }
    };
#pragma unroll
    for (int k = 0; k < K; ++k) {
        next[k] = u32x4{0, 0, 0, 0};
        if constexpr (RES) next_res[k] = next[k];
    }
    if (row < a.rows) request(row);
    float w[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) load_param<T, TAIL>(a.w, a.param_f32, (k * TPR + t) * V, D, 1.f, w[k]);
    // every group of the workgroup goes through the same number of turns, so that all meet at the barriers
    for (int64_t base = (int64_t)blockIdx.x * GROUPS, turn = 0; base < a.rows; base += step, row += step, ++turn) {
        float v[K][V], s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            unpack_vec(in_place<T, TAIL>(next[k], (k * TPR + t) * V, D), v[k], T{});
            if constexpr (RES) {
                float q[V];
                unpack_vec(in_place<T, TAIL>(next_res[k], (k * TPR + t) * V, D), q, T{});
#pragma unroll
                for (int i = 0; i < V; ++i) v[k][i] += q[i];
                if (row < a.rows) store_row_vec<T, TAIL, STREAM>((T *)a.r + row * D, (k * TPR + t) * V, D, v[k]);
                unpack_vec(pack_vec(v[k], T{}), v[k], T{});
            }
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] = fmaf(v[k][i], v[k][i], s[0]);
        }
        if (row + step < a.rows) request(row + step);
        row_sum<TPR, 1>(s, slots[turn & 1]);
        const float rstd = 1.0f / sqrtf(s[0] * a.inv_d + a.eps);
        if (row < a.rows) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * TPR + t) * V;
                float y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = v[k][i] * rstd * w[k][i];
                if constexpr (OUT8) store_f8<V, false, STREAM>(a.codes + row * a.Dp, a.scales + row * a.S, c, a.Dp, y);
                else store_row_vec<T, TAIL, STREAM>((T *)a.y + row * D, c, D, y);
            }
            if constexpr (OUT8) {
                if (t < a.S - a.Dp / kBlockF8) a.scales[row * a.S + a.Dp / kBlockF8 + t] = 127;
            }
            if (a.rstd && t == 0) a.rstd[row] = rstd;
        }
    }
}

struct RmsBwd {
    const void *dy, *r, *dr;
    const float *rstd;
    const void *w;
    void *dx;
    float *partial;             // (workgroups, D): dw over a workgroup's rows
    int64_t rows;
    int32_t D;
    float inv_d;
    int32_t param_f32;
};

// A lane keeps 8 columns (K vectors) of its row and, over all rows it walks, of dw, and requests the next row while one is
// worked on.  Above 8192 columns it has 32, and registers for neither the next row nor w nor dr.
template <typename T, int TPR, int K, bool ADD, bool TAIL, bool STREAM>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void rms_norm_bwd_kernel(RmsBwd a)
{
    constexpr int V = kVec<T>, THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
    constexpr bool AHEAD = K * V <= 8;
    __shared__ float slots[2][THREADS / kWave];
    __shared__ float sums[GROUPS > 1 ? TPR * K * V : 1];
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR, D = a.D;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t row = (int64_t)blockIdx.x * GROUPS + group;

    // (without requests ahead a row is waited for anyway)
    constexpr bool PLACE = TAIL && AHEAD;
    const auto load = [&](const void *p, int64_t r, int c) {
        if constexpr (PLACE) return request_row_vec<T, true, STREAM>((const T *)p + r * D, c, D);
        else return load_row_vec<T, TAIL, STREAM>((const T *)p + r * D, c, D);
    };
    u32x4 next_dy[K], next_r[K], next_dr[ADD && AHEAD ? K : 1];
    float next_rstd = 0.f;
    const auto request = [&](int64_t r) {
        next_rstd = a.rstd[r];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * TPR + t) * V;
            next_dy[k] = load(a.dy, r, c);
            next_r[k] = load(a.r, r, c);
            if constexpr (ADD && AHEAD) next_dr[k] = load(a.dr, r, c);
        }
    };
    // the row's dy and xh of vector k (absent columns: zeros, which count for nothing)
    const auto values = [&](int k, float (&dy)[V], float (&xh)[V], float rstd) {
        unpack_vec(in_place<T, PLACE>(next_dy[k], (k * TPR + t) * V, D), dy, T{});
        unpack_vec(in_place<T, PLACE>(next_r[k], (k * TPR + t) * V, D), xh, T{});
#pragma unroll
        for (int i = 0; i < V; ++i) xh[i] *= rstd;
    };
    const auto weights = [&](int k, float (&w)[V]) { load_param<T, TAIL>(a.w, a.param_f32, (k * TPR + t) * V, D, 1.f, w); };
    float w[AHEAD ? K : 1][V], dw[K][V];
    if constexpr (AHEAD) {
        if (row < a.rows) request(row);
#pragma unroll
        for (int k = 0; k < K; ++k) weights(k, w[k]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = 0.f;
    for (int64_t base = (int64_t)blockIdx.x * GROUPS, turn = 0; base < a.rows; base += step, row += step, ++turn) {
        const bool here = row < a.rows;
        if (!AHEAD && here) request(row);
        float dy[AHEAD ? K : 1][V], xh[AHEAD ? K : 1][V];
        u32x4 dr[AHEAD && ADD ? K : 1];
        const float rstd = next_rstd;
        if constexpr (AHEAD) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                values(k, dy[k], xh[k], rstd);
                if constexpr (ADD) dr[k] = next_dr[k];
            }
            if (row + step < a.rows) request(row + step);
        }
        float s[1] = {0.f};
        if (here) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int at = AHEAD ? k : 0;
                if constexpr (!AHEAD) {
                    values(k, dy[0], xh[0], rstd);
                    weights(k, w[0]);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s[0] = fmaf(dy[at][i] * w[at][i], xh[at][i], s[0]);
                    dw[k][i] = fmaf(dy[at][i], xh[at][i], dw[k][i]);
                }
            }
        }
        row_sum<TPR, 1>(s, slots[turn & 1]);
        if (here) {
            const float c2 = s[0] * a.inv_d;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int at = AHEAD ? k : 0;
                if constexpr (!AHEAD) {
                    asm volatile("" : "+v"(next_dy[k]));        // converted again here, not kept in fp32 over the barrier
                    asm volatile("" : "+v"(next_r[k]));
                    values(k, dy[0], xh[0], rstd);
                    weights(k, w[0]);
                }
                float dx[V], more[V];
                if constexpr (ADD && AHEAD) unpack_vec(in_place<T, PLACE>(dr[at], (k * TPR + t) * V, D), more, T{});
                else if constexpr (ADD) unpack_vec(load_row_vec<T, TAIL, STREAM>((const T *)a.dr + row * D, (k * TPR + t) * V, D), more, T{});
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    dx[i] = rstd * (dy[at][i] * w[at][i] - xh[at][i] * c2);
                    if constexpr (ADD) dx[i] += more[i];
                }
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
                    for (int i = 0; i < V; ++i) sums[(k * V + i) * TPR + t] = dw[k][i];
            }
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) dw[k][i] += sums[(k * V + i) * TPR + t];
            }
        }
    }
    if (group == 0) {
        float *to = a.partial + (int64_t)blockIdx.x * D;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = (k * TPR + t) * V + i;
                if (c < D) to[c] = dw[k][i];
            }
    }
}

// dw from the workgroups' partial sums, in a fixed order: 32 columns a workgroup, 32 threads a column
template <typename P> __global__ __launch_bounds__(1024) void rms_norm_reduce_kernel(const float *partial, int n, int D, P *dw)
{
    __shared__ float part[32][33];
    const int lane = threadIdx.x % 32, slice = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < D) {
#pragma unroll 8
        for (int i = slice; i < n; i += 32) s += partial[(int64_t)i * D + c];
    }
    part[slice][lane] = s;
    __syncthreads();
    s = part[lane][slice];
#pragma unroll
    for (int d = 16; d > 0; d /= 2) s += __shfl_xor(s, d);
    const int out = blockIdx.x * 32 + slice;
    if (lane == 0 && out < D) Elem<P>::store(dw + out, s);
}

// Lanes of a row and vectors of a lane, as in the layer norm's kernels.  Rows that end inside a vector go without the streaming hint.
template <typename T, int TPR, int K, bool RES, bool OUT8> int fwd_launch(const RmsFwd &a, hipStream_t st)
{
    constexpr int THREADS = TPR > 256 ? TPR : 256;
    const int64_t need = (a.rows + THREADS / TPR - 1) / (THREADS / TPR), most = 256 * 2048 / THREADS;
    const dim3 grid((unsigned)(need < most ? need : most)), block(THREADS);
    if (a.D % kVec<T>) return launch_main(rms_norm_fwd_kernel<T, TPR, K, RES, OUT8, true, false>, grid, block, st, a);
    return a.rows * a.D * (int64_t)sizeof(T) > kStreamBytes
               ? launch_main(rms_norm_fwd_kernel<T, TPR, K, RES, OUT8, false, true>, grid, block, st, a)
               : launch_main(rms_norm_fwd_kernel<T, TPR, K, RES, OUT8, false, false>, grid, block, st, a);
}
template <typename T, bool RES, bool OUT8> int fwd_width(const RmsFwd &a, hipStream_t st)
{
    const int vecs = (a.D + kVec<T> - 1) / kVec<T>;
    if (vecs <= 64) return fwd_launch<T, 64, 1, RES, OUT8>(a, st);
    if (vecs <= 128) return fwd_launch<T, 64, 2, RES, OUT8>(a, st);
    if (vecs <= 256) return fwd_launch<T, 64, 4, RES, OUT8>(a, st);
    if (vecs <= 512) return fwd_launch<T, 256, 2, RES, OUT8>(a, st);
    if (vecs <= 1024) return fwd_launch<T, 256, 4, RES, OUT8>(a, st);
    // at most 16384 columns
    return fwd_launch<T, 1024, 16 / kVec<T>, RES, OUT8>(a, st);
}
template <typename T> int fwd_t(const RmsFwd &a, hipStream_t st)
{
    if (a.codes) return a.residual ? fwd_width<T, true, true>(a, st) : fwd_width<T, false, true>(a, st);
    return a.residual ? fwd_width<T, true, false>(a, st) : fwd_width<T, false, false>(a, st);
}

// lanes that hold a row of the backward, and its workgroups, each of which writes a set of partial sums
int bwd_lanes(int D)
{
    int tpr = 64;
    while (tpr * 8 < D && tpr < 1024) tpr *= 2;
    return D > 8192 ? 512 : tpr;
}
int bwd_blocks(int64_t rows, int D)
{
    const int tpr = bwd_lanes(D), threads = tpr > 256 ? tpr : 256;
    const int64_t need = (rows + threads / tpr - 1) / (threads / tpr), most = threads >= 1024 || D > 8192 ? 256 : 512;
    return (int)(need < most ? need : most);
}
template <typename T, int TPR, bool ADD, int COLUMNS = 8> int bwd_launch(const RmsBwd &a, hipStream_t st)
{
    constexpr int K = COLUMNS / kVec<T>;
    const dim3 grid((unsigned)bwd_blocks(a.rows, a.D)), block(TPR > 256 ? TPR : 256);
    if (a.D % kVec<T>) return launch_main(rms_norm_bwd_kernel<T, TPR, K, ADD, true, false>, grid, block, st, a);
    return a.rows * a.D * (int64_t)sizeof(T) > kStreamBytes ? launch_main(rms_norm_bwd_kernel<T, TPR, K, ADD, false, true>, grid, block, st, a)
                                                            : launch_main(rms_norm_bwd_kernel<T, TPR, K, ADD, false, false>, grid, block, st, a);
}
template <typename T, bool ADD> int bwd_width(const RmsBwd &a, hipStream_t st)
{
    switch (bwd_lanes(a.D)) {
    case 64: return bwd_launch<T, 64, ADD>(a, st);
    case 128: return bwd_launch<T, 128, ADD>(a, st);
    case 256: return bwd_launch<T, 256, ADD>(a, st);
    case 512: return a.D <= 8192 ? bwd_launch<T, 512, ADD>(a, st) : bwd_launch<T, 512, ADD, 32>(a, st);
    default: return bwd_launch<T, 1024, ADD>(a, st);
    }
}
template <typename T> int bwd_t(const RmsBwd &a, hipStream_t st) { return a.dr ? bwd_width<T, true>(a, st) : bwd_width<T, false>(a, st); }

int tensor_code(int dtype) { return dtype == GCG_BF16_F32 ? GCG_BF16 : dtype == GCG_F16_F32 ? GCG_F16 : dtype; }

} // namespace

size_t rms_norm_bwd_workspace(int64_t rows, int D) { return (size_t)bwd_blocks(rows, D) * D * sizeof(float); }

int rms_norm_fwd_launch(int dtype, const void *x, const void *residual, const void *w, void *y, void *r, uint8_t *codes, uint8_t *scales,
                        float *rstd, int64_t rows, int D, float eps, hipStream_t st)
{
    const RmsFwd a = {x, residual, w, y, r, codes, scales, rstd, rows, D, (int32_t)f8_cols(D), (int32_t)f8_scales(D), 1.0f / (float)D, eps,
                      tensor_code(dtype) != dtype};
    switch (tensor_code(dtype)) {
    case GCG_F32: return fwd_t<float>(a, st);
    case GCG_BF16: return fwd_t<bf16_t>(a, st);
    default: return fwd_t<f16_t>(a, st);
    }
}

int rms_norm_bwd_launch(int dtype, const void *dy, const void *r, const void *dr, const float *rstd, const void *w, void *dx, void *dw,
                        void *ws, int64_t rows, int D, hipStream_t st)
{
    const RmsBwd a = {dy, r, dr, rstd, w, dx, dw ? (float *)ws : nullptr, rows, D, 1.0f / (float)D, tensor_code(dtype) != dtype};
    int rc;
    switch (tensor_code(dtype)) {
    case GCG_F32: rc = bwd_t<float>(a, st); break;
    case GCG_BF16: rc = bwd_t<bf16_t>(a, st); break;
    default: rc = bwd_t<f16_t>(a, st); break;
    }
    if (rc || !a.partial) return rc;
    const dim3 grid((unsigned)((D + 31) / 32)), block(1024);
    const int n = bwd_blocks(rows, D);
    switch (dtype) {
    case GCG_BF16: return launch_plain(rms_norm_reduce_kernel<bf16_t>, grid, block, st, (const float *)ws, n, D, (bf16_t *)dw);
    case GCG_F16: return launch_plain(rms_norm_reduce_kernel<f16_t>, grid, block, st, (const float *)ws, n, D, (f16_t *)dw);
    default: return launch_plain(rms_norm_reduce_kernel<float>, grid, block, st, (const float *)ws, n, D, (float *)dw);
    }
}

} // namespace gcg
