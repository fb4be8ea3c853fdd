// Gated linear recurrence, channel by channel: a decay that the data choose, and an output gate.
//
//   a_t = sigmoid(f_t + bias),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = gate_t h_t
//   backward, from the last row: G_t = gate_t dy_t + K_t,  K_{t-1} = a_t G_t  (K of the last row: the final state's gradient),
//   dgate_t = dy_t h_t,  dx_t = (1 - a_t) G_t,  df_t = G_t (h_{t-1} - x_t) a_t (1 - a_t),  dbias = sum df,  dh_0 = K before the first row
//
// Bound by memory: 4 s bytes an element forward (x, f, gate, y; s the element's size) and 7 s backward, for some 25 and 50 vector
// instructions, if every tensor is read once.  A recurrence from row to row would leave the card empty, so time is cut into chunks, and
// a chunk's rows stay in registers from the first reading on: a row's step h -> a h + u is a pair (a, u), pairs combine, and
//   1. each of a workgroup's waves (a slot: R rows of 64 lanes) combines its rows, the workgroup its slots, through shared memory;
//   2. the chunk's pair is published, and the state that enters it is put together of the pairs published before it;
//   3. the rows are gone through once more, from that state.
// Chunks form groups.  The last chunk of a group also publishes the state behind it, and a chunk waits for the state before its group and for
// the pairs of the chunks before it in the group, always the same ones in the same order: results are the same on every run.  A
// word of 64 bits holds a pair (or a state) and says by its upper half that it is there, so no fence orders anything.
// Workgroups take their chunks in the order of a ticket, chunks of the same time first, so whoever waits, waits for workgroups that took their
// tickets earlier, are at work, and wait for earlier ones at most: every wait ends.
//
// Measured: 2 x 8192 x 4096 bf16 forward 117 us (4.7 TB/s), backward 204 + 4 for the bias (4.8), and 4 + 6 for clearing the words; 1 x 131072 x 512 fp32
// forward 193 (5.6); 4 x 701 x 2560 f16 16 (15.3 to 17.6): one after the other, all rows' arrival, the sums, the words' way, and all rows' leaving.  Rows off
// the lines of memory take longer, and those on 2 bytes, one channel a lane, longest: of 4096, 4094, 4095 channels forward 119, 148, 168, backward 205, 291,
// 369, with the clearing.  A token of 64, 256, 512, 1024 x 8192 bf16, launches
// after each other on the same tensors: 4, 5.6, 13, 22.
//
// The backward needs the states inside a chunk again; the forward keeps the one before every kChunk rows (1 / 32 of a
// 16-bit tensor), and the rest is made again from x and f, which it reads anyway.
#include "gcg_row.h"

namespace gcg {
namespace {

constexpr int kChunk = 64;              // rows between kept states, and of a chunk of the backward

// ---- elements -----------------------------------------------------------------------------------------------------------
// A lane has C channels side by side: two of 16 bits where rows lie on 4 bytes, else one.
template <typename T, int C> __device__ __forceinline__ uint32_t load_channels(win_t w, uint32_t off)
{
    if constexpr (C * sizeof(T) == 4) return win_load_aux<WIN_NT, uint32_t>(w, off);
    else return win_load_u16(w, off);
}
__device__ __forceinline__ void channels(uint32_t r, float (&v)[1], float) { v[0] = __uint_as_float(r); }
template <int C> __device__ __forceinline__ void channels(uint32_t r, float (&v)[C], bf16_t)
{
    v[0] = __uint_as_float(r << 16);
    if constexpr (C == 2) v[1] = __uint_as_float(r & 0xffff0000u);
}
template <int C> __device__ __forceinline__ void channels(uint32_t r, float (&v)[C], f16_t)
{
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    h2 h;
    __builtin_memcpy(&h, &r, 4);
    v[0] = (float)h[0];
    if constexpr (C == 2) v[1] = (float)h[1];
}
__device__ __forceinline__ void store_channels(win_t w, uint32_t off, const float (&v)[1], float) { win_store(w, off, __float_as_uint(v[0])); }
template <int C> __device__ __forceinline__ void store_channels(win_t w, uint32_t off, const float (&v)[C], bf16_t)
{
    if constexpr (C == 2) win_store(w, off, pack_bf16x2(v[0], v[1]));
    else __builtin_amdgcn_raw_buffer_store_b16((short)float_to_bf16_bits(v[0]), w, (int)off, 0, WIN_NT_ST);
}
template <int C> __device__ __forceinline__ void store_channels(win_t w, uint32_t off, const float (&v)[C], f16_t)
{
    if constexpr (C == 2) win_store(w, off, pack_f16x2(v[0], v[1]));
    else {
        const _Float16 h = (_Float16)v[0];
        short s;
        __builtin_memcpy(&s, &h, 2);
        __builtin_amdgcn_raw_buffer_store_b16(s, w, (int)off, 0, WIN_NT_ST);
    }
}

// a = sigmoid(z) and b = 1 - a = sigmoid(-z): with e = exp(-|z|) the smaller is e / (1 + e), the larger 1 less it, to half a unit of its last bit.  (As
// a reciprocal of its own, a whole unit off, it takes 1e-6 from a state in some hundred rows: the decays multiply.)  EXACT (fp32 tensors): what
// the rounding of |z| log2(e) takes from e is put back.
template <bool EXACT> __device__ __forceinline__ void sigmoids(float z, float &a, float &b)
{
    const float m = fmaxf(-fabsf(z), -200.f), t = m * 1.44269504f;
    float e = __builtin_amdgcn_exp2f(t);
    if constexpr (EXACT) e = fmaf(e * 0.693147181f, fmaf(m, 1.44269504f, -t), e);
    const float s = e * __builtin_amdgcn_rcpf(1.f + e), l = 1.f - s;
    a = z < 0.f ? s : l;
    b = z < 0.f ? l : s;
    if (z != z) a = b = z;
}

// ---- pairs between workgroups ------------------------------------------------------------------------------------------------
// The pair (A, H) of h -> A h + H, A in [0, 1], with the sign of A set where it is there (memory is cleared to zeros first).
__device__ __forceinline__ uint64_t word_of(float A, float H)
{
    return (uint64_t)(__float_as_uint(A) | 0x80000000u) << 32 | __float_as_uint(H);
}
__device__ __forceinline__ float word_A(uint64_t w) { return __uint_as_float((uint32_t)(w >> 32) & 0x7fffffffu); }
__device__ __forceinline__ float word_H(uint64_t w) { return __uint_as_float((uint32_t)w); }
__device__ __forceinline__ void publish(uint64_t *p, uint64_t w) { __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t look(const uint64_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t wait_for(const uint64_t *p, uint64_t w)
{
    while ((uint32_t)(w >> 32) == 0) {
        __builtin_amdgcn_s_sleep(2);
        w = look(p);
    }
    return w;
}
// A product of decays that left fp32 stays the smallest normal number, unless one of them was zero: 0 times an infinite state is NaN
__device__ __forceinline__ float kept_decay(float A, float least) { return least > 0.f ? fmaxf(A, 0x1p-126f) : A; }

struct ScanTensor { const void *p; int64_t batch, time; };      // strides in elements
struct Scan {
    ScanTensor x, f, gate, dy, y, dx, df, dgate;                // forward: x, f, gate, y
    const float *bias, *initial, *dfinal;
    const int32_t *lengths;
    float *final, *states, *dinitial, *partial;
    uint64_t *pairs, *carries;                                  // (bs, chunks, D), (bs, groups, D); null with one chunk
    uint32_t *ticket;
    int64_t L;
    int32_t D, bs, cols, chunks, group, kept;                   // kept: states of a batch entry
};

// what a workgroup works on
struct Place { int c, b, col; };
__device__ __forceinline__ Place place_of(const Scan &p, uint32_t *shared, bool backward)
{
    uint32_t id = blockIdx.x;
    if (p.ticket) {
        if (threadIdx.x == 0) *shared = __hip_atomic_fetch_add(p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        id = __builtin_amdgcn_readfirstlane(*shared);
    }
    const uint32_t per = (uint32_t)p.bs * p.cols, c = id / per, rest = id - c * per;
    return {backward ? p.chunks - 1 - (int)c : (int)c, (int)(rest / p.cols), (int)(rest % p.cols)};
}
template <typename T> __device__ __forceinline__ win_t window_of(const ScanTensor &t, int b, int64_t row, int rows, int D)
{
    return make_window((const T *)t.p + b * t.batch + row * t.time, rows > 0 ? ((int64_t)(rows - 1) * t.time + D) * (int64_t)sizeof(T) : 0);
}

// The pair (A, H) of the n pairs at first, first + step, ...: what a chunk's predecessors in its group do to the state.  (Put together before the
// state of the group's start is waited for, so that a state passes a group in the time of one word's way.)
template <int C> __device__ __forceinline__ void together(const uint64_t *first, int64_t step, int n, bool here, float (&A)[C], float (&H)[C])
{
    constexpr int B = 4 / C;
#pragma unroll
    for (int c = 0; c < C; ++c) { A[c] = 1.f; H[c] = 0.f; }
    for (int i = 0; i < n; i += B) {
        uint64_t w[B][C];
#pragma unroll
        for (int k = 0; k < B; ++k)
#pragma unroll
            for (int c = 0; c < C; ++c) w[k][c] = here && i + k < n ? look(first + (i + k) * step + c) : 1ull << 63;
#pragma unroll
        for (int k = 0; k < B; ++k)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                if (i + k < n) {
                    w[k][c] = wait_for(first + (i + k) * step + c, w[k][c]);
                    const float Ak = word_A(w[k][c]);
                    H[c] = fmaf(Ak, H[c], word_H(w[k][c]));
                    A[c] = kept_decay(A[c] * Ak, fminf(A[c], Ak));
                }
            }
    }
}

// ---- forward --------------------------------------------------------------------------------------------------------------------
template <typename T, int C, int R, int W, bool GATE> __global__ __launch_bounds__(W * 64, 4) void scan_fwd_kernel(Scan p)
{
    constexpr int ROWS = R * W, E = (int)sizeof(T);
    __shared__ float pairA[W][64 * C], pairH[W][64 * C], enter[64 * C];
    __shared__ uint32_t ticket;
    const int lane = threadIdx.x % 64, slot = threadIdx.x / 64;
    const Place at = place_of(p, &ticket, false);
    const int ch = (at.col * 64 + lane) * C;
    const bool here = ch < p.D;
    const int64_t t0 = (int64_t)at.c * ROWS;
    int64_t len = p.lengths ? p.lengths[at.b] : p.L;
    len = len < 0 ? 0 : len > p.L ? p.L : len;
    const int rows = (int)(len - t0 < ROWS ? (len - t0 > 0 ? len - t0 : 0) : ROWS);         // inside the sequence
    const int out_rows = (int)(p.L - t0 < ROWS ? p.L - t0 : ROWS);
    const uint32_t lane_off = here ? (uint32_t)(ch * E) : WIN_OFF;

    const win_t wx = window_of<T>(p.x, at.b, t0, rows, p.D), wf = window_of<T>(p.f, at.b, t0, rows, p.D);
    const win_t wg = window_of<T>(GATE ? p.gate : p.x, at.b, t0, rows, p.D), wy = window_of<T>(p.y, at.b, t0, out_rows, p.D);
    const uint32_t sx = (uint32_t)(p.x.time * E), sf = (uint32_t)(p.f.time * E), sg = (uint32_t)(p.gate.time * E), sy = (uint32_t)(p.y.time * E);
    uint32_t rx[R], rf[R], rg[GATE ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const uint32_t row = slot * R + i;
        rf[i] = load_channels<T, C>(wf, lane_off + row * sf);
        rx[i] = load_channels<T, C>(wx, lane_off + row * sx);
    }
    if constexpr (GATE) {
#pragma unroll
        for (int i = 0; i < R; ++i) rg[i] = load_channels<T, C>(wg, lane_off + (slot * R + i) * sg);
    }
    float bias[C];
#pragma unroll
    for (int c = 0; c < C; ++c) bias[c] = p.bias && here ? p.bias[ch + c] : 0.f;

    float a[R][C], u[R][C], A[C], H[C], least[C];
#pragma unroll
    for (int c = 0; c < C; ++c) { A[c] = 1.f; H[c] = 0.f; least[c] = 1.f; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float x[C], f[C];
        channels(rx[i], x, T{});
        channels(rf[i], f, T{});
        const bool inside = slot * R + i < rows;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float b;
            sigmoids<E == 4>(f[c] + bias[c], a[i][c], b);
            a[i][c] = inside ? a[i][c] : 1.f;
            u[i][c] = inside ? b * x[c] : 0.f;
            A[c] *= a[i][c];
            H[c] = fmaf(a[i][c], H[c], u[i][c]);
            least[c] = fminf(least[c], a[i][c]);
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        A[c] = kept_decay(A[c], least[c]);
        pairA[slot][lane * C + c] = A[c];
        pairH[slot][lane * C + c] = H[c];
    }
    __syncthreads();
    // the pair of the slots before this one
    float PA[C], PH[C];
#pragma unroll
    for (int c = 0; c < C; ++c) { PA[c] = 1.f; PH[c] = 0.f; }
    for (int s = 0; s < slot; ++s) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float As = pairA[s][lane * C + c];
            PH[c] = fmaf(As, PH[c], pairH[s][lane * C + c]);
            PA[c] = kept_decay(PA[c] * As, fminf(PA[c], As));
        }
    }
    if (slot == W - 1) {
        float TA[C], TH[C], h[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            TH[c] = fmaf(A[c], PH[c], H[c]);
            TA[c] = kept_decay(A[c] * PA[c], fminf(A[c], PA[c]));
            h[c] = p.initial && here ? p.initial[(int64_t)at.b * p.D + ch + c] : 0.f;
        }
        if (p.pairs && rows > 0) {
            const int g = at.c / p.group, j = at.c - g * p.group;
            uint64_t *mine = p.pairs + ((int64_t)at.b * p.chunks + at.c) * p.D + ch;
            if (here && j + 1 < p.group) {
#pragma unroll
                for (int c = 0; c < C; ++c) publish(mine + c, word_of(TA[c], TH[c]));
            }
            float GA[C], GH[C];
            together<C>(mine - (int64_t)j * p.D, p.D, j, here, GA, GH);
            if (g > 0 && here) {
                const uint64_t *from = p.carries + ((int64_t)at.b * ((p.chunks + p.group - 1) / p.group) + g) * p.D + ch;
#pragma unroll
                for (int c = 0; c < C; ++c) h[c] = word_H(wait_for(from + c, look(from + c)));
            }
#pragma unroll
            for (int c = 0; c < C; ++c) h[c] = fmaf(GA[c], h[c], GH[c]);
            if (here && j + 1 == p.group && at.c + 1 < p.chunks) {
                uint64_t *to = p.carries + ((int64_t)at.b * ((p.chunks + p.group - 1) / p.group) + g + 1) * p.D + ch;
#pragma unroll
                for (int c = 0; c < C; ++c) publish(to + c, word_of(1.f, fmaf(TA[c], h[c], TH[c])));
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c) enter[lane * C + c] = h[c];
        // the state behind the last row (of an empty sequence: the one given)
        if (p.final && here && (rows > 0 ? t0 + rows == len : t0 == 0)) {
#pragma unroll
            for (int c = 0; c < C; ++c) p.final[(int64_t)at.b * p.D + ch + c] = fmaf(TA[c], h[c], TH[c]);
        }
    }
    __syncthreads();
    float h[C];
#pragma unroll
    for (int c = 0; c < C; ++c) h[c] = fmaf(PA[c], enter[lane * C + c], PH[c]);
    if (p.states && here && slot * R % kChunk == 0 && slot * R < out_rows) {
#pragma unroll
        for (int c = 0; c < C; ++c) p.states[((int64_t)at.b * p.kept + (t0 + slot * R) / kChunk) * p.D + ch + c] = h[c];
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float y[C], g[C];
        if constexpr (GATE) channels(rg[i], g, T{});
        const bool inside = slot * R + i < rows;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            h[c] = fmaf(a[i][c], h[c], u[i][c]);
            y[c] = GATE ? g[c] * h[c] : h[c];
            y[c] = inside ? y[c] : 0.f;
        }
        store_channels(wy, lane_off + (slot * R + i) * sy, y, T{});
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------
template <typename T, int C, int R, int W, bool GATE> __global__ __launch_bounds__(W * 64, 4) void scan_bwd_kernel(Scan p)
{
    constexpr int ROWS = R * W, E = (int)sizeof(T);
    static_assert(ROWS == kChunk, "a chunk starts at a kept state");
    __shared__ float pairA[W][64 * C], pairH[W][64 * C], pairK[W][64 * C], enter[64 * C];
    __shared__ uint32_t ticket;
    const int lane = threadIdx.x % 64, slot = threadIdx.x / 64;
    const Place at = place_of(p, &ticket, true);
    const int ch = (at.col * 64 + lane) * C;
    const bool here = ch < p.D;
    const int64_t t0 = (int64_t)at.c * ROWS;
    int64_t len = p.lengths ? p.lengths[at.b] : p.L;
    len = len < 0 ? 0 : len > p.L ? p.L : len;
    const int rows = (int)(len - t0 < ROWS ? (len - t0 > 0 ? len - t0 : 0) : ROWS);
    const int out_rows = (int)(p.L - t0 < ROWS ? p.L - t0 : ROWS);
    const uint32_t lane_off = here ? (uint32_t)(ch * E) : WIN_OFF;

    const win_t wx = window_of<T>(p.x, at.b, t0, rows, p.D), wf = window_of<T>(p.f, at.b, t0, rows, p.D);
    const win_t wg = window_of<T>(GATE ? p.gate : p.x, at.b, t0, rows, p.D), wd = window_of<T>(p.dy, at.b, t0, rows, p.D);
    const win_t wdx = window_of<T>(p.dx, at.b, t0, out_rows, p.D), wdf = window_of<T>(p.df, at.b, t0, out_rows, p.D);
    const win_t wdg = window_of<T>(GATE ? p.dgate : p.dx, at.b, t0, out_rows, p.D);
    const uint32_t sx = (uint32_t)(p.x.time * E), sf = (uint32_t)(p.f.time * E), sg = (uint32_t)(p.gate.time * E), sd = (uint32_t)(p.dy.time * E);
    const uint32_t sdx = (uint32_t)(p.dx.time * E), sdf = (uint32_t)(p.df.time * E), sdg = (uint32_t)(p.dgate.time * E);
    uint32_t rx[R], rf[R], rd[R], rg[GATE ? R : 1];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const uint32_t row = slot * R + i;
        rf[i] = load_channels<T, C>(wf, lane_off + row * sf);
        rx[i] = load_channels<T, C>(wx, lane_off + row * sx);
        // (a row that is not in the sequence may lie inside the window where rows share their elements: a sum's gradient is one row for all)
        const bool inside = (int)row < rows;
        rd[i] = load_channels<T, C>(wd, inside ? lane_off + row * sd : WIN_OFF);
        if constexpr (GATE) rg[i] = load_channels<T, C>(wg, inside ? lane_off + row * sg : WIN_OFF);
    }
    float bias[C], h0[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        bias[c] = p.bias && here ? p.bias[ch + c] : 0.f;
        h0[c] = here ? p.states[((int64_t)at.b * p.kept + at.c) * p.D + ch + c] : 0.f;
    }

    float a[R][C], b[R][C], A[C], H[C], K[C], least[C];
    // gate dy of row i
    const auto weighted = [&](int i, float (&v)[C]) {
        channels(rd[i], v, T{});
        if constexpr (GATE) {
            float g[C];
            channels(rg[i], g, T{});
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] *= g[c];
        }
    };
#pragma unroll
    for (int c = 0; c < C; ++c) { A[c] = 1.f; H[c] = 0.f; K[c] = 0.f; least[c] = 1.f; }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float x[C], f[C];
        channels(rx[i], x, T{});
        channels(rf[i], f, T{});
        const bool inside = slot * R + i < rows;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            sigmoids<E == 4>(f[c] + bias[c], a[i][c], b[i][c]);
            a[i][c] = inside ? a[i][c] : 1.f;
            b[i][c] = inside ? b[i][c] : 0.f;
            A[c] *= a[i][c];
            H[c] = fmaf(a[i][c], H[c], b[i][c] * x[c]);
            least[c] = fminf(least[c], a[i][c]);
        }
    }
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
        float gd[C];
        weighted(i, gd);
#pragma unroll
        for (int c = 0; c < C; ++c) K[c] = a[i][c] * (gd[c] + K[c]);
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        A[c] = kept_decay(A[c], least[c]);
        pairA[slot][lane * C + c] = A[c];
        pairH[slot][lane * C + c] = H[c];
        pairK[slot][lane * C + c] = K[c];
    }
    __syncthreads();
    // the state before this slot; the pair of the slots behind it
    float h[C], PA[C], PK[C];
#pragma unroll
    for (int c = 0; c < C; ++c) { h[c] = h0[c]; PA[c] = 1.f; PK[c] = 0.f; }
    for (int s = 0; s < slot; ++s) {
#pragma unroll
        for (int c = 0; c < C; ++c) h[c] = fmaf(pairA[s][lane * C + c], h[c], pairH[s][lane * C + c]);
    }
    for (int s = W - 1; s > slot; --s) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float As = pairA[s][lane * C + c];
            PK[c] = fmaf(As, PK[c], pairK[s][lane * C + c]);
            PA[c] = kept_decay(PA[c] * As, fminf(PA[c], As));
        }
    }
    if (slot == 0) {
        float TA[C], TK[C], k[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            TK[c] = fmaf(A[c], PK[c], K[c]);
            TA[c] = kept_decay(A[c] * PA[c], fminf(A[c], PA[c]));
            k[c] = p.dfinal && here ? p.dfinal[(int64_t)at.b * p.D + ch + c] : 0.f;
        }
        if (p.pairs && rows > 0) {
            const int g = at.c / p.group, last = (int)((len - 1) / ROWS), end = g * p.group + p.group - 1;
            uint64_t *mine = p.pairs + ((int64_t)at.b * p.chunks + at.c) * p.D + ch;
            if (here && at.c > g * p.group) {
#pragma unroll
                for (int c = 0; c < C; ++c) publish(mine + c, word_of(TA[c], TK[c]));
            }
            const int behind = end < last ? end : last;
            float GA[C], GK[C];
            together<C>(mine + (int64_t)(behind - at.c) * p.D, -(int64_t)p.D, behind - at.c, here, GA, GK);
            if (end < last && here) {
                const uint64_t *from = p.carries + ((int64_t)at.b * ((p.chunks + p.group - 1) / p.group) + g) * p.D + ch;
#pragma unroll
                for (int c = 0; c < C; ++c) k[c] = word_H(wait_for(from + c, look(from + c)));
            }
#pragma unroll
            for (int c = 0; c < C; ++c) k[c] = fmaf(GA[c], k[c], GK[c]);
            if (here && at.c == g * p.group && g > 0) {
                uint64_t *to = p.carries + ((int64_t)at.b * ((p.chunks + p.group - 1) / p.group) + g - 1) * p.D + ch;
#pragma unroll
                for (int c = 0; c < C; ++c) publish(to + c, word_of(1.f, fmaf(TA[c], k[c], TK[c])));
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c) enter[lane * C + c] = k[c];
        if (p.dinitial && here && at.c == 0) {
#pragma unroll
            for (int c = 0; c < C; ++c) p.dinitial[(int64_t)at.b * p.D + ch + c] = rows > 0 ? fmaf(TA[c], k[c], TK[c]) : k[c];
        }
    }
    // dgate, and what df is times G, while the first slot waits.  (The raw rows are converted again, not kept in fp32 over the barrier.)
    float q[R][C];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        asm volatile("" : "+v"(rd[i]), "+v"(rx[i]));
        if constexpr (GATE) asm volatile("" : "+v"(rg[i]));
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float x[C], d[C], dg[C];
        channels(rx[i], x, T{});
        channels(rd[i], d, T{});
#pragma unroll
        for (int c = 0; c < C; ++c) {
            q[i][c] = (h[c] - x[c]) * (a[i][c] * b[i][c]);
            h[c] = fmaf(a[i][c], h[c], b[i][c] * x[c]);
            dg[c] = slot * R + i < rows ? d[c] * h[c] : 0.f;
        }
        if constexpr (GATE) store_channels(wdg, lane_off + (slot * R + i) * sdg, dg, T{});
    }
    __syncthreads();
    float k[C], sum[C];
#pragma unroll
    for (int c = 0; c < C; ++c) { k[c] = fmaf(PA[c], enter[lane * C + c], PK[c]); sum[c] = 0.f; }
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
        float dx[C], df[C], gd[C];
        weighted(i, gd);
        const bool inside = slot * R + i < rows;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float G = gd[c] + k[c];
            dx[c] = inside ? b[i][c] * G : 0.f;
            df[c] = inside ? q[i][c] * G : 0.f;
            sum[c] += df[c];
            k[c] = a[i][c] * G;
        }
        store_channels(wdx, lane_off + (slot * R + i) * sdx, dx, T{});
        store_channels(wdf, lane_off + (slot * R + i) * sdf, df, T{});
    }
    if (!p.partial) return;
#pragma unroll
    for (int c = 0; c < C; ++c) pairH[slot][lane * C + c] = sum[c];         // (read last before the barrier above)
    __syncthreads();
    if (slot == 0 && here) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float s = sum[c];
#pragma unroll
            for (int w = 1; w < W; ++w) s += pairH[w][lane * C + c];
            p.partial[((int64_t)at.b * p.chunks + at.c) * p.D + ch + c] = s;
        }
    }
}

// dbias of the chunks' sums, in a fixed order: 32 channels a workgroup, 32 threads a channel
__global__ __launch_bounds__(1024) void scan_bias_kernel(const float *partial, int64_t n, int D, float *dbias)
{
    __shared__ float part[32][33];
    const int lane = threadIdx.x % 32, slice = threadIdx.x / 32, c = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (c < D) {
#pragma unroll 8
        for (int64_t i = slice; i < n; i += 32) s += partial[i * D + c];
    }
    part[slice][lane] = s;
    __syncthreads();
    s = part[lane][slice];
#pragma unroll
    for (int d = 16; d > 0; d /= 2) s += __shfl_xor(s, d);
    const int out = blockIdx.x * 32 + slice;
    if (lane == 0 && out < D) dbias[out] = s;
}

__global__ __launch_bounds__(256) void scan_clear_kernel(u32x4 *p, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = u32x4{0, 0, 0, 0};
}

// ---- one token ------------------------------------------------------------------------------------------------------------------
struct ScanStep {
    const void *x, *f, *gate;
    const float *bias;
    float *state;
    void *y;
    int64_t sx, sf, sg;         // rows' strides in elements
    int32_t bs, D;
};
template <typename T, bool GATE> __global__ __launch_bounds__(256) void scan_step_kernel(ScanStep p)
{
    const int ch = blockIdx.x * 256 + threadIdx.x;
    if (ch >= p.D) return;
    for (uint32_t b = blockIdx.y; b < (uint32_t)p.bs; b += gridDim.y) {         // (a step beyond the last entry may pass 2^31)
        const int64_t i = (int64_t)b * p.D + ch;
        const float x = Elem<T>::load((const T *)p.x + b * p.sx + ch), f = Elem<T>::load((const T *)p.f + b * p.sf + ch);
        const float g = GATE ? Elem<T>::load((const T *)p.gate + b * p.sg + ch) : 1.f, before = p.state[i];
        float a, u;
        sigmoids<sizeof(T) == 4>(f + (p.bias ? p.bias[ch] : 0.f), a, u);
        const float h = fmaf(a, before, u * x);
        p.state[i] = h;
        Elem<T>::store((T *)p.y + i, GATE ? g * h : h);
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------
// Rows of a chunk of the forward: 128, two workgroups a CU, which overlap one's loads with the other's sums.  256, one workgroup a CU, where the card
// holds all of those at once and they are whole sequences, or those of 128 more than a CU's one or very many: what counts then is the chain of waits.
// In chunks of 128 and 256, launches after each other: 4 x 701 x 2560 f16 17.8 and 15.9 us, 1 x 8192 x 1024 bf16 28.6 and 23.4, 16 x 256 x 1024 fp32 22.7 and 11.9; but
// 1 x 512 x 4096 14.1 and 16.1, 64 x 256 x 4096 112 and 122, 2 x 8192 x 4096 118 and 131.  So also with many chunks after each other: 32768 x 128 fp32 36
// and 25, 16384 x 256 bf16 26 and 23, 8192 x 512 20 and 21.
int fwd_rows(int64_t bs, int64_t L, int64_t D)
{
    const int64_t cols = (D + 127) / 128, high = bs * ((L + 255) / 256) * cols, low = bs * ((L + 127) / 128) * cols;
    return L > 128 && high <= 256 && (L <= 256 || low > 256 || L > 12288) ? 256 : 128;
}
// Chunks of a group: 8 where there is enough to do beside the words' way (131072 x 512 fp32 193 us with 8, 196 with 16, 223 with 32; 2 x 8192 x 4096 bf16 113,
// 118 and 131; the backward of 27733 x 984 bf16 130 with 8, 148 with 32).  Where two workgroups (fp32: four) at most have the same time, a
// group's step is most of it: 65536 x 64 bf16 39 us with 8, 30 with 32, backward 113 and 57; 24531 x 109 fp32, backward, 57 and 39.
int group_of(int64_t bs, int64_t chunks, int64_t D)
{
    if (chunks <= 64 || bs * ((D + 127) / 128) > 2) return 8;
    return chunks <= 256 ? 16 : 32;
}

struct Layout { int64_t chunks, group, groups, pairs, carries, total; };
Layout layout_of(int64_t bs, int64_t L, int64_t D, bool backward)
{
    Layout l;
    const int rows = backward ? kChunk : fwd_rows(bs, L, D);
    l.chunks = (L + rows - 1) / rows;
    l.group = group_of(bs, l.chunks, D);
    l.groups = (l.chunks + l.group - 1) / l.group;
    l.pairs = 256;
    l.carries = l.pairs + bs * l.chunks * D * 8;
    l.total = l.chunks > 1 ? (l.carries + bs * l.groups * D * 8 + 255) / 256 * 256 : 0;
    return l;
}

// The words' part of the workspace, cleared; what follows it is the bias's partial sums.
int set_up(Scan &p, const Layout &l, void *ws, hipStream_t st)
{
    p.chunks = (int32_t)l.chunks;
    p.group = (int32_t)l.group;
    p.pairs = p.carries = nullptr;
    p.ticket = nullptr;
    if (l.chunks == 1) return 0;
    p.ticket = (uint32_t *)ws;
    p.pairs = (uint64_t *)((char *)ws + l.pairs);
    p.carries = (uint64_t *)((char *)ws + l.carries);
    const int64_t n = l.total / 16, blocks = (n + 1023) / 1024;
    return launch_plain(scan_clear_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), st, (u32x4 *)ws, n);
}

bool even(const ScanTensor &t, bool given) { return !given || (((uintptr_t)t.p & 3) == 0 && t.batch % 2 == 0 && t.time % 2 == 0); }

template <typename T, int C, int W> int fwd_w(const Scan &p, int64_t n, hipStream_t st)
{
    if (!launch_holds(n, W * 64)) return (int)hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)n), block(W * 64);
    return p.gate.p ? launch_main(scan_fwd_kernel<T, C, 16, W, true>, grid, block, st, p) : launch_main(scan_fwd_kernel<T, C, 16, W, false>, grid, block, st, p);
}
template <typename T, int C> int fwd_c(Scan &p, hipStream_t st)
{
    p.cols = (p.D + 64 * C - 1) / (64 * C);
    const int64_t n = (int64_t)p.chunks * p.bs * p.cols;
    return fwd_rows(p.bs, p.L, p.D) == 256 ? fwd_w<T, C, 16>(p, n, st) : fwd_w<T, C, 8>(p, n, st);
}
template <typename T, int C> int bwd_c(Scan &p, hipStream_t st)
{
    p.cols = (p.D + 64 * C - 1) / (64 * C);
    const int64_t n = (int64_t)p.chunks * p.bs * p.cols;
    if (!launch_holds(n, 512)) return (int)hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)n), block(512);
    return p.gate.p ? launch_main(scan_bwd_kernel<T, C, 8, 8, true>, grid, block, st, p) : launch_main(scan_bwd_kernel<T, C, 8, 8, false>, grid, block, st, p);
}
ScanTensor tensor(const void *p, const int64_t *s, int i) { return {p, s[2 * i], s[2 * i + 1]}; }

} // namespace

size_t scan_workspace(int64_t bs, int64_t L, int D, bool backward)
{
    const Layout l = layout_of(bs, L, D, backward);
    return (size_t)(l.total + (backward ? bs * l.chunks * D * 4 : 0));
}
int64_t scan_states(int64_t L) { return (L + kChunk - 1) / kChunk; }

int scan_fwd_launch(int dtype, const void *x, const void *f, const void *gate, const int64_t *strides, const float *bias, const float *initial,
                    const int32_t *lengths, void *y, float *final, float *states, void *ws, int64_t bs, int64_t L, int D, hipStream_t st)
{
    Scan p = {};
    p.x = tensor(x, strides, 0);
    p.f = tensor(f, strides, 1);
    p.gate = tensor(gate, strides, 2);
    p.y = tensor(y, strides, 3);
    p.bias = bias; p.initial = initial; p.lengths = lengths; p.final = final; p.states = states;
    p.L = L; p.D = D; p.bs = (int32_t)bs; p.kept = (int32_t)scan_states(L);
    const int rc = set_up(p, layout_of(bs, L, D, false), ws, st);
    if (rc) return rc;
    const bool two = D % 2 == 0 && even(p.x, true) && even(p.f, true) && even(p.gate, gate != nullptr) && even(p.y, true);
    switch (dtype) {
    case GCG_F32: return fwd_c<float, 1>(p, st);
    case GCG_BF16: return two ? fwd_c<bf16_t, 2>(p, st) : fwd_c<bf16_t, 1>(p, st);
    default: return two ? fwd_c<f16_t, 2>(p, st) : fwd_c<f16_t, 1>(p, st);
    }
}

int scan_bwd_launch(int dtype, const void *dy, const void *x, const void *f, const void *gate, const int64_t *strides, const float *bias,
                    const float *states, const int32_t *lengths, const float *dfinal, void *dx, void *df, void *dgate, float *dbias,
                    float *dinitial, void *ws, int64_t bs, int64_t L, int D, hipStream_t st)
{
    Scan p = {};
    p.dy = tensor(dy, strides, 0);
    p.x = tensor(x, strides, 1);
    p.f = tensor(f, strides, 2);
    p.gate = tensor(gate, strides, 3);
    p.dx = tensor(dx, strides, 4);
    p.df = tensor(df, strides, 5);
    p.dgate = tensor(dgate, strides, 6);
    p.bias = bias; p.states = const_cast<float *>(states); p.lengths = lengths; p.dfinal = dfinal; p.dinitial = dinitial;
    p.L = L; p.D = D; p.bs = (int32_t)bs; p.kept = (int32_t)scan_states(L);
    const Layout l = layout_of(bs, L, D, true);
    int rc = set_up(p, l, ws, st);
    if (rc) return rc;
    p.partial = dbias ? (float *)((char *)ws + l.total) : nullptr;
    const bool g = gate != nullptr;
    const bool two = D % 2 == 0 && even(p.dy, true) && even(p.x, true) && even(p.f, true) && even(p.gate, g) && even(p.dx, true) &&
                     even(p.df, true) && even(p.dgate, g);
    switch (dtype) {
    case GCG_F32: rc = bwd_c<float, 1>(p, st); break;
    case GCG_BF16: rc = two ? bwd_c<bf16_t, 2>(p, st) : bwd_c<bf16_t, 1>(p, st); break;
    default: rc = two ? bwd_c<f16_t, 2>(p, st) : bwd_c<f16_t, 1>(p, st); break;
    }
    if (rc || !dbias) return rc;
    return launch_plain(scan_bias_kernel, dim3((unsigned)((D + 31) / 32)), dim3(1024), st, (const float *)p.partial, bs * l.chunks, D, dbias);
}

int scan_step_launch(int dtype, const void *x, const void *f, const void *gate, const int64_t *strides, const float *bias, float *state, void *y,
                     int64_t bs, int D, hipStream_t st)
{
    const ScanStep p = {x, f, gate, bias, state, y, strides[0], strides[1], strides[2], (int32_t)bs, D};
    // (as many entries beside each other as a launch's 2^32 threads hold)
    const int64_t across = (D + 255) / 256, most = ((1ll << 24) - 1) / across, deep = most < 65535 ? most : 65535;
    const dim3 grid((unsigned)across, (unsigned)(bs < deep ? bs : deep)), block(256);
    switch (dtype) {
    case GCG_F32: return gate ? launch_main(scan_step_kernel<float, true>, grid, block, st, p) : launch_main(scan_step_kernel<float, false>, grid, block, st, p);
    case GCG_BF16: return gate ? launch_main(scan_step_kernel<bf16_t, true>, grid, block, st, p) : launch_main(scan_step_kernel<bf16_t, false>, grid, block, st, p);
    default: return gate ? launch_main(scan_step_kernel<f16_t, true>, grid, block, st, p) : launch_main(scan_step_kernel<f16_t, false>, grid, block, st, p);
    }
}

} // namespace gcg
