// Products of tensors in 8-bit floating point with a scale for each block of 128 (format: gcg_float8.h):
//
//   y[m, n] = sum over blocks k of 2^(sa[m, k] + sb[n, k] - 254) * sum over the block of a[m, i] b[n, i]
//
// The matrix instruction takes 16 rows of each operand and a whole block, 128 elements, and applies the two rows' scale bytes by itself, so
// the inner loop holds no vector arithmetic but a shift of the scales' words.  Which element of the block a lane's bytes are does not
// matter as long as both operands agree, so a lane takes two 16-byte pieces of its row, 64 bytes apart.  Accumulators are fp32.  (Inside an
// instruction groups of eight products are aligned to their largest and cut at 2^-14.6 of it, as measured; results
// are given in 16 bits, whose rounding is larger.)
#include "gcg_float8.h"

namespace gcg {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_t;

// 16 bytes a lane from the window at off + at straight into shared memory, lane after lane from `to` on (the host pass, which knows neither
// the target nor the width, is not to see it)
__device__ __forceinline__ void load_to_lds(win_t w, uint8_t *to, uint32_t off, int at)
{
#ifdef __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_raw_ptr_buffer_load_lds(w, (lds_t)to, 16, (int)off, at, 0, 0);
#endif
}

struct Product8 {
    const uint8_t *a, *a_scales, *b, *b_scales;
    void *y;
    float *partial;             // (splits, M, N), or null
    int64_t M, N;
    int64_t Kp;                 // bytes of a row
    int32_t S;                  // scales of a row
    int32_t steps;              // blocks of a row
    int32_t split_steps;        // blocks of a part, a multiple of four
    uint32_t tiles_m, tiles_n;
};

template <bool A5, bool B5> __device__ __forceinline__ f32x4 mfma8(const i32x8 &a, const i32x8 &b, const f32x4 &c, uint32_t sa, uint32_t sb)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, A5 ? 1 : 0, B5 ? 1 : 0, 0, (int)sa, 0, (int)sb);
}

template <typename T> __device__ __forceinline__ void store4(T *p, const f32x4 &v, int64_t left, bool vec)
{
    if (left >= 4 && vec) {
        if constexpr (sizeof(T) == 4) *(f32x4 *)p = v;
        else if constexpr (std::is_same_v<T, bf16_t>) *(u32x2 *)p = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        else *(u32x2 *)p = u32x2{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) Elem<T>::store(p + i, v[i]);
    }
}

// A workgroup of WM x WN waves makes a tile of BM x BN.  Both operands' rows of a block go straight into shared memory, 16 bytes a lane;
// a row's eight pieces lie at exchanged places (by row / 2), so that 16 rows' pieces are in different banks.  Two such stages: the next
// one is requested when a stage's fragments have been read, and has all of the products' time to arrive.
template <int BM, int BN, int WM, int WN, typename T, bool A5, bool B5>
__global__ __launch_bounds__(WM * WN * 64) void product8_kernel(Product8 p)
{
    constexpr int THREADS = WM * WN * 64, MT = BM / WM / 16, NT = BN / WN / 16;
    constexpr int LA = BM * 8 / THREADS, LB = BN * 8 / THREADS;        // 16-byte loads of a thread
    __shared__ __attribute__((aligned(1024))) uint8_t stage[2][(BM + BN) * 128];
    const int t = threadIdx.x, wave = t / 64, lane = t % 64;
    const uint32_t tile = xcd_contiguous_u32(blockIdx.x, p.tiles_m * p.tiles_n);
    // tiles in groups of eight rows of tiles, so that those at work at once share their operands' rows
    const uint32_t group = tile / (8 * p.tiles_n), first = group * 8, high = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
    const uint32_t in = tile - group * 8 * p.tiles_n;
    const int64_t m0 = (int64_t)(first + in % high) * BM, n0 = (int64_t)(in / high) * BN;
    const int k0 = blockIdx.y * p.split_steps, k1 = p.steps - k0 < p.split_steps ? p.steps : k0 + p.split_steps;

    // a thread's pieces: row t / 8 + i * THREADS / 8 of the tile (rows beyond the tensor: its last), the piece that belongs to place t % 8
    const win_t wa = make_window(p.a + m0 * p.Kp, 0x7fffffff), wb = make_window(p.b + n0 * p.Kp, 0x7fffffff);
    uint32_t oa[LA], ob[LB];
#pragma unroll
    for (int i = 0; i < LA; ++i) {
        const int r = t / 8 + i * (THREADS / 8);
        const int64_t last = p.M - 1 - m0;
        oa[i] = (uint32_t)((r < last ? r : last) * p.Kp) + ((t % 8) ^ ((r >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
        const int r = t / 8 + i * (THREADS / 8);
        const int64_t last = p.N - 1 - n0;
        ob[i] = (uint32_t)((r < last ? r : last) * p.Kp) + ((t % 8) ^ ((r >> 1) & 7)) * 16;
    }
    const auto request = [&](int k, int s) {
#pragma unroll
        for (int i = 0; i < LA; ++i)
            load_to_lds(wa, stage[s] + (i * THREADS + wave * 64) * 16, oa[i], k * 128);
#pragma unroll
        for (int i = 0; i < LB; ++i)
            load_to_lds(wb, stage[s] + BM * 128 + (i * THREADS + wave * 64) * 16, ob[i], k * 128);
    };
    const int wm = wave % WM, wn = wave / WM, r16 = lane % 16, quarter = lane / 16;
    // where a lane's two pieces of fragment 0 lie; a fragment's 16 rows leave (row / 2) % 8 as it is
    const int swap = (r16 >> 1) & 7;
    const int fa = (wm * MT * 16 + r16) * 128, fb = BM * 128 + (wn * NT * 16 + r16) * 128;
    const int p0 = (quarter ^ swap) * 16, p1 = ((quarter + 4) ^ swap) * 16;
    const auto fragment = [&](int s, int at) {
        const u32x4 lo = *(const u32x4 *)(stage[s] + at + p0), hi = *(const u32x4 *)(stage[s] + at + p1);
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
    // the scales of the fragments' rows, four blocks in a word
    const uint32_t *sa[MT], *sb[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t r = m0 + (wm * MT + i) * 16 + r16;
        sa[i] = (const uint32_t *)(p.a_scales + (r < p.M ? r : p.M - 1) * p.S);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t r = n0 + (wn * NT + j) * 16 + r16;
        sb[j] = (const uint32_t *)(p.b_scales + (r < p.N ? r : p.N - 1) * p.S);
    }
    uint32_t ca[MT], cb[NT], na[MT], nb[NT];
    const auto scales = [&](int word) {
#pragma unroll
        for (int i = 0; i < MT; ++i) na[i] = sa[i][word];
#pragma unroll
        for (int j = 0; j < NT; ++j) nb[j] = sb[j][word];
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    scales(k0 / 4);
    request(k0, 0);
    for (int k = k0; k < k1; ++k) {
        const int s = (k - k0) & 1;
        // the stage is there (a barrier alone does not wait for loads into shared memory), and nobody reads the other one any more
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (((k - k0) & 3) == 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i) ca[i] = na[i];
#pragma unroll
            for (int j = 0; j < NT; ++j) cb[j] = nb[j];
        }
        i32x8 fragA[MT], fragB[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) fragB[j] = fragment(s, fb + j * 16 * 128);
#pragma unroll
        for (int i = 0; i < MT; ++i) fragA[i] = fragment(s, fa + i * 16 * 128);
        __builtin_amdgcn_sched_barrier(0);
        if (k + 1 < k1) {
            request(k + 1, s ^ 1);
            if (((k - k0) & 3) == 0 && k + 4 < k1) scales(k / 4 + 1);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mfma8<B5, A5>(fragB[j], fragA[i], acc[i][j], cb[j], ca[i]);
#pragma unroll
        for (int i = 0; i < MT; ++i) ca[i] >>= 8;
#pragma unroll
        for (int j = 0; j < NT; ++j) cb[j] >>= 8;
    }
    // a lane has row m = lane % 16 and four columns n of every 16 x 16
    T *y = p.partial ? (T *)(p.partial + (int64_t)blockIdx.y * p.M * p.N) : (T *)p.y;
    const bool vec = p.N % 4 == 0 && (((uintptr_t)y) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + (wm * MT + i) * 16 + r16;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int64_t n = n0 + (wn * NT + j) * 16 + quarter * 4;
            store4(y + m * p.N + n, acc[i][j], p.N - n, vec);
        }
    }
}

// the parts of a product that was split over its blocks, added in their order
template <typename T> __global__ __launch_bounds__(256) void product8_join_kernel(const float *partial, T *y, int64_t n, int splits)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = partial[i];
        for (int k = 1; k < splits; ++k) s += partial[k * n + i];
        Elem<T>::store(y + i, s);
    }
}

struct Plan8 { int tile; int splits; int split_steps; };
Plan8 plan_of(int64_t M, int64_t N, int64_t K)
{
    const int steps = (int)(f8_cols(K) / 128);
    const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128);
    Plan8 p = {128, 1, (steps + 3) / 4 * 4};
    while (tiles * p.splits < 256 && p.split_steps >= 8) {
        p.splits *= 2;
        p.split_steps = ((steps + p.splits - 1) / p.splits + 3) / 4 * 4;
    }
    p.splits = (steps + p.split_steps - 1) / p.split_steps;
    return p;
}

template <int BM, int BN, int WM, int WN, typename T, bool A5, bool B5> int tile_launch(Product8 &p, const Plan8 &plan, hipStream_t st)
{
    p.tiles_m = (uint32_t)((p.M + BM - 1) / BM);
    p.tiles_n = (uint32_t)((p.N + BN - 1) / BN);
    return launch_main(product8_kernel<BM, BN, WM, WN, T, A5, B5>, dim3(p.tiles_m * p.tiles_n, (unsigned)plan.splits), dim3(WM * WN * 64), st, p);
}
template <typename T, bool A5, bool B5> int product_launch(Product8 &p, const Plan8 &plan, hipStream_t st)
{
#ifdef GCG_TUNING
    if constexpr (!A5 && !B5) {
    const char *e = tuning_env("GCG_P8");
    switch (e ? atoi(e) : 0) {
    case 1: return tile_launch<256, 256, 2, 2, T, A5, B5>(p, plan, st);
    case 2: return tile_launch<256, 256, 2, 4, T, A5, B5>(p, plan, st);
    case 3: return tile_launch<256, 128, 2, 2, T, A5, B5>(p, plan, st);
    case 4: return tile_launch<128, 256, 2, 2, T, A5, B5>(p, plan, st);
    case 5: return tile_launch<256, 256, 4, 2, T, A5, B5>(p, plan, st);
    case 6: return tile_launch<256, 128, 4, 2, T, A5, B5>(p, plan, st);
    }
    }
#endif
    p.tiles_m = (uint32_t)((p.M + 127) / 128);
    p.tiles_n = (uint32_t)((p.N + 127) / 128);
    return launch_main(product8_kernel<128, 128, 2, 2, T, A5, B5>, dim3(p.tiles_m * p.tiles_n, (unsigned)plan.splits), dim3(256), st, p);
}
template <typename T> int product_format(Product8 &p, int a5, int b5, const Plan8 &plan, hipStream_t st)
{
    if (a5) return b5 ? product_launch<T, true, true>(p, plan, st) : product_launch<T, true, false>(p, plan, st);
    return b5 ? product_launch<T, false, true>(p, plan, st) : product_launch<T, false, false>(p, plan, st);
}
template <typename T> int product_type(Product8 &p, int a5, int b5, const Plan8 &plan, hipStream_t st)
{
    if (plan.splits == 1) return product_format<T>(p, a5, b5, plan, st);
    const int rc = product_format<float>(p, a5, b5, plan, st);
    if (rc) return rc;
    const int64_t n = p.M * p.N, blocks = (n + 255) / 256;
    return launch_plain(product8_join_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), st, (const float *)p.partial,
                        (T *)p.y, n, plan.splits);
}

} // namespace

size_t product8_workspace(int64_t M, int64_t N, int64_t K)
{
    const Plan8 plan = plan_of(M, N, K);
    return plan.splits > 1 ? (size_t)plan.splits * M * N * sizeof(float) : 0;
}

int product8_launch(int dtype, int a5, int b5, const uint8_t *a, const uint8_t *a_scales, const uint8_t *b, const uint8_t *b_scales, void *y,
                    void *ws, int64_t M, int64_t N, int64_t K, hipStream_t st)
{
    const Plan8 plan = plan_of(M, N, K);
    Product8 p = {a, a_scales, b, b_scales, y, plan.splits > 1 ? (float *)ws : nullptr, M, N, f8_cols(K), (int32_t)f8_scales(K),
                  (int32_t)(f8_cols(K) / 128), plan.split_steps, 0, 0};
    return dtype == GCG_BF16 ? product_type<bf16_t>(p, a5, b5, plan, st) : product_type<f16_t>(p, a5, b5, plan, st);
}

} // namespace gcg
