// Products of tensors in 8-bit floating point with a scale for each block of 128 (format: gcg_float8.h):
//
//   y[m, n] = sum over blocks k of 2^(sa[m, k] + sb[n, k] - 254) * sum over the block of a[m, i] b[n, i]
//
// The matrix instruction takes 16 rows of each operand and a whole block, 128 elements, and applies the two rows' scale bytes by itself, so
// the inner loop holds no vector arithmetic but a shift of the scales' words.  Which element of the block a lane's bytes are does not
// matter as long as both operands agree, so a lane takes two 16-byte pieces of its row, 64 bytes apart.  Accumulators are fp32.  (Inside an
// instruction groups of eight products are aligned to their largest and cut at 2^-14.6 of it, as measured; results
// are given in 16 bits, whose rounding is larger, but where a sum cancels: it keeps an error relative to the largest products in it.)
//
// Large products go by product8_wide_kernel and are bound by the matrix units at the clock that the power leaves them: 16384 x 12288 x 4096 takes
// 510 us on zeros, 680 on normal numbers (2.4 PFLOP/s) and 640 to 740 on a residual stream's, as the clock goes; 8192 x 8192 x 8192 387 (2.8).  Few rows go by
// product8_tokens_kernel and are bound by b's bytes: 12288 x 4096 with one row 10.4 us (4.8 TB/s), 24576 x 8192 with eight 37 (5.4).
// What lies between goes by whichever of these or product8_kernel takes least time (gcg_product8_plan.h).
#include "gcg_float8.h"
#include "gcg_product8_plan.h"

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
    int32_t splits;
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

// The same by four waves, one a SIMD, of 128 x 128 (BN = 256) or 128 x 64 (BN = 128) each.  A fragment is then read from shared memory for eight
// products, twice as many as in the other kernel (four and eight), and a block takes as long as 64 (32) products; to keep those fed without a second
// wave, a block goes in four phases, each of one half of the wave's rows and one half of its columns, and each reads the half that is needed next
// where the one that is no longer needed was:
//
//   (A0 B0) reads B1,  (A0 B1) reads A1,  barrier,  (A1 B1) reads the next block's A0,  (A1 B0) reads its B1;  the next block starts with (A0 B1)
//
// At the barrier a stage has been read and the next one has arrived; the one after the last that is under way is requested into it: with tiles of 256 x
// 256 the shared memory holds two stages, with 256 x 128 three, so that operands have two blocks' time to arrive (512 x 12288 x 4096 from HBM 46 us with
// two, 36 with three, 4096 x 512 x 8192 85 and 65; operands from the cache 5 to 8 % less).  Four blocks, whose scales are a word
// of each row, are one turn of the loop, without a branch in it: past the end the last block is requested again, and not used.  One to
// three blocks that are left go one after the other.
//
// The requests are written out because the compiler makes every read of shared memory wait for all requests under way, whichever stage they go to.
// They have no register to write, and the wait for them stands before the barrier.
//
// The kernel stays on its CU and goes from tile to tile: the next one's first block is requested before the last one's results leave, which go through
// shared memory, so that whole lines are written.  16384 x 12288 x 4096: 1065 us by product8_kernel's two waves a SIMD of 64 x 64, 734 by this
// one, 677 with the tiles after each other.  Eight waves, or phases that the compiler orders, spill (69 registers, 300 and more); tiles in groups
// of 4, 6, 16 rows take 713, 699, 757.
template <int BYTES> __device__ __forceinline__ void request_to_lds(win_t w, uint32_t to, uint32_t off, int at)
{
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (BYTES == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(off), "s"(w), "s"(at) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(to), "v"(off), "s"(w), "s"(at) : "memory", "m0");
#endif
}
// The instruction with its accumulator where the compiler would not leave it by itself, in the 256 registers that only matrix instructions use.
// An operand that a vector instruction has just written has to be two wait states old.
template <bool A5, bool B5, int BYTE> __device__ __forceinline__ void mfma8_acc(const i32x8 &a, const i32x8 &b, f32x4 &c, uint32_t sa, uint32_t sb)
{
#ifdef __HIP_DEVICE_COMPILE__
#define GCG_MFMA8(SEL) \
    asm volatile("s_nop 1\n\tv_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SEL " cbsz:%5 blgp:%6" \
                 : "+a"(c) : "v"(a), "v"(b), "v"(sa), "v"(sb), "n"(A5 ? 1 : 0), "n"(B5 ? 1 : 0))
    if constexpr (BYTE == 0) GCG_MFMA8("op_sel_hi:[0,0,0]");
    else if constexpr (BYTE == 1) GCG_MFMA8("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
    else if constexpr (BYTE == 2) GCG_MFMA8("op_sel_hi:[1,1,0]");
    else GCG_MFMA8("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef GCG_MFMA8
#endif
}

template <int BN, typename T, bool A5, bool B5, bool STREAM> __global__ __launch_bounds__(256, 1) void product8_wide_kernel(Product8 p)
{
    constexpr int BM = 256, LA = 8, LB = BN / 32, STAGE = (BM + BN) * 128, STAGES = BN == 128 ? 3 : 2;
    constexpr int COLS = BN / 2, HALF = COLS / 32;              // a wave's columns, and fragments of half of them
    __shared__ __attribute__((aligned(1024))) uint8_t stage[STAGES][STAGE];
    __shared__ uint32_t words[2][BM + BN];
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t / 64), lane = t % 64;
    const uint32_t tiles = p.tiles_m * p.tiles_n, items = tiles * p.splits;
    int64_t m0, n0;
    int k0, k1, split;
    win_t wa, wb, wsa, wsb;
    const auto take = [&](uint32_t item) {
        split = (int)(item / tiles);
        const uint32_t tile = xcd_contiguous_u32(item - split * tiles, tiles);
        const uint32_t group = tile / (8 * p.tiles_n), first = group * 8, high = p.tiles_m - first < 8 ? p.tiles_m - first : 8;
        const uint32_t in = tile - group * 8 * p.tiles_n;
        // tiles that would reach beyond the tensor start earlier and make some of their neighbours' results again, the same bits (M >= 256, N >= BN)
        m0 = (int64_t)(first + in % high) * BM;
        n0 = (int64_t)(in / high) * BN;
        m0 = m0 < p.M - BM ? m0 : p.M - BM;
        n0 = n0 < p.N - BN ? n0 : p.N - BN;
        k0 = split * p.split_steps;
        k1 = p.steps - k0 < p.split_steps ? p.steps : k0 + p.split_steps;
        wa = make_window(p.a + m0 * p.Kp, 0x7fffffff);
        wb = make_window(p.b + n0 * p.Kp, 0x7fffffff);
        wsa = make_window(p.a_scales + m0 * p.S, 0x7fffffff);
        wsb = make_window(p.b_scales + n0 * p.S, 0x7fffffff);
    };

    // a thread's pieces: row t / 8 + 32 i of the tile, the piece that belongs to place t % 8
    const uint32_t piece = (uint32_t)(t / 8 * p.Kp) + ((t % 8) ^ ((t >> 4) & 7)) * 16;
    const int rows32 = __builtin_amdgcn_readfirstlane((int)(32 * p.Kp));
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_t)stage[0] + wave * 1024, lds_words = (uint32_t)(uintptr_t)(lds_t)words[0] + wave * 256;
    const auto request_a = [&](int at, int s, int i) { request_to_lds<16>(wa, lds + s * STAGE + i * 4096, piece, at + i * rows32); };
    const auto request_b = [&](int at, int s, int i) { request_to_lds<16>(wb, lds + s * STAGE + BM * 128 + i * 4096, piece, at + i * rows32); };
    const auto place_of = [&](int k) { return __builtin_amdgcn_readfirstlane((k < k1 ? k : k1 - 1) * 128); };
    const auto request = [&](int k, int s) {
        const int at = place_of(k);
#pragma unroll
        for (int i = 0; i < LA; ++i) request_a(at, s, i);
#pragma unroll
        for (int i = 0; i < LB; ++i) request_b(at, s, i);
    };
    // the scales of the tile's rows for four blocks from k on, a word a row
    const uint32_t row_scales = (uint32_t)(t * p.S);
    const auto request_words = [&](int k, int s) {
        const int at = __builtin_amdgcn_readfirstlane((k < k1 ? k : k1 - 1) / 4 * 4);
        request_to_lds<4>(wsa, lds_words + s * ((BM + BN) * 4), row_scales, at);
        if (BN == 256 || wave < BN / 64) request_to_lds<4>(wsb, lds_words + s * ((BM + BN) * 4) + BM * 4, row_scales, at);
    };

    const int wm = wave & 1, wn = wave >> 1, r16 = lane % 16, quarter = lane / 16, swap = (r16 >> 1) & 7;
    const int fa = (wm * 128 + r16) * 128, fb = BM * 128 + (wn * COLS + r16) * 128;
    const int p0 = (quarter ^ swap) * 16, p1 = ((quarter + 4) ^ swap) * 16;
    const auto fragment = [&](int s, int at) {
        const u32x4 lo = *(const u32x4 *)(stage[s] + at + p0), hi = *(const u32x4 *)(stage[s] + at + p1);
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
    uint32_t ca[8], cb[2 * HALF];
    const auto take_words = [&](int s) {
#pragma unroll
        for (int i = 0; i < 8; ++i) ca[i] = words[s][wm * 128 + i * 16 + r16];
#pragma unroll
        for (int j = 0; j < 2 * HALF; ++j) cb[j] = words[s][BM + wn * COLS + j * 16 + r16];
    };
    f32x4 acc[8][2 * HALF];
    i32x8 A[2][4], B[2][HALF];
    // The products of half I of the rows and half J of the columns, and between them the FRAGMENTS fragments at `from` of stage s into `to`, and with
    // `more` the requests for the block at `at` into stage r.  (These statements stay in the order they are written in.)
    const auto phase = [&](auto i_, auto j_, auto byte_, auto &to, int s, int from, auto more_, int at, int r) {
        constexpr int i = decltype(i_)::value, j = decltype(j_)::value, byte = decltype(byte_)::value;
        constexpr bool more = decltype(more_)::value;
        constexpr int FRAGMENTS = (int)(sizeof(to) / sizeof(i32x8)), TURNS = 2 * HALF, READS = 2 * FRAGMENTS;
#pragma unroll
        for (int q = 0; q < TURNS; ++q) {
#pragma unroll
            for (int f = q * READS / TURNS; f < (q + 1) * READS / TURNS; ++f) {
                const u32x4 part = *(const u32x4 *)(stage[s] + from + f / 2 * 16 * 128 + (f % 2 ? p1 : p0));
#pragma unroll
                for (int e = 0; e < 4; ++e) to[f / 2][f % 2 * 4 + e] = (int)part[e];
            }
            if constexpr (more) {
#pragma unroll
                for (int f = q * LA / TURNS; f < (q + 1) * LA / TURNS; ++f) request_a(at, r, f);
#pragma unroll
                for (int f = q * LB / TURNS; f < (q + 1) * LB / TURNS; ++f) request_b(at, r, f);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int x = (q * 2 + h) / HALF, y = (q * 2 + h) % HALF;
                mfma8_acc<B5, A5, byte>(B[j][y], A[i][x], acc[i * 4 + x][j * HALF + y], cb[j * HALF + y], ca[i * 4 + x]);
            }
        }
    };
    constexpr std::integral_constant<int, 0> zero;
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    constexpr std::integral_constant<int, 3> three;
    constexpr std::true_type yes;
    constexpr std::false_type no;
    const auto hand_over = [&](auto under_way) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(decltype(under_way)::value) : "memory");
        __syncthreads();
    };
    constexpr std::integral_constant<int, (STAGES - 2) * (LA + LB)> later;          // the requests behind the next block's
    // one block, in stage s, whose first half of columns is J (whose fragments, and those of A's first half, are there)
    const auto block = [&](int k, auto j_, auto byte_, int s) {
        constexpr int J = decltype(j_)::value, notJ = 1 - J;
        constexpr std::integral_constant<int, J> j;
        constexpr std::integral_constant<int, notJ> not_j;
        const int next = s + 1 < STAGES ? s + 1 : 0;
        phase(zero, j, byte_, B[notJ], s, fb + notJ * HALF * 16 * 128, no, 0, 0);
        phase(zero, not_j, byte_, A[1], s, fa + 64 * 128, no, 0, 0);
        hand_over(later);
        phase(one, not_j, byte_, A[0], next, fa, yes, place_of(k + STAGES), s);
        phase(one, j, byte_, B[notJ], next, fb + notJ * HALF * 16 * 128, no, 0, 0);
        return next;
    };

    take(blockIdx.x);
    request_words(k0, 0);
#pragma unroll
    for (int s = 0; s < STAGES; ++s) request(k0 + s, s);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 1) * (LA + LB)) : "memory");     // the scales and the first block
    for (uint32_t item = blockIdx.x;;) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 2 * HALF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q) A[0][q] = fragment(0, fa + q * 16 * 128);
#pragma unroll
    for (int q = 0; q < HALF; ++q) B[0][q] = fragment(0, fb + q * 16 * 128);
    int k = k0, w = 0, s = 0;
    for (; k + 4 <= k1; k += 4, w ^= 1) {
        take_words(w);
        request_words(k + 4, w ^ 1);
        s = block(k, zero, zero, STAGES == 2 ? 0 : s);
        s = block(k + 1, one, one, STAGES == 2 ? 1 : s);
        s = block(k + 2, zero, two, STAGES == 2 ? 0 : s);
        s = block(k + 3, one, three, STAGES == 2 ? 1 : s);
    }
    if (k < k1) take_words(w);
    for (; k < k1; ++k) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int q = 0; q < 4; ++q) A[h][q] = fragment(s, fa + (h * 4 + q) * 16 * 128);
#pragma unroll
            for (int q = 0; q < HALF; ++q) B[h][q] = fragment(s, fb + (h * HALF + q) * 16 * 128);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 2 * HALF; ++j) mfma8_acc<B5, A5, 0>(B[j / HALF][j % HALF], A[i / 4][i % 4], acc[i][j], cb[j], ca[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) ca[i] >>= 8;
#pragma unroll
        for (int j = 0; j < 2 * HALF; ++j) cb[j] >>= 8;
        hand_over(later);
        request(k + STAGES, s);
        s = s + 1 < STAGES ? s + 1 : 0;
    }
    // A wave's results leave in whole rows of its columns, which lie together in shared memory first: a pass of 64 rows (fp32: 32) in its quarter of
    // the last stage, the 16-byte pieces of a row at exchanged places.  The next tile's first blocks are on their way to the others by then.
    constexpr int ROWS = 128 / (int)sizeof(T), PIECES = COLS * (int)sizeof(T) / 16;
    static_assert(4 * ROWS * PIECES * 16 <= STAGE, "in the last stage");
    const auto exchanged = [](int piece, int row) { return piece ^ (PIECES >= 16 ? row & 15 : (row >> 1) & 7); };
    uint8_t *y = (uint8_t *)((p.partial ? (T *)(p.partial + (int64_t)split * p.M * p.N) : (T *)p.y) + (m0 + wm * 128) * p.N + n0 + wn * COLS);
    hand_over(zero);                                                            // nobody reads a stage any more, and nothing arrives
    item += gridDim.x;
    const bool more = item < items;
    if (more) {
        take(item);
        request_words(k0, 0);
#pragma unroll
        for (int i = 0; i + 1 < STAGES; ++i) request(k0 + i, i);
    }
    asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");             // the last products have written their accumulators
    int l = lane;
    asm volatile("" : "+v"(l));                                                 // (addresses are formed here, not kept over the products)
    uint8_t *mine = stage[STAGES - 1] + wave * (ROWS * PIECES * 16);
    const int64_t down = 64 / PIECES * p.N * (int64_t)sizeof(T);                // from one store's rows to the next one's
    const int64_t off = l / PIECES * p.N * (int64_t)sizeof(T) + l % PIECES * 16;
#pragma unroll
    for (int r = 0; r < 128; r += ROWS) {
#pragma unroll
        for (int i = r / 16; i < (r + ROWS) / 16; ++i) {
            const int row = i * 16 - r + l % 16;
#pragma unroll
            for (int j = 0; j < 2 * HALF; ++j) {
                asm volatile("" : "+a"(acc[i][j]));         // (read after that wait)
                const int at = (j * 16 + l / 16 * 4) * (int)sizeof(T);
                store4((T *)(mine + row * (PIECES * 16) + exchanged(at / 16, row) * 16 + at % 16), acc[i][j], 4, true);
            }
        }
        // (a wave reads what it has written itself)
#pragma unroll
        for (int q = 0; q < ROWS * PIECES / 64; ++q) {
            const int row = (q * 64 + l) / PIECES, piece = l % PIECES;
            const u32x4 v = *(const u32x4 *)(mine + row * (PIECES * 16) + exchanged(piece, row) * 16);
            put<STREAM>((u32x4_any *)(y + off), v);
            y += down;
        }
    }
    if (!more) return;
    __syncthreads();
    request(k0 + STAGES - 1, STAGES - 1);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LA + LB) : "memory");           // all but the last one
    }
}

// Few rows of a (tokens, 64 at most): what counts is how fast b's rows arrive.  A workgroup takes 16 NT of them and all of a's, its W waves each a
// part of the blocks; a wave keeps R blocks on their way into its own ring in shared memory, and waits for nobody.  (Straight into registers a
// fragment's load takes a line a lane, since neighbouring lanes hold neighbouring rows: four times the cycles of one that goes along the rows, and
// more than the memory's time from some rows of a on: 12288 x 4096 with 1 row 13.3, with 64 rows 43 us.)  With FUSED, a is
// a tensor of type T, and the workgroup quantises it into shared memory while b's first rows are on their way: kTokenBytes of codes at most, since
// every workgroup does.  The waves' sums join in shared memory, in their order.
constexpr int kTokenBytes = 16384;
struct Tokens8 {
    Product8 p;
    const void *x;              // FUSED: a in its own type
    int64_t K;
};
template <typename T, int MT, int NT, int W, bool FUSED, bool A5, bool B5> __global__ __launch_bounds__(W * 64) void product8_tokens_kernel(Tokens8 s)
{
    static_assert(!FUSED || MT == 1, "tokens that are quantised here are 16 at most");
    constexpr int AT = FUSED ? 0 : MT, TILES = AT + NT, STAGE = TILES * 2048;
    constexpr int FIT = 32768 / (W * STAGE), R = FIT < 2 ? 2 : FIT;
    constexpr int WORDS = (kTokenBlocks + 3) / 4 + 1, ROWS = (TILES + 3) / 4 * 64;
    constexpr int SUMS = W * MT * NT * 1024;
    const Product8 &p = s.p;
    __shared__ __attribute__((aligned(1024))) uint8_t ring[W * R * STAGE > SUMS ? W * R * STAGE : SUMS];
    __shared__ uint32_t words[W][WORDS][ROWS];
    __shared__ __attribute__((aligned(16))) uint8_t own[FUSED ? kTokenBytes : 16];
    __shared__ uint8_t own_scales[FUSED ? kTokenBytes / 128 : 1];
    // (the wave's number in a scalar register: a product ignores the lanes' mask, so its conditions have to be branches)
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), r16 = lane % 16, quarter = lane / 16;
    // groups of a's rows that read the same rows of b follow each other
    const uint32_t item = xcd_contiguous_u32(blockIdx.x, gridDim.x);
    const int64_t m0 = (int64_t)(item % p.tiles_m) * (MT * 16), n0 = (int64_t)(item / p.tiles_m) * (NT * 16);
    const int per = (p.steps + W - 1) / W, k0 = wave * per, n = p.steps - k0 < per ? p.steps - k0 : per;
    const win_t wa = make_window(p.a + m0 * p.Kp, 0x7fffffff), wb = make_window(p.b + n0 * p.Kp, 0x7fffffff);
    // a load's eight rows of 128 bytes, their pieces at exchanged places
    uint32_t off[TILES][2];
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = h * 8 + lane / 8, row = (i < AT ? i : i - AT) * 16 + r;
            const int64_t last = i < AT ? p.M - 1 - m0 : p.N - 1 - n0;
            off[i][h] = (uint32_t)((row < last ? row : last) * p.Kp) + ((lane % 8) ^ ((r >> 1) & 7)) * 16;
        }
    const uint32_t to = (uint32_t)(uintptr_t)(lds_t)ring + wave * (R * STAGE);
    const auto request = [&](int i, int slot) {
        const int at = (k0 + i) * 128;
        const uint32_t q = to + slot * STAGE;
#pragma unroll
        for (int f = 0; f < TILES; ++f)
#pragma unroll
            for (int h = 0; h < 2; ++h) request_to_lds<16>(f < AT ? wa : wb, q + f * 2048 + h * 1024, off[f][h], at);
    };
    if (n > 0) {
        // the rows' scales, a word of four at a time, one row a lane
        const win_t wsa = make_window(p.a_scales + m0 * p.S, 0x7fffffff), wsb = make_window(p.b_scales + n0 * p.S, 0x7fffffff);
        const uint32_t first = (uint32_t)(uintptr_t)(lds_t)words[wave][0];
#pragma unroll
        for (int c = 0; c < ROWS; c += 64) {
            const int f = (c + lane) / 16, row = (f < AT ? f : f - AT) * 16 + r16;
            const int64_t last = f < AT ? p.M - 1 - m0 : p.N - 1 - n0;
            const uint32_t at = (uint32_t)((row < last ? row : last) * p.S);
            for (int w = 0; w <= (k0 + n - 1) / 4 - k0 / 4; ++w) {
                if (f < AT) request_to_lds<4>(wsa, first + (w * ROWS + c) * 4, at, (k0 / 4 + w) * 4);
                else if (f < TILES) request_to_lds<4>(wsb, first + (w * ROWS + c) * 4, at, (k0 / 4 + w) * 4);
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i < n) request(i, i);
    }
    if constexpr (FUSED) {
        // sixteen lanes a block, whole waves at a time; everything is requested before the first is waited for
        constexpr int TURNS = kTokenBytes / 128 / (W * 4);
        const int blocks = (int)p.M * p.steps, c = threadIdx.x % 16 * 8;
        u32x4 raw[TURNS];
#pragma unroll
        for (int q = 0; q < TURNS; ++q) {
            const int i = q * (W * 4) + threadIdx.x / 16, row = i / p.steps, k = i - row * p.steps;
            const int64_t left = s.K - (k * 128 + c);
            raw[q] = u32x4{0, 0, 0, 0};
            if (i < blocks && left > 0) raw[q] = load_row_vec<T, true, false>((const T *)s.x + row * s.K + k * 128 + c, 0, (int)(left < 8 ? left : 8));
        }
#pragma unroll
        for (int q = 0; q < TURNS; ++q) {
            const int i = q * (W * 4) + threadIdx.x / 16;
            if (q * (W * 4) + wave * 4 >= blocks) break;
            float v[8];
            unpack_vec(raw[q], v, T{});
            store_f8<8, A5, false>(own + i * 128, own_scales + i, c, i < blocks ? 128 : 0, v);
        }
        __syncthreads();
    }
    const int swap = (r16 >> 1) & 7, p0 = r16 * 128 + (quarter ^ swap) * 16, p1 = r16 * 128 + ((quarter + 4) ^ swap) * 16;
    const int64_t m_own = r16 < p.M ? r16 : p.M - 1;
    const auto fragment = [](const uint8_t *lo_at, const uint8_t *hi_at) {
        const u32x4 lo = *(const u32x4 *)lo_at, hi = *(const u32x4 *)hi_at;
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int i = 0, slot = 0; i < n; ++i, slot = slot + 1 < R ? slot + 1 : 0) {
        // the block is there: all but the R - 1 after it have arrived
        if (n - i >= R) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((R - 1) * TILES * 2) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const uint8_t *from = ring + wave * (R * STAGE) + slot * STAGE;
        const int k = k0 + i, shift = k % 4 * 8;
        const uint32_t *w = words[wave][k / 4 - k0 / 4];
        i32x8 A[MT], B[NT];
        uint32_t ca[MT], cb[NT];
#pragma unroll
        for (int f = 0; f < MT; ++f) {
            const uint8_t *mine = own + m_own * p.Kp + k * 128 + quarter * 16;
            A[f] = FUSED ? fragment(mine, mine + 64) : fragment(from + f * 2048 + p0, from + f * 2048 + p1);
            ca[f] = FUSED ? own_scales[m_own * p.steps + k] : w[f * 16 + r16] >> shift;
        }
#pragma unroll
        for (int f = 0; f < NT; ++f) {
            B[f] = fragment(from + (AT + f) * 2048 + p0, from + (AT + f) * 2048 + p1);
            cb[f] = w[(AT + f) * 16 + r16] >> shift;
        }
        if (i + R < n) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");              // read, before it is written over
            request(i + R, slot);
        }
#pragma unroll
        for (int x = 0; x < MT; ++x)
#pragma unroll
            for (int y = 0; y < NT; ++y) acc[x][y] = mfma8<B5, A5>(B[y], A[x], acc[x][y], cb[y], ca[x]);
    }
    __syncthreads();
    f32x4 *sums = (f32x4 *)ring;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[(wave * (MT * NT) + i * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int f0 = 0; f0 < MT * NT; f0 += W) {
        const int f = f0 + wave;
        if (f < MT * NT) {
            f32x4 v = sums[f * 64 + lane];
#pragma unroll
            for (int w = 1; w < W; ++w) v += sums[(w * (MT * NT) + f) * 64 + lane];
            const int64_t m = m0 + f / NT * 16 + r16, col = n0 + f % NT * 16 + quarter * 4;
            if (m < p.M) store4((T *)p.y + m * p.N + col, v, p.N - col, p.N % 4 == 0 && ((uintptr_t)p.y & (4 * sizeof(T) - 1)) == 0);
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

Plan8 plan_of(int64_t M, int64_t N, int64_t K)
{
    return plan8(M, N, (int)(f8_cols(K) / kBlockF8), tuning_env("GCG_P8"), tuning_env("GCG_P8S"));
}

template <int BM, int BN, int WM, int WN, typename T, bool A5, bool B5> int tile_launch(Product8 &p, const Plan8 &plan, hipStream_t st)
{
    p.tiles_m = (uint32_t)((p.M + BM - 1) / BM);
    p.tiles_n = (uint32_t)((p.N + BN - 1) / BN);
    return launch_main(product8_kernel<BM, BN, WM, WN, T, A5, B5>, dim3(p.tiles_m * p.tiles_n, (unsigned)plan.splits), dim3(WM * WN * 64), st, p);
}
template <typename T, int MT, int NT, int W, bool FUSED, bool A5, bool B5> int tokens_go(const Tokens8 &s, hipStream_t st)
{
    Tokens8 q = s;
    q.p.tiles_m = (uint32_t)((s.p.M + MT * 16 - 1) / (MT * 16));
    const dim3 grid((unsigned)((s.p.N + NT * 16 - 1) / (NT * 16) * q.p.tiles_m));
    return launch_main(product8_tokens_kernel<T, MT, NT, W, FUSED, A5, B5>, grid, dim3(W * 64), st, q);
}
// Rows of b for a workgroup, of up to 32 rows of a: 16 while the card's CUs have one workgroup each, else 32, which share a's fragments.  Eight waves where
// a wave of four would have sixteen blocks and the CU no other workgroup.  (FUSED changes nothing in it, so that sums are in the same order.)
template <typename T, int MT, bool FUSED, bool A5, bool B5> int tokens_tiles(const Tokens8 &s, hipStream_t st)
{
    const int64_t sixteens = (s.p.N + 15) / 16;
    if (s.p.steps > 4 * kTokenBlocks || (s.p.steps >= 64 && sixteens <= 256)) return tokens_go<T, MT, 1, 8, FUSED, A5, B5>(s, st);
    return sixteens <= 256 ? tokens_go<T, MT, 1, 4, FUSED, A5, B5>(s, st) : tokens_go<T, MT, 2, 4, FUSED, A5, B5>(s, st);
}
template <typename T, bool A5, bool B5> int product_launch(Product8 &p, const Plan8 &plan, hipStream_t st)
{
    if constexpr (sizeof(T) == 2) {
        if (plan.kernel == TOKENS) {
            const Tokens8 s = {p, nullptr, 0};
            if (p.M <= 16) return tokens_tiles<T, 1, false, A5, B5>(s, st);
            if (p.M <= 32) return tokens_tiles<T, 2, false, A5, B5>(s, st);
            const int tiles = tokens_estimate(p.M, p.N, p.steps).tiles;
            return tiles == 1 ? tokens_go<T, 4, 1, 4, false, A5, B5>(s, st) : tiles == 2 ? tokens_go<T, 4, 2, 4, false, A5, B5>(s, st)
                                                                                         : tokens_go<T, 4, 4, 4, false, A5, B5>(s, st);
        }
    }
    if (plan.kernel == TILE) return tile_launch<128, 128, 2, 2, T, A5, B5>(p, plan, st);
    // Results that the last-level cache does not hold go past it: 16384 x 12288 x 4096, 402 MB, with the kernel that quantises its operand before it
    // 830 us without the hint, 790 with it.
    const bool stream = sizeof(T) == 2 && p.M * p.N * (int64_t)sizeof(T) > kStreamBytes;
    const auto go = [&](auto launch, auto kernel, int64_t m0, int64_t M, int bn) {
        Product8 q = p;
        q.a += m0 * p.Kp;
        q.a_scales += m0 * p.S;
        q.y = (T *)p.y + m0 * p.N;
        q.M = M;
        q.tiles_m = (uint32_t)((M + 255) / 256);
        q.tiles_n = (uint32_t)((p.N + bn - 1) / bn);
        const int64_t items = (int64_t)q.tiles_m * q.tiles_n * plan.splits;
        return launch(kernel, dim3((unsigned)(items < 256 ? items : 256)), dim3(256), st, q);
    };
    const auto main_one = [](auto... a) { return launch_main(a...); };
    const auto plain_one = [](auto... a) { return launch_plain(a...); };
    if (plan.kernel == TALL) return go(main_one, product8_wide_kernel<128, T, A5, B5, false>, 0, p.M, 128);
    const int64_t M = p.M - plan.rest;
    const int rc = stream ? go(main_one, product8_wide_kernel<256, T, A5, B5, sizeof(T) == 2>, 0, M, 256)
                          : go(main_one, product8_wide_kernel<256, T, A5, B5, false>, 0, M, 256);
    return rc || plan.rest == 0 ? rc : go(plain_one, product8_wide_kernel<128, T, A5, B5, false>, M, plan.rest, 128);
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
    if (!holds(plan, M, N, (int)(f8_cols(K) / kBlockF8))) return (int)hipErrorInvalidValue;
    Product8 p = {a, a_scales, b, b_scales, y, plan.splits > 1 ? (float *)ws : nullptr, M, N, f8_cols(K), (int32_t)f8_scales(K),
                  (int32_t)(f8_cols(K) / 128), plan.split_steps, plan.splits, 0, 0};
    return dtype == GCG_BF16 ? product_type<bf16_t>(p, a5, b5, plan, st) : product_type<f16_t>(p, a5, b5, plan, st);
}

bool linear8_fits(int64_t M, int64_t K) { return M <= 16 && M * f8_cols(K) <= kTokenBytes; }

int linear8_launch(int dtype, int b5, const void *x, const uint8_t *b, const uint8_t *b_scales, void *y, int64_t M, int64_t N, int64_t K,
                   hipStream_t st)
{
    const Product8 p = {nullptr, nullptr, b, b_scales, y, nullptr, M, N, f8_cols(K), (int32_t)f8_scales(K), (int32_t)(f8_cols(K) / 128), 0, 1, 0, 0};
    const Tokens8 s = {p, x, K};
    if (dtype == GCG_BF16) return b5 ? tokens_tiles<bf16_t, 1, true, false, true>(s, st) : tokens_tiles<bf16_t, 1, true, false, false>(s, st);
    return b5 ? tokens_tiles<f16_t, 1, true, false, true>(s, st) : tokens_tiles<f16_t, 1, true, false, false>(s, st);
}

} // namespace gcg
