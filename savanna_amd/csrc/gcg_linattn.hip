// Linear attention with a decay for each head.  With f = exp(log_decay[h]) and a state S of dk x dv a batch entry and head:
//
//   S_t = f S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t
//
// Everything a sequence needs -- o, and the gradients dq, dk, dv -- has one form, a "walk" over rows
//
//   out_t = sum_{s <= t} f^(t-s) (a_t . b_s) c_s  +  f^(t+1) a_t S_0
//
// forward in time with (a, b, c) = (q, k, v) for o and (do, v, k) for dq (whose state is S transposed), and backward in time
// with (v, do, q) for dk and (k, q, do) for dv.  A walk goes over chunks of 64 rows.  Inside a chunk the sum is two
// matrix products with the decayed, masked scores P = (a b^T) * f^(t-s) between them; the rows before it come in through
// the state, out += f^(r+1) a S, and the state moves on by S = f^64 S + (b * f^(63-r))^T c.  Only non-negative powers
// of f are formed, so no decay over- or underflows into a wrong result (f = 0 and f = 1 included).
//
// A workgroup of four waves walks one head's rows for 32 columns of c, with its da x 32 state in fp32 in the waves' accumulation
// registers.  Wave w makes rows 16 w .. 16 w + 15 of P and of the output, and keeps a quarter of the state's rows.  P passes from
// one product to the next in registers: the scores are made transposed, so that a lane's four results of a tile are four
// consecutive positions of the next product's inner dimension; the products run over those positions in that order on both sides.
// b, c, the weighted c and the state's rounded copy are in LDS, two sets of each, so one barrier a chunk is enough.
//
// Rounding of 16-bit walks: the matrix instructions take 16-bit operands, so P and the state's copy are rounded to the type once,
// as the output is; the weighted c is given as a sum of two 16-bit parts (three where the state itself is a result), whose
// remainder, 2^-16 (2^-24), does not show in the fp32 state.  f16 has no range to spare: rows of P and blocks of the
// state's copy are scaled by powers of two, and the later parts of the weighted c too, so that neither large states nor
// small gradients leave it.  fp32 walks run on the fp32 matrix instructions, with nothing rounded.
#include "gcg_common.h"

namespace gcg {
namespace {

constexpr int CHUNK = 64, COLS = 32;        // rows of a chunk; columns of c a workgroup
constexpr int THREADS = 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// ---- operands of the matrix instructions ------------------------------------------------------------------
// A fragment is a lane's part of a 16 x KF operand: row (of the first operand) or column (of the second) lane % 16, and in
// KF / 4 inner positions of its lane group g = lane / 16.
template <typename T> struct Mat;
template <> struct Mat<bf16_t> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static constexpr int V = 8, KF = 32;
    static constexpr float MORE = 1.f;          // by how much a part is larger than what it stands for, times the part before
    static __device__ __forceinline__ f32x4 mul(const u32x4 &a, const u32x4 &b, const f32x4 &c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
    static __device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
};
template <> struct Mat<f16_t> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    static constexpr int V = 8, KF = 32;
    static constexpr float MORE = 4096.f;
    static __device__ __forceinline__ f32x4 mul(const u32x4 &a, const u32x4 &b, const f32x4 &c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
    static __device__ __forceinline__ float low(uint32_t w) { return (float)__builtin_bit_cast(v2, w)[0]; }
    static __device__ __forceinline__ float high(uint32_t w) { return (float)__builtin_bit_cast(v2, w)[1]; }
};
template <> struct Mat<float> {
    static constexpr int V = 4, KF = 16;
    static __device__ __forceinline__ f32x4 mul(const u32x4 &a, const u32x4 &b, f32x4 c)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    }
};

// KF rows of a tile in LDS as the inner dimension, 16 of its columns as the operand's rows: rows row0 + 4 g .. + 3 (and, in 16
// bits, row0 + 16 + 4 g .. + 3), the order in which a lane holds four results of a product in each of two tiles.  The columns are
// col0 + lane % 16, or, SPREAD, col0 + 8 (lane % 16 / 4) + lane % 4, so that two such tiles four columns apart give a lane eight
// columns side by side.  In 16 bits by the transposing LDS load, which hands lane i of 16 the i-th column of four rows of
// four lanes' 8 bytes each.
template <typename T, bool SPREAD>
__device__ __forceinline__ u32x4 inner_rows(const T *tile, int stride, int row0, int col0, int lane)
{
    const int l = lane & 15, g = lane >> 4;
    if constexpr (sizeof(T) == 2) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 *lds_p;
        const T *p = tile + (row0 + 4 * g + (l >> 2)) * stride + col0 + (SPREAD ? 8 : 4) * (l & 3);
        const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)p));
        const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p + 16 * stride)));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
        const int col = SPREAD ? 8 * (l >> 2) + (l & 3) : l;
        const float *p = (const float *)tile + (row0 + 4 * g) * stride + col0 + col;
        return u32x4{__float_as_uint(p[0]), __float_as_uint(p[stride]), __float_as_uint(p[2 * stride]), __float_as_uint(p[3 * stride])};
    }
}

// The powers of two that bring a largest magnitude to 1/2 .. 1 and back; 1 for none, infinities and NaN.
struct Range { float down, up; };
__device__ __forceinline__ Range range(float top)
{
    const uint32_t e = __float_as_uint(top) >> 23;
    if (e < 20 || e > 230) return {1.f, 1.f};
    return {__uint_as_float((253 - e) << 23), __uint_as_float((e + 1) << 23)};
}
__device__ __forceinline__ float wave_max(float x)
{
    for (int d = 1; d < 64; d *= 2) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}

// ---- arguments ----------------------------------------------------------------------------------------------
struct Rows { const void *p; int64_t sb, st, sh; };                    // strides of batch, time and head in elements
struct Walk {
    Rows a, b, c, out;
    const float *first;         // (bs, H, ., .) state before the first row, or null: element (i of a, j of c) at i * si + j * sj
    float *last;                // state after the last row, or null; same layout
    int64_t si, sj;
    float first_mul, last_mul, out_mul;
    int32_t da, dc;
    int32_t reverse;            // rows are walked from the sequence's end
    int32_t lead;               // a row r rows after the first sees `first` by f^(r + lead): 1, or 0 for a final state's gradient
    int32_t last_decays;        // `last` gets one factor f more (unless the sequence is empty)
};
struct Walks {
    Walk w[3];
    const float *log_decay;
    const int32_t *lengths;     // of the batch entries, or null: L
    float *seg;                 // states of the segments, [walk][bs][H][segment][da][dc]
    int64_t seg_walk[3];        // where a walk's begin
    int64_t L, seg_rows;        // seg_rows: multiple of 64
    int32_t n, bs, H, segments;
    int64_t groups;             // n * bs * H * segments
};

__device__ __forceinline__ float clamp_decay(float g) { return g < -1e4f ? -1e4f : g; }         // exp(-inf * 0) is 1 here, not NaN

// f^n as a sum of two floats: a state passes through thousands of such factors
__device__ __forceinline__ void power(float g, int n, float &hi, float &lo)
{
    const double p = exp((double)g * n);
    hi = (float)p;
    lo = (float)(p - (double)hi);
}

// vector of row elements at column c of D; FULL: the caller knows that all are there
template <typename T, bool FULL> __device__ __forceinline__ u32x4 load_cols(const T *row, int c, int D)
{
    constexpr int V = Mat<T>::V;
    if (FULL || c + V <= D) return *(const u32x4_any *)(row + c);
    u32x4 r = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (c + i < D) {
            if constexpr (sizeof(T) == 2) r[i / 2] |= (uint32_t)((const uint16_t *)row)[c + i] << (16 * (i & 1));
            else r[i] = ((const uint32_t *)row)[c + i];
        }
    return r;
}

// (group, slice) of a workgroup: the slices of a head follow one another on one XCD, whose L2 then holds the a and b they share
__device__ __forceinline__ void place(int64_t id, int slices, int64_t &group, int &slice)
{
    const int64_t block = id / (8 * slices);
    const int rest = (int)(id - block * 8 * slices);
    slice = rest >> 3;
    group = block * 8 + (rest & 7);
}

// OUT: the walk with its output; otherwise the state alone, of a segment that starts from nothing.  PARTS: 16-bit parts of the
// weighted c.  FULL: da is DA and dc a multiple of COLS.
template <typename T, int DA, bool OUT, int PARTS, bool FULL>
__global__ __launch_bounds__(THREADS) void walk_kernel(Walks args, int slices)
{
    typedef Mat<T> M;
    constexpr int V = M::V, KF = M::KF, KB = DA / KF, KG = CHUNK / KF;
    constexpr int BS = DA + V, CS = COLS + 16 / (int)sizeof(T), SS = DA + V;       // LDS row strides: 16 bytes past the row
    constexpr int SETS = (size_t)2 * (CHUNK * BS + (PARTS + 1) * CHUNK * CS + (OUT ? COLS * SS : 0)) * sizeof(T) <= 160 * 1024 ? 2 : 1;
    // 16-row tiles of the state a wave keeps, and of its two 16-column ones: whole blocks of KF rows in 16 bits
    constexpr int NW = DA == 64 ? 1 : 2, MT = DA == 64 ? 2 : DA / 64;
    constexpr bool F16 = __is_same(T, f16_t);
    constexpr size_t LDS = (size_t)SETS * (CHUNK * BS + (PARTS + 1) * CHUNK * CS + (OUT ? COLS * SS : 0)) * sizeof(T);
    static_assert(LDS <= 160 * 1024, "workgroup exceeds the 160 KB of LDS");
    __shared__ __align__(16) unsigned char lds_raw[LDS];
    __shared__ float lds_range[SETS][F16 && OUT ? KB : 1][2];
    T *const lds_b = (T *)lds_raw, *const lds_c = lds_b + SETS * CHUNK * BS, *const lds_w = lds_c + SETS * CHUNK * CS,
            *const lds_s = lds_w + SETS * PARTS * CHUNK * CS;

    int64_t group;
    int slice;
    place(blockIdx.x, slices, group, slice);
    if (group >= args.groups) return;
    const int seg = (int)(group % args.segments);
    group /= args.segments;
    const int h = (int)(group % args.H);
    group /= args.H;
    const int b = (int)(group % args.bs), job = (int)(group / args.bs);
    const Walk &wk = args.w[job];
    const int da = wk.da, dc = wk.dc, n0 = slice * COLS;
    if (n0 >= dc) return;
    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

    int64_t length = args.L;
    if (args.lengths) {
        length = args.lengths[b];
        length = length < 0 ? 0 : length > args.L ? args.L : length;
    }
    const int64_t from = seg * args.seg_rows, to = from + args.seg_rows < length ? from + args.seg_rows : length;
    const T *const pa = (const T *)wk.a.p + b * wk.a.sb + h * wk.a.sh, *const pb = (const T *)wk.b.p + b * wk.b.sb + h * wk.b.sh,
                  *const pc = (const T *)wk.c.p + b * wk.c.sb + h * wk.c.sh;
    T *const po = (T *)wk.out.p + b * wk.out.sb + h * wk.out.sh;
    const auto row_of = [&](int64_t r) { return wk.reverse ? length - 1 - r : r; };     // walk's row -> time
    const float decay = clamp_decay(args.log_decay[h]), l2 = decay * 1.44269504f;
    const int64_t state_at = (int64_t)(b * args.H + h) * da * dc;

    // ---- what does not change from chunk to chunk
    float f[4][4];              // OUT: f^(t-s) of this wave's rows (lane % 16) and the four columns of each score tile
    float row_mul = 0.f;
    if constexpr (OUT) {
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 16 * (wave - st) + l16 - 4 * g4 - i;
                f[st][i] = d >= 0 ? exp2f(l2 * d) : 0.f;
            }
        row_mul = exp2f(l2 * (16 * wave + l16));
    }
    float chunk_hi, chunk_lo;
    power(decay, CHUNK, chunk_hi, chunk_lo);

    // ---- the state: tile (mt, nw) holds rows m0 + 16 mt + 4 g4 .. + 3 of the slice's column c0 + 16 nw + l16
    const int m0 = DA == 64 ? (wave >> 1) * 32 : wave * (DA / 4), c0 = DA == 64 ? (wave & 1) * 16 : 0;
    f32x4 S[MT][NW];
    const float *first = nullptr;
    int64_t fi = wk.si, fj = wk.sj;
    float first_mul = 1.f;
    int lead = 1;
    if (OUT && args.segments > 1) {         // (the segments' states are joined: each begins from its own)
        first = args.seg + args.seg_walk[job] + ((int64_t)(b * args.H + h) * args.segments + seg) * da * dc;
        fi = dc; fj = 1;
        lead = seg == 0 ? wk.lead : 1;
    } else if (OUT && wk.first) {
        first = wk.first + state_at;
        first_mul = wk.first_mul;
        lead = wk.lead;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nw = 0; nw < NW; ++nw)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = m0 + 16 * mt + 4 * g4 + i, n = n0 + c0 + 16 * nw + l16;
                S[mt][nw][i] = first && m < da && n < dc ? first[m * fi + n * fj] * first_mul : 0.f;
            }
    const auto publish = [&](int set) {     // the state's rounded copy, columns as rows
        if constexpr (OUT) {
#pragma unroll
            for (int nw = 0; nw < NW; ++nw) {
                float by[MT / 2 ? MT / 2 : 1];
                if constexpr (F16) {
#pragma unroll
                    for (int kb = 0; kb < MT / 2; ++kb) {
                        float top = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(S[2 * kb + i / 4][nw][i & 3]));
                        const Range r = range(wave_max(top));
                        by[kb] = r.down;
                        if (lane == 0) lds_range[set][m0 / KF + kb][c0 / 16 + nw] = r.up;
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    T *to = lds_s + set * COLS * SS + (c0 + 16 * nw + l16) * SS + m0 + 16 * mt + 4 * g4;
                    f32x4 v = S[mt][nw];
                    if constexpr (F16) v *= by[mt / 2];
                    if constexpr (sizeof(T) == 2) *(u32x2 *)to = u32x2{M::pack(v[0], v[1]), M::pack(v[2], v[3])};
                    else *(f32x4 *)to = v;
                }
            }
        }
    };

    // ---- rows from memory: b in passes over the chunk's rows, c's 32 columns, and a's fragments of this wave's rows
    constexpr int BT = DA / V, BR = THREADS / BT, BP = CHUNK / BR;      // threads a row, rows a pass, passes
    constexpr int CT = COLS / V, CR = THREADS / CT, CP = CHUNK / CR;
    const int b_row = tid / BT, b_col = tid % BT * V, c_row = tid / CT, c_col = tid % CT * V;
    u32x4 rb[BP], rc[CP], ra[OUT ? KB : 1];
    const auto request = [&](int64_t at) {                              // the chunk of rows at ..; rows past the end repeat the last one
#pragma unroll
        for (int i = 0; i < BP; ++i) {
            const int64_t r = at + b_row + i * BR;
            rb[i] = load_cols<T, FULL>(pb + row_of(r < to ? r : to - 1) * wk.b.st, b_col, da);
        }
#pragma unroll
        for (int i = 0; i < CP; ++i) {
            const int64_t r = at + c_row + i * CR;
            rc[i] = load_cols<T, FULL>(pc + row_of(r < to ? r : to - 1) * wk.c.st, n0 + c_col, dc);
        }
        if constexpr (OUT) {
            const int64_t r = at + 16 * wave + l16;
            const T *row = pa + row_of(r < to ? r : to - 1) * wk.a.st;
#pragma unroll
            for (int k = 0; k < KB; ++k) ra[k] = load_cols<T, FULL>(row, k * KF + g4 * V, da);
        }
    };
    // into LDS: b, c and c weighted by f^(rows - 1 - r); rows past the end count for nothing
    const auto deposit = [&](int set, int rows) {
#pragma unroll
        for (int i = 0; i < BP; ++i) *(u32x4 *)(lds_b + (set * CHUNK + b_row + i * BR) * BS + b_col) = rb[i];
#pragma unroll
        for (int i = 0; i < CP; ++i) {
            const int r = c_row + i * CR;
            const float w = r < rows ? exp2f(l2 * (rows - 1 - r)) : 0.f;
            u32x4 v = rc[i];
            if (r >= rows) v = u32x4{0, 0, 0, 0};
            T *const to_c = lds_c + (set * CHUNK + r) * CS + c_col;
            if constexpr (OUT) *(u32x4 *)to_c = v;
            T *const to_w = lds_w + (set * PARTS * CHUNK + r) * CS + c_col;
            if constexpr (sizeof(T) == 2) {
                u32x4 part[PARTS];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float lo = M::low(v[j]) * w, hi = M::high(v[j]) * w;
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        part[p][j] = M::pack(lo, hi);
                        // the remainder is that of the part as stored, not of one that the compiler rounds again from the exact
                        // product (its mixed-precision f16 instructions do, an f16 step apart now and then)
                        asm("" : "+v"(part[p][j]));
                        if (p + 1 < PARTS) { lo = (lo - M::low(part[p][j])) * M::MORE; hi = (hi - M::high(part[p][j])) * M::MORE; }
                    }
                }
#pragma unroll
                for (int p = 0; p < PARTS; ++p) *(u32x4 *)(to_w + p * CHUNK * CS) = part[p];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * w);
                *(u32x4 *)to_w = v;
            }
        }
    };

    u32x4 a[OUT ? KB : 1];
    if (from < to) {
        request(from);
        const int rows = (int)(to - from < CHUNK ? to - from : CHUNK);
        deposit(0, rows);
        publish(0);
        __syncthreads();
    }
    int set = 0;
    for (int64_t at = from; at < to; at += CHUNK) {
        const int rows = (int)(to - at < CHUNK ? to - at : CHUNK);
        const bool more = at + CHUNK < to;
        if constexpr (OUT) {
#pragma unroll
            for (int k = 0; k < KB; ++k) a[k] = ra[k];
        }
        if (more) request(at + CHUNK);
        const T *const tb = lds_b + set * CHUNK * BS, *const tc = lds_c + set * CHUNK * CS, *const tw = lds_w + set * PARTS * CHUNK * CS,
                      *const ts = lds_s + set * COLS * SS;
        if constexpr (OUT) {
            // scores, transposed: rows 16 st + .. of b by this wave's rows of a
            f32x4 P[4];
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                P[st] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (st <= wave) {
#pragma unroll
                    for (int k = 0; k < KB; ++k)
                        P[st] = M::mul(*(const u32x4 *)(tb + (16 * st + l16) * BS + k * KF + g4 * V), a[k], P[st]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) P[st][i] = f[st][i] != 0.f ? P[st][i] * f[st][i] : 0.f;
                }
            }
            // output, transposed: this wave's rows by columns 8 g4 .. + 7 of the slice
            f32x4 O[2];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                O[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
                const int n = 8 * (l16 >> 2) + (l16 & 3) + 4 * nt;
#pragma unroll
                for (int k = 0; k < KB; ++k) {
                    const u32x4 x = *(const u32x4 *)(ts + n * SS + k * KF + g4 * V);
                    if constexpr (F16) O[nt] += M::mul(x, a[k], f32x4{0.f, 0.f, 0.f, 0.f}) * lds_range[set][k][g4 >> 1];
                    else O[nt] = M::mul(x, a[k], O[nt]);
                }
                const float m = row_mul * (at == from && lead == 0 ? 1.f : exp2f(l2));
#pragma unroll
                for (int i = 0; i < 4; ++i) O[nt][i] *= m;
            }
            // (f16: the scores of a row, like the state's copy, by a power of two that brings the largest to about 1)
            f32x4 inside[2] = {O[0], O[1]};
            float up = 1.f;
            if constexpr (F16) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(P[i >> 2][i & 3]));
                top = fmaxf(top, __shfl_xor(top, 16));
                const Range r = range(fmaxf(top, __shfl_xor(top, 32)));
                up = r.up;
#pragma unroll
                for (int st = 0; st < 4; ++st) P[st] *= r.down;
                inside[0] = inside[1] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int p = 0; p < KG; ++p) {
                u32x4 x;
                if constexpr (sizeof(T) == 2) {
                    if (2 * p > wave) continue;
                    x = u32x4{M::pack(P[2 * p][0], P[2 * p][1]), M::pack(P[2 * p][2], P[2 * p][3]), M::pack(P[2 * p + 1][0], P[2 * p + 1][1]),
                              M::pack(P[2 * p + 1][2], P[2 * p + 1][3])};
                } else {
                    if (p > wave) continue;
                    x = __builtin_bit_cast(u32x4, P[p]);
                }
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) inside[nt] = M::mul(inner_rows<T, true>(tc, CS, p * KF, 4 * nt, lane), x, inside[nt]);
            }
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) O[nt] = F16 ? O[nt] + inside[nt] * up : inside[nt];
            if (16 * wave + l16 < rows) {
                T *row = po + row_of(at + 16 * wave + l16) * wk.out.st;
                const int n = n0 + 8 * g4;
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = O[i >> 2][i & 3] * wk.out_mul;
                if (FULL || n + 8 <= dc) {
                    if constexpr (sizeof(T) == 2) {
                        *(u32x4_any *)(row + n) = u32x4{M::pack(v[0], v[1]), M::pack(v[2], v[3]), M::pack(v[4], v[5]), M::pack(v[6], v[7])};
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            *(u32x4_any *)(row + n + 4 * j) = u32x4{__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                                                    __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3])};
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (n + i < dc) Elem<T>::store(row + n + i, v[i]);
                }
            }
        }
        // the state moves on
        float hi = chunk_hi, lo = chunk_lo;
        const int turns = rows - (at == from && lead == 0 ? 1 : 0);
        if (turns != CHUNK) power(decay, turns, hi, lo);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nw = 0; nw < NW; ++nw)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[mt][nw][i] = fmaf(S[mt][nw][i], hi, S[mt][nw][i] * lo);
        if constexpr (F16) {
            // parts after the first are stored 2^12, 2^24 times larger and added up on their own, the smallest first
            f32x4 R[MT][NW];
#pragma unroll
            for (int part = PARTS - 1; part >= 0; --part) {
                if (part == PARTS - 1) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int nw = 0; nw < NW; ++nw) R[mt][nw] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int p = 0; p < KG; ++p)
#pragma unroll
                    for (int nw = 0; nw < NW; ++nw) {
                        const u32x4 y = inner_rows<T, false>(tw + part * CHUNK * CS, CS, p * KF, c0 + 16 * nw, lane);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) R[mt][nw] = M::mul(inner_rows<T, false>(tb, BS, p * KF, m0 + 16 * mt, lane), y, R[mt][nw]);
                    }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int nw = 0; nw < NW; ++nw) {
                        if (part > 0) R[mt][nw] *= 0x1p-12f;
                        else S[mt][nw] += R[mt][nw];
                    }
            }
        } else {
#pragma unroll
            for (int p = 0; p < KG; ++p) {
                u32x4 x[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) x[mt] = inner_rows<T, false>(tb, BS, p * KF, m0 + 16 * mt, lane);
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
#pragma unroll
                    for (int nw = 0; nw < NW; ++nw) {
                        const u32x4 y = inner_rows<T, false>(tw + part * CHUNK * CS, CS, p * KF, c0 + 16 * nw, lane);
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) S[mt][nw] = M::mul(x[mt], y, S[mt][nw]);
                    }
            }
        }
        if (more) {
            if constexpr (SETS == 1) __syncthreads();
            else set ^= 1;
            deposit(set, (int)(to - at - CHUNK < CHUNK ? to - at - CHUNK : CHUNK));
            publish(set);
            __syncthreads();
        }
    }

    // ---- the state after the last row
    float *last = nullptr;
    int64_t li = wk.si, lj = wk.sj;
    float last_mul = 1.f;
    if (!OUT) {
        last = args.seg + args.seg_walk[job] + ((int64_t)(b * args.H + h) * args.segments + seg) * da * dc;
        li = dc; lj = 1;
    } else if (args.segments == 1 && wk.last) {
        last = wk.last + state_at;
        last_mul = wk.last_mul * (wk.last_decays && length > 0 ? exp2f(l2) : 1.f);
    }
    if (last) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nw = 0; nw < NW; ++nw)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int m = m0 + 16 * mt + 4 * g4 + i, n = n0 + c0 + 16 * nw + l16;
                    if (m < da && n < dc) last[m * li + n * lj] = S[mt][nw][i] * last_mul;
                }
    }
    // rows of the segment's time span past the sequence's end
    if constexpr (OUT) {
        const int64_t end = from + args.seg_rows < args.L ? from + args.seg_rows : args.L;
        for (int64_t t = (from > length ? from : length) + (tid >> 5); t < end; t += THREADS / 32)
            if (n0 + (tid & 31) < dc) Elem<T>::store(po + t * wk.out.st + n0 + (tid & 31), 0.f);
    }
}

// The segments' states one after the other: in place of the state that a segment adds comes the one it begins with.
__global__ __launch_bounds__(THREADS) void join_kernel(Walks args)
{
    const int64_t heads = (int64_t)args.bs * args.H;
    const int job = blockIdx.z;
    const int64_t bh = blockIdx.y;
    const Walk &wk = args.w[job];
    const int e = blockIdx.x * THREADS + threadIdx.x, size = wk.da * wk.dc;
    if (e >= size || bh >= heads) return;
    int64_t length = args.L;
    if (args.lengths) {
        length = args.lengths[bh / args.H];
        length = length < 0 ? 0 : length > args.L ? args.L : length;
    }
    const float decay = clamp_decay(args.log_decay[bh % args.H]);
    float whole_hi, whole_lo;
    power(decay, (int)args.seg_rows, whole_hi, whole_lo);
    const int64_t at = bh * size + (e / wk.dc) * wk.si + (e % wk.dc) * wk.sj;
    float s = wk.first ? wk.first[at] * wk.first_mul : 0.f;
    float *p = args.seg + args.seg_walk[job] + bh * args.segments * size + e;
    for (int i = 0; i < args.segments; ++i, p += size) {
        const int64_t left = length - i * args.seg_rows;
        const int rows = (int)(left < 0 ? 0 : left < args.seg_rows ? left : args.seg_rows);
        const bool final = i + 1 == args.segments;
        const float add = final && !wk.last ? 0.f : *p;
        *p = s;
        if (rows > 0) {
            float hi = whole_hi, lo = whole_lo;
            const int turns = rows - (i == 0 && wk.first && wk.lead == 0 ? 1 : 0);
            if (turns != args.seg_rows) power(decay, turns, hi, lo);
            s = fmaf(s, hi, s * lo) + add;
        }
    }
    if (wk.last) wk.last[at] = s * wk.last_mul * (wk.last_decays && length > 0 ? expf(decay) : 1.f);
}

// ---- one token ------------------------------------------------------------------------------------------------
struct Step {
    const void *q, *k, *v;
    void *o;
    int64_t qb, qh, kb, kh, vb, vh, ob, oh;
    const float *log_decay;
    float *state;
    int32_t bs, H, dk, dv, cols;        // cols: columns of the state a workgroup takes, a multiple of 4
    float scale;
};

// A workgroup takes some columns of one head's state: each thread four columns of every R-th row, read, moved on, written back and
// multiplied with q on the way; the threads of a column add up through LDS.  ALIGNED: dv is a multiple of 4.
template <typename T, bool ALIGNED> __global__ __launch_bounds__(THREADS) void step_kernel(Step a)
{
    __shared__ float lq[GCG_LINEAR_MAX_DIM], lk[GCG_LINEAR_MAX_DIM];
    __shared__ __align__(16) float part[4 * THREADS];           // [thread of a column][column]
    const int slices = (a.dv + a.cols - 1) / a.cols;
    const int64_t bh = blockIdx.x / slices;
    const int slice = blockIdx.x % slices, h = (int)(bh % a.H), tid = threadIdx.x;
    const int64_t b = bh / a.H;
    const T *q = (const T *)a.q + b * a.qb + h * a.qh, *k = (const T *)a.k + b * a.kb + h * a.kh, *v = (const T *)a.v + b * a.vb + h * a.vh;
    const int quads = a.cols / 4, R = THREADS / quads, col = slice * a.cols + tid % quads * 4, row0 = tid / quads;
    const float f = expf(clamp_decay(a.log_decay[h]));
    float vv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vv[i] = col + i < a.dv ? Elem<T>::load(v + col + i) : 0.f;
    for (int i = tid; i < a.dk; i += THREADS) {
        lq[i] = Elem<T>::load(q + i);
        lk[i] = Elem<T>::load(k + i);
    }
    float *const s = a.state + bh * a.dk * a.dv + col;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    if (row0 < R && col < a.dv) {
        constexpr int U = 8;
        for (int m = row0; m < a.dk; m += U * R) {
            f32x4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = m + u * R;
                x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (r < a.dk) {
                    if (ALIGNED) x[u] = *(const f32x4 *)(s + (int64_t)r * a.dv);
                    else
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (col + i < a.dv) x[u][i] = s[(int64_t)r * a.dv + i];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = m + u * R;
                if (r < a.dk) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[u][i] = fmaf(x[u][i], f, lk[r] * vv[i]);
                        o[i] = fmaf(lq[r], x[u][i], o[i]);
                    }
                    if (ALIGNED) *(f32x4 *)(s + (int64_t)r * a.dv) = x[u];
                    else
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (col + i < a.dv) s[(int64_t)r * a.dv + i] = x[u][i];
                }
            }
        }
    }
    if (row0 < R) *(f32x4 *)(part + (row0 * quads + tid % quads) * 4) = o;
    __syncthreads();
    if (tid < a.cols && slice * a.cols + tid < a.dv) {
        float sum = 0.f;
        for (int r = 0; r < R; ++r) sum += part[r * a.cols + tid];
        Elem<T>::store((T *)a.o + b * a.ob + h * a.oh + slice * a.cols + tid, sum * a.scale);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------
template <typename T, int DA, bool OUT, int PARTS> int walk_go(const Walks &w, int slices, bool full, hipStream_t st)
{
    const int64_t blocks = (w.groups + 7) / 8 * 8 * slices;
    const dim3 grid((unsigned)blocks), block(THREADS);
    if (blocks > 0x7fffffffLL) return (int)hipErrorInvalidConfiguration;
    if (full) return launch_plain(walk_kernel<T, DA, OUT, PARTS, true>, grid, block, st, w, slices);
    return launch_plain(walk_kernel<T, DA, OUT, PARTS, false>, grid, block, st, w, slices);
}
template <typename T, bool OUT, int PARTS> int walk_width(const Walks &w, hipStream_t st)
{
    int da = 0, dc = 0;
    bool full = true;
    for (int i = 0; i < w.n; ++i) {
        da = w.w[i].da > da ? w.w[i].da : da;
        dc = w.w[i].dc > dc ? w.w[i].dc : dc;
    }
    const int DA = da <= 64 ? 64 : da <= 128 ? 128 : 256;
    for (int i = 0; i < w.n; ++i) full = full && w.w[i].da == DA && w.w[i].dc % COLS == 0;
    const int slices = (dc + COLS - 1) / COLS;
    if (DA == 64) return walk_go<T, 64, OUT, PARTS>(w, slices, full, st);
    if (DA == 128) return walk_go<T, 128, OUT, PARTS>(w, slices, full, st);
    return walk_go<T, 256, OUT, PARTS>(w, slices, full, st);
}
// the states alone (segments) or the outputs; parts: of the weighted c, 3 where a state is a result
template <typename T, bool OUT> int walk_parts(const Walks &w, bool states, hipStream_t st)
{
    if constexpr (sizeof(T) == 4) return walk_width<T, OUT, 1>(w, st);
    else return states ? walk_width<T, OUT, 3>(w, st) : walk_width<T, OUT, 2>(w, st);
}
template <typename T> int run_walks(const Walks &w, bool states, hipStream_t st)
{
    if (w.segments > 1) {
        int rc = walk_parts<T, false>(w, states, st);
        if (rc) return rc;
        int size = 0;
        for (int i = 0; i < w.n; ++i) size = w.w[i].da * w.w[i].dc > size ? w.w[i].da * w.w[i].dc : size;
        const dim3 grid((unsigned)((size + THREADS - 1) / THREADS), (unsigned)(w.bs * w.H), (unsigned)w.n), block(THREADS);
        rc = launch_plain(join_kernel, grid, block, st, w);
        if (rc) return rc;
    }
    return walk_parts<T, true>(w, states && w.segments == 1, st);
}

// Segments of a walk: as many as give every CU two workgroups, of at least 512 rows, where the heads alone do not.
int segments_of(int64_t walks, int64_t bs, int64_t L, int H, int dc)
{
    const int64_t units = walks * bs * H * ((dc + COLS - 1) / COLS);
    if (units >= 256) return 1;
    int64_t n = (512 + units - 1) / units, most = L / 512;
    n = n < most ? n : most;
    return n < 1 ? 1 : (int)n;
}
int64_t seg_rows_of(int64_t L, int segments) { return ((L + segments - 1) / segments + CHUNK - 1) / CHUNK * CHUNK; }

void plan(Walks &w, int64_t L, int dc)
{
    w.segments = segments_of(w.n, w.bs, L, w.H, dc);
    w.seg_rows = seg_rows_of(L, w.segments);
    w.segments = (int)((L + w.seg_rows - 1) / w.seg_rows);
    w.L = L;
    w.groups = (int64_t)w.n * w.bs * w.H * w.segments;
    int64_t at = 0;
    for (int i = 0; i < w.n; ++i) {
        w.seg_walk[i] = at;
        at += (int64_t)w.bs * w.H * w.segments * w.w[i].da * w.w[i].dc;
    }
}

int run_t(int dtype, const Walks &w, bool states, hipStream_t st)
{
    switch (dtype) {
    case GCG_F32: return run_walks<float>(w, states, st);
    case GCG_BF16: return run_walks<bf16_t>(w, states, st);
    default: return run_walks<f16_t>(w, states, st);
    }
}

Rows rows_of(const void *p, const int64_t *s) { return {p, s[0], s[1], s[2]}; }

} // namespace

size_t linear_attn_workspace(int64_t bs, int64_t L, int H, int dk, int dv, bool backward)
{
    const int walks = backward ? 3 : 1, dc = backward && dk > dv ? dk : dv;
    int segments = segments_of(walks, bs, L, H, dc);
    const int64_t rows = seg_rows_of(L, segments);
    segments = (int)((L + rows - 1) / rows);
    return segments > 1 ? (size_t)walks * bs * H * segments * dk * dv * sizeof(float) : 0;
}

int linear_attn_fwd_launch(int dtype, const void *q, const void *k, const void *v, const int64_t *strides, const float *log_decay,
                           const float *initial, const int32_t *lengths, void *o, float *final, void *ws, int64_t bs, int64_t L, int H,
                           int dk, int dv, float scale, hipStream_t st)
{
    Walks w = {};
    w.n = 1; w.bs = (int)bs; w.H = H;
    w.log_decay = log_decay;
    w.lengths = lengths;
    w.seg = (float *)ws;
    w.w[0] = {rows_of(q, strides), rows_of(k, strides + 3), rows_of(v, strides + 6), rows_of(o, strides + 9), initial, final, dv, 1, 1.f, 1.f,
              scale, dk, dv, 0, 1, 0};
    plan(w, L, dv);
    return run_t(dtype, w, final != nullptr, st);
}

int linear_attn_bwd_launch(int dtype, const void *d_o, const void *q, const void *k, const void *v, const int64_t *strides,
                           const float *log_decay, const float *initial, const int32_t *lengths, const float *dfinal, void *dq, void *d_k,
                           void *d_v, float *dinitial, void *ws, int64_t bs, int64_t L, int H, int dk, int dv, float scale, hipStream_t st)
{
    Walks w = {};
    w.n = 3; w.bs = (int)bs; w.H = H;
    w.log_decay = log_decay;
    w.lengths = lengths;
    w.seg = (float *)ws;
    const Rows o_ = rows_of(d_o, strides), q_ = rows_of(q, strides + 3), k_ = rows_of(k, strides + 6), v_ = rows_of(v, strides + 9);
    // the scale multiplies outputs, and what a given state's gradient adds to them carries none: it goes in divided by it
    w.w[0] = {o_, v_, k_, rows_of(dq, strides + 12), initial, nullptr, 1, dv, 1.f, 1.f, scale, dv, dk, 0, 1, 0};
    w.w[1] = {v_, o_, q_, rows_of(d_k, strides + 15), dfinal, nullptr, 1, dv, 1.f / scale, 1.f, scale, dv, dk, 1, 0, 0};
    w.w[2] = {k_, q_, o_, rows_of(d_v, strides + 18), dfinal, dinitial, dv, 1, 1.f / scale, scale, scale, dk, dv, 1, dfinal ? 0 : 1, 1};
    plan(w, L, dk > dv ? dk : dv);
    return run_t(dtype, w, dinitial != nullptr, st);
}

int linear_attn_step_launch(int dtype, const void *q, const void *k, const void *v, void *o, const int64_t *s, const float *log_decay,
                            float *state, int64_t bs, int H, int dk, int dv, float scale, hipStream_t st)
{
    Step a = {q, k, v, o, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], log_decay, state, (int32_t)bs, H, dk, dv, 0, scale};
    a.cols = (dv + 3) / 4 * 4;
    while (a.cols > 32 && bs * H * ((dv + a.cols - 1) / a.cols) < 512) a.cols = (a.cols / 2 + 3) / 4 * 4;
    const int64_t blocks = bs * H * ((dv + a.cols - 1) / a.cols);
    if (blocks > 0x7fffffffLL) return (int)hipErrorInvalidConfiguration;
    const dim3 grid((unsigned)blocks), block(THREADS);
    const bool aligned = dv % 4 == 0 && ((uintptr_t)state & 15) == 0;
    switch (dtype) {
    case GCG_F32: return aligned ? launch_main(step_kernel<float, true>, grid, block, st, a) : launch_main(step_kernel<float, false>, grid, block, st, a);
    case GCG_BF16: return aligned ? launch_main(step_kernel<bf16_t, true>, grid, block, st, a) : launch_main(step_kernel<bf16_t, false>, grid, block, st, a);
    default: return aligned ? launch_main(step_kernel<f16_t, true>, grid, block, st, a) : launch_main(step_kernel<f16_t, false>, grid, block, st, a);
    }
}

} // namespace gcg
