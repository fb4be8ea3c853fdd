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
// A workgroup of twelve waves walks one head's rows for 32 columns of c: four waves make the output, 16 rows of a chunk each, four
// hold the da x 32 state in fp32 in their accumulation registers and move it on, and four bring rows from memory, two chunks
// ahead, into LDS.  The three meet at one barrier a chunk; b, c, the weighted c and the state's rounded copy have two sets in
// LDS.  P passes from one product to the next in registers: the scores are made transposed, so that a lane's four results of a
// tile are four consecutive positions of the next product's inner dimension; the products run over those positions in that order
// on both sides.  Narrow slices fill the card from few heads (2 sequences of 32 heads of 128: 256 workgroups) and keep the
// state small; a and b, which a head's slices share, come from the XCD's L2, where they are put side by side.
//
// Measured, bf16, 2 x 8192 rows of 32 heads of 128: forward 152 us, backward (three walks in one launch) 467 us, 3.5 and 3.4
// TB/s of what it has to move (167 and 456 when launched back to back).  Neither LDS (busy for 35 % of a chunk's time) nor the
// matrix units (24 %) bound it, but a chunk's chain: LDS reads, two dependent products, rounding, the next state's copy, the
// barrier; and HBM's latency, which shows through: back to back the forward takes 149 us where a head's rows follow each other
// in memory and 117 where every head reads the same ones from L2.  Tried, within 5 % or slower: two workgroups of 128 registers a
// CU, three sets in LDS with the scores and the state's operands a chunk ahead, other orders of heads over XCDs; waves for both
// the state and the rows, 8 a workgroup, 165 and 510 us.
//
// Few heads, long sequences: the rows are cut into segments whose states are made first, each from nothing, and joined by a scan
// over segments; then all segments run at once (8 heads, 131072 rows: 488 us in three launches; in one segment 2.0 ms).
//
// Rounding of 16-bit walks: the matrix instructions take 16-bit operands, so P and the state's copy are rounded to the type once,
// as the output is (against 64 bits that makes 0.0023 of the 0.0017 that rounding the output alone gives in bf16, 0.00029 of 0.00021 in
// f16); the weighted c is given as a sum of two 16-bit parts (three where the state itself is a result), whose
// remainder, 2^-16 (2^-24), does not show in the fp32 state.  f16 has no range to spare: rows of P and the
// columns of the state's copy, 32 rows at a time, are scaled by powers of two, and the later parts of the weighted c too, so that neither
// large states nor small gradients leave it.  fp32 walks run on the fp32 matrix instructions, with nothing rounded.
#include "gcg_common.h"

namespace gcg {
namespace {

constexpr int CHUNK = 64, COLS = 32;        // rows of a chunk; columns of c a workgroup
constexpr int THREADS = 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));

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
    // (rounding is off by at most 16, which 2^11 brings to 32768: the next part and its own rounding stay in range for every f16)
    static constexpr float MORE = 2048.f;
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

// ---- tiles in LDS -------------------------------------------------------------------------------------------
// A tile's rows lie one after the other without padding; inside a row, 16-byte pieces (in b and the state's copy) or halves (in
// c and the weighted c) change places by the row, so that the lanes that one LDS cycle serves touch every bank once.  Measured
// with 16 waves, cycles a wave: 16-byte reads of 16 rows 4.0 (rows padded by 16 bytes: 8.0); transposing reads 2.3 (padded,
// rows in their own order: 4.0).
//
// b, and the state's copy with a slice's columns as rows: rows of DA elements
template <typename T, int DA> __device__ __forceinline__ int wide_at(int row, int piece)
{
    const int swap = DA * sizeof(T) >= 256 ? row & 15 : (row & 2) | (row & 8) >> 1 | (row >> 2 & 1);
    return row * DA + (piece ^ swap) * Mat<T>::V;
}
// c and the weighted c: rows of COLS elements (fp32: padded by 16 bytes, which serves its plain loads)
template <typename T> constexpr int kSliceRow = sizeof(T) == 2 ? COLS : COLS + 4;
template <typename T, int BIT> __device__ __forceinline__ int slice_at(int row, int col)
{
    if constexpr (sizeof(T) == 2) return row * COLS + (col ^ (row >> BIT & 1) << 4);
    else return row * kSliceRow<T> + col;
}
constexpr int C_BIT = 2, W_BIT = 3;

// The order of a tile's 16 rows as a product's inner dimension: lane group g takes four of them, its lanes' results or loads in
// this order on both sides.  The scores' (and c's) order is that of the product that makes them; the state's update has
// one that suits both b's and the weighted c's banks.
__device__ __forceinline__ int score_row(int g, int i) { return 4 * g + i; }
template <typename T> __device__ __forceinline__ int update_row(int g, int i)
{
    return sizeof(T) == 2 ? 8 * (g & 1) + 2 * i + ((i >> 1 ^ g >> 1) & 1) : 4 * g + i;
}
// A lane's part of KF rows at p (the lane's own element there) as the inner dimension, 16 columns as the operand's rows.  In 16
// bits by the transposing load, which hands lane i of 16 the i-th column of four rows, of which four lanes each
// address 8 bytes; `far` is the distance of the next 16 rows.  In fp32 by the offsets of the group's four rows.
template <typename T> __device__ __forceinline__ u32x4 load_inner(const T *p, int far)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 *lds_p;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)p));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p + far)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ u32x4 load_inner(const float *p, const int (&row)[4])
{
    return u32x4{__float_as_uint(p[row[0]]), __float_as_uint(p[row[1]]), __float_as_uint(p[row[2]]), __float_as_uint(p[row[3]])};
}
// Where column n of a slice lies in LDS as a row of the state's copy and as a column of c: a product's 16 of them side by side
// give a lane columns 8 g .. 8 g + 3, the next 16 columns 8 g + 4 .. 8 g + 7 of the output.
__device__ __forceinline__ int spread(int n) { return 16 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3); }

// The powers of two that bring a largest magnitude to 1/2 .. 1 and back; 1 for none, infinities and NaN.
struct Range { float down, up; };
__device__ __forceinline__ Range range(float top)
{
    const uint32_t e = __float_as_uint(top) >> 23;
    if (e < 20 || e > 230) return {1.f, 1.f};
    return {__uint_as_float((253 - e) << 23), __uint_as_float((e + 1) << 23)};
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
    int32_t L, seg_rows;        // seg_rows: multiple of 64
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

// (group, slice) of a workgroup: the slices of a head follow one another on one XCD, whose L2 then holds the a and b they share
__device__ __forceinline__ void place(int64_t id, int slices, int64_t &group, int &slice)
{
    const int64_t block = id / (8 * slices);
    const int rest = (int)(id - block * 8 * slices);
    slice = rest >> 3;
    group = block * 8 + (rest & 7);
}

// One workgroup's walk: its place, its rows in memory and in LDS, and the parts of a chunk's work.
//
// OUT: with an output; otherwise the state alone, of a segment that starts from nothing.  PARTS: 16-bit parts of the weighted
// c.  FULL: da is DA and dc a multiple of COLS; otherwise both are multiples of a vector.
template <typename T, int DA, bool OUT, int PARTS, bool FULL> struct Walker {
    typedef Mat<T> M;
    static constexpr bool F16 = __is_same(T, f16_t);
    static constexpr int V = M::V, KF = M::KF, KB = DA / KF, KG = CHUNK / KF;
    static constexpr int CS = kSliceRow<T>;
    static constexpr size_t ONE = (size_t)(CHUNK * DA + (PARTS + OUT) * CHUNK * CS + (OUT ? COLS * DA : 0)) * sizeof(T) +
                                  (F16 && OUT ? KB * COLS : 0);
    static constexpr int SETS = 2 * ONE <= 160 * 1024 ? 2 : 1;
    static_assert(SETS * ONE <= 160 * 1024, "workgroup exceeds the 160 KB of LDS");
    // 16-row tiles of the state a wave keeps, and of its two 16-column ones: whole blocks of KF rows in 16 bits
    static constexpr int NW = DA == 64 ? 1 : 2, MT = DA == 64 ? 2 : DA / 64;
    static constexpr bool DEEP = DA * sizeof(T) <= 256;     // registers for the rows of two chunks ahead (else one)
    // The output's, the state's and the fetching waves, four each: 168 registers a lane.  Walks with rows of more than 256 bytes do
    // not fit in that but for bf16's; there the state's waves fetch too (JOINT).
    static constexpr bool JOINT = OUT && !DEEP && !__is_same(T, bf16_t);
    static constexpr int WAVES = 4 + (OUT ? 4 : 0) + (JOINT ? 0 : 4);
    static constexpr int BT = DA / V, BR = 256 / BT, BP = CHUNK / BR;      // b: threads a row, rows a pass, passes
    static constexpr int CT = COLS / V, CR = 256 / CT, CP = CHUNK / CR;    // c

    struct Lds {
        __align__(16) T b[SETS][CHUNK * DA];
        __align__(16) T c[SETS][OUT ? CHUNK * CS : 1];
        __align__(16) T w[SETS][PARTS][CHUNK * CS];
        __align__(16) T s[SETS][OUT ? COLS * DA : 1];
    };

    const Walks &args;
    const Walk &wk;
    Lds &lds;
    // f16: by how much KF rows of a column of the state's copy are smaller, as an fp32 exponent (a workgroup without a copy has no
    // place for it either).  Every column has its own, so that neither a neighbour 2^14 times larger nor one without finite values
    // takes its bits.  (Two exchanges of lanes find it, six one for 16 columns: f16, 2 x 8192 rows of 32 heads of 128, forward 182 us
    // and 188 with one for 16, backward 533 and 561.)
    static __device__ __forceinline__ uint8_t *range_of(int set, int block)
    {
        __shared__ __align__(8) uint8_t place[SETS][KB][COLS];
        return place[set][block];
    }
    // columns 8 g4 + 4 nt .. + 3
    static __device__ __forceinline__ f32x4 ranges(uint32_t w)
    {
        return f32x4{__uint_as_float(w << 23 & 0x7f800000u), __uint_as_float(w << 15 & 0x7f800000u), __uint_as_float(w << 7 & 0x7f800000u),
                     __uint_as_float(w >> 1 & 0x7f800000u)};
    }
    int b, h, seg, job, da, dc, n0, lane, l16, g4, wave, tid;
    int length, from, rows;     // of the sequence; the segment's first row and its rows
    int64_t state_at;
    float decay, l2;
    int lead;                   // of the first chunk

    __device__ Walker(const Walks &args_, const Walk &wk_, Lds &lds_) : args(args_), wk(wk_), lds(lds_) {}

    // ---- rows in memory
    // A chunk of one tensor is a window from its lowest row to its highest row's last column; a lane's place in it is a 32-bit
    // offset that does not change from chunk to chunk but for a shift (a chunk of fewer rows, walked backwards).  Rows past the end
    // lie outside the window, and so do columns past the row's end, whose lanes hold an offset beyond any window: such
    // loads return zero and such stores are dropped, so no access is conditional, and the waits before the use of one chunk's rows
    // leave the next chunks' requests in flight.  A stream hands out the windows of one chunk after the other; what it needs is in
    // scalar registers (through readfirstlane, or the compiler loads it from the kernel's arguments again in every chunk and
    // waits for that).
    static constexpr uint32_t NOWHERE = 0xc0000000u;
    struct Chunk { win_t win; uint32_t shift; };
    struct Stream {
        uint64_t base;          // of the chunk's lowest row, if the chunk is full
        int64_t step;
        int unit, tail, left;   // bytes from row to row, and of a row; rows from this chunk on
        bool reverse;
        __device__ __forceinline__ Chunk next()
        {
            const int rows = left < 0 ? 0 : left < CHUNK ? left : CHUNK;
            const int absent = reverse ? (CHUNK - rows) * unit : 0;
            const Chunk c = {make_window((const void *)(base + (uint32_t)absent), rows ? (rows - 1) * unit + tail : 0), 0u - (uint32_t)absent};
            base += step;
            left -= CHUNK;
            return c;
        }
    };
    static __device__ __forceinline__ uint64_t uniform(uint64_t x)
    {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32)) << 32 |
               (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x);
    }
    __device__ __forceinline__ Stream stream(const Rows &r, int cols) const
    {
        Stream s;
        const int64_t row = wk.reverse ? (int64_t)length - from - CHUNK : from;
        s.reverse = __builtin_amdgcn_readfirstlane(wk.reverse) != 0;
        s.base = uniform((uint64_t)r.p + (uint64_t)((b * r.sb + h * r.sh + row * r.st) * (int64_t)sizeof(T)));
        s.unit = __builtin_amdgcn_readfirstlane((int)r.st * (int)sizeof(T));
        s.step = s.reverse ? -(int64_t)CHUNK * s.unit : (int64_t)CHUNK * s.unit;
        s.tail = __builtin_amdgcn_readfirstlane(cols * (int)sizeof(T));
        s.left = __builtin_amdgcn_readfirstlane(rows);
        return s;
    }
    __device__ __forceinline__ uint32_t offset(const Rows &r, int i, int col, int cols) const
    {
        if (!FULL && col >= cols) return NOWHERE;
        return (uint32_t)(wk.reverse ? CHUNK - 1 - i : i) * (uint32_t)r.st * (uint32_t)sizeof(T) + (uint32_t)(col * sizeof(T));
    }
    static __device__ __forceinline__ u32x4 load(const Chunk &c, uint32_t off) { return win_load_aux<0, u32x4>(c.win, off + c.shift); }
    __device__ __forceinline__ int rows_in(int chunk) const { return rows - chunk * CHUNK < CHUNK ? rows - chunk * CHUNK : CHUNK; }

    // ---- the fetching waves: rows into LDS
    struct Fetch { u32x4 b[BP], c[CP]; };
    uint32_t ob[BP], oc[CP];
    int b_row, b_col, c_row, c_col;
    Stream sb, sc;

    __device__ __forceinline__ void fetch(Fetch &f)
    {
        const Chunk cb = sb.next(), cc = sc.next();
#pragma unroll
        for (int i = 0; i < BP; ++i) f.b[i] = load(cb, ob[i]);
#pragma unroll
        for (int i = 0; i < CP; ++i) f.c[i] = load(cc, oc[i]);
        __builtin_amdgcn_sched_barrier(0);      // requests stay in order, which is what the waits count by
    }
    __device__ __forceinline__ void deposit_b(int set, const Fetch &f) const
    {
#pragma unroll
        for (int i = 0; i < BP; ++i) *(u32x4 *)(lds.b[set] + wide_at<T, DA>(b_row + i * BR, b_col / V)) = f.b[i];
    }
    // b, c and c weighted by f^(rows - 1 - r); rows past the end count for nothing.  Waves that do nothing else weight c first, while
    // the others' reads have LDS to themselves.
    __device__ __forceinline__ void deposit(int set, const Fetch &f, int rows) const
    {
        if constexpr (JOINT) deposit_b(set, f);
        u32x4 v[CP], part[CP][sizeof(T) == 2 ? PARTS : 1];
#pragma unroll
        for (int i = 0; i < CP; ++i) {
            const int r = c_row + i * CR;
            const float w = r < rows ? exp2f(l2 * (rows - 1 - r)) : 0.f;
            v[i] = f.c[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = r < rows ? v[i][j] : 0;
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float lo = M::low(v[i][j]) * w, hi = M::high(v[i][j]) * w;
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        part[i][p][j] = M::pack(lo, hi);
                        // the remainder is that of the part as stored, not of one that the compiler rounds again from the exact
                        // product (its mixed-precision f16 instructions do, an f16 step apart now and then)
                        asm("" : "+v"(part[i][p][j]));
                        if (p + 1 < PARTS) { lo = (lo - M::low(part[i][p][j])) * M::MORE; hi = (hi - M::high(part[i][p][j])) * M::MORE; }
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) part[i][0][j] = __float_as_uint(__uint_as_float(v[i][j]) * w);
            }
        }
        if constexpr (!JOINT) {
            __builtin_amdgcn_sched_barrier(0);
            deposit_b(set, f);
        }
#pragma unroll
        for (int i = 0; i < CP; ++i) {
            const int r = c_row + i * CR;
            if constexpr (OUT) {
                *(u32x2 *)(lds.c[set] + slice_at<T, C_BIT>(r, spread(c_col))) = u32x2{v[i][0], v[i][1]};
                *(u32x2 *)(lds.c[set] + slice_at<T, C_BIT>(r, spread(c_col + V / 2))) = u32x2{v[i][2], v[i][3]};
            }
#pragma unroll
            for (int p = 0; p < (sizeof(T) == 2 ? PARTS : 1); ++p) *(u32x4 *)(lds.w[set][p] + slice_at<T, W_BIT>(r, c_col)) = part[i][p];
        }
    }
    __device__ __forceinline__ void fetch_setup(int t)
    {
        b_row = t / BT; b_col = t % BT * V; c_row = t / CT; c_col = t % CT * V;
        sb = stream(wk.b, da);
        sc = stream(wk.c, dc);
#pragma unroll
        for (int i = 0; i < BP; ++i) ob[i] = offset(wk.b, b_row + i * BR, b_col, da);
#pragma unroll
        for (int i = 0; i < CP; ++i) oc[i] = offset(wk.c, c_row + i * CR, n0 + c_col, dc);
    }
    // `even` and `odd` hold the rows of the next two chunks (not DEEP: one is both)
    __device__ __forceinline__ void fetch_first(Fetch &even, Fetch &odd)
    {
        fetch(even);
        if constexpr (DEEP) fetch(odd);
        deposit(0, even, rows_in(0));
        fetch(even);
    }
    // in chunk's turn: `next`, the rows of the chunk after it (none after the last), into LDS, and the next ones not yet requested
    template <int PARITY> __device__ __forceinline__ void supply(int chunk, Fetch &next)
    {
        deposit(SETS == 2 ? PARITY ^ 1 : 0, next, rows_in(chunk + 1));
        fetch(next);
    }
    template <int PARITY> __device__ __forceinline__ void fetch_turn(int chunk, Fetch &next)
    {
        if constexpr (SETS == 1) __syncthreads();
        supply<PARITY>(chunk, next);
        __syncthreads();
    }
    __device__ __forceinline__ void fetch_walk(int t)
    {
        if (rows <= 0) return;
        __builtin_amdgcn_s_setprio(2);          // the turn's longest way is theirs (7B training step: 181 -> 173, 479 -> 469 us)
        fetch_setup(t);
        const int chunks = (rows + CHUNK - 1) / CHUNK;
        Fetch even, second, &odd = DEEP ? second : even;
        fetch_first(even, odd);
        __syncthreads();
        // (in pairs, an odd chunk after the loop: were a turn skipped on one way through it, the waits would have to suit both ways)
        for (int chunk = 0; chunk + 1 < chunks; chunk += 2) {
            fetch_turn<0>(chunk, odd);
            fetch_turn<1>(chunk + 1, even);
        }
        if (chunks & 1) fetch_turn<0>(chunks - 1, odd);
    }

    // ---- the state waves: the state from chunk to chunk
    float first_hi, first_lo, chunk_hi, chunk_lo, last_hi, last_lo;     // f^rows of the first, a full and the last chunk
    int m0, c0;                 // tile (mt, nw): rows m0 + 16 mt + 4 g4 .. + 3, the slice's column c0 + 16 nw + l16
    f32x4 S[NW][MT];

    __device__ __forceinline__ void state_setup(int t)
    {
        const int early = lead == 0 ? 1 : 0, last_rows = rows > 0 ? (rows - 1) % CHUNK + 1 : 0;
        power(decay, CHUNK - early, first_hi, first_lo);
        power(decay, CHUNK, chunk_hi, chunk_lo);
        power(decay, last_rows - (rows <= CHUNK ? early : 0), last_hi, last_lo);
        const int q = t / 64;
        m0 = DA == 64 ? (q >> 1) * 32 : q * (DA / 4);
        c0 = DA == 64 ? (q & 1) * 16 : 0;
        const float *first = nullptr;
        int64_t fi = wk.si, fj = wk.sj;
        float mul = 1.f;
        if (OUT && args.segments > 1) {     // (the segments' states are joined: each begins from its own)
            first = args.seg + args.seg_walk[job] + ((int64_t)(b * args.H + h) * args.segments + seg) * da * dc;
            fi = dc; fj = 1;
        } else if (OUT && wk.first) {
            first = wk.first + state_at;
            mul = wk.first_mul;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nw = 0; nw < NW; ++nw)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int m = m0 + 16 * mt + 4 * g4 + i, n = n0 + c0 + 16 * nw + l16;
                    S[nw][mt][i] = first && m < da && n < dc ? first[m * fi + n * fj] * mul : 0.f;
                }
    }
    // the state's rounded copy, columns as rows
    __device__ __forceinline__ void publish(int set) const
    {
        if constexpr (OUT) {
#pragma unroll
            for (int nw = 0; nw < NW; ++nw) {
                float by[MT / 2];
                if constexpr (F16) {
#pragma unroll
                    for (int kb = 0; kb < MT / 2; ++kb) {
                        float top = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(S[nw][2 * kb + i / 4][i & 3]));
                        top = fmaxf(top, __shfl_xor(top, 16));
                        const Range r = range(fmaxf(top, __shfl_xor(top, 32)));
                        by[kb] = r.down;
                        if (g4 == 0) range_of(set, m0 / KF + kb)[c0 + 16 * nw + l16] = (uint8_t)(__float_as_uint(r.up) >> 23);
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    constexpr int LANES = V / 4;            // lane groups that share a piece
                    T *to = lds.s[set] + wide_at<T, DA>(spread(c0 + 16 * nw + l16), (m0 + 16 * mt) / V + g4 / LANES) + g4 % LANES * 4;
                    f32x4 v = S[nw][mt];
                    if constexpr (F16) v *= by[mt / 2];
                    if constexpr (sizeof(T) == 2) *(u32x2 *)to = u32x2{M::pack(v[0], v[1]), M::pack(v[2], v[3])};
                    else *(f32x4 *)to = v;
                }
            }
        }
    }
    // fragments of b and of the weighted c, rows as the inner dimension
    __device__ __forceinline__ u32x4 inner_b(int set, int p, int mt) const
    {
        if constexpr (sizeof(T) == 2) {
            const int at = wide_at<T, DA>(update_row<T>(g4, l16 >> 2), (m0 + 16 * mt) / V + (l16 >> 1 & 1)) + (l16 & 1) * 4;
            return load_inner(lds.b[set] + p * KF * DA + at, 16 * DA);
        } else {
            int at[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) at[i] = wide_at<T, DA>(update_row<T>(g4, i), (m0 + 16 * mt + l16) / V) + l16 % V;
            return load_inner(lds.b[set] + p * KF * DA, at);
        }
    }
    __device__ __forceinline__ u32x4 inner_w(int set, int part, int p, int nw) const
    {
        if constexpr (sizeof(T) == 2) {
            const int at = slice_at<T, W_BIT>(update_row<T>(g4, l16 >> 2), c0 + 16 * nw + 4 * (l16 & 3));
            return load_inner(lds.w[set][part] + p * KF * CS + at, 16 * CS);
        } else {
            const int at[4] = {4 * g4 * CS, (4 * g4 + 1) * CS, (4 * g4 + 2) * CS, (4 * g4 + 3) * CS};
            return load_inner(lds.w[set][part] + p * KF * CS + c0 + 16 * nw + l16, at);
        }
    }
    __device__ __forceinline__ u32x4 inner_c(int set, int p, int nt) const
    {
        if constexpr (sizeof(T) == 2) {
            const int at = slice_at<T, C_BIT>(score_row(g4, l16 >> 2), 16 * nt + 4 * (l16 & 3));
            return load_inner(lds.c[set] + p * KF * CS + at, 16 * CS);
        } else {
            const int at[4] = {4 * g4 * CS, (4 * g4 + 1) * CS, (4 * g4 + 2) * CS, (4 * g4 + 3) * CS};
            return load_inner(lds.c[set] + p * KF * CS + 16 * nt + l16, at);
        }
    }
    // S = f^rows S + (weighted c)^T b of the chunk in `set`.  Where registers allow it (DEEP) its fragments are requested before
    // anything else of the turn; otherwise one inner block at a time.
    struct Frags { u32x4 x[KG][MT], y[PARTS][KG][NW]; };
    __device__ __forceinline__ void gather(Frags &f, int set) const
    {
        if constexpr (DEEP) {
#pragma unroll
            for (int p = 0; p < KG; ++p) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) f.x[p][mt] = inner_b(set, p, mt);
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
#pragma unroll
                    for (int nw = 0; nw < NW; ++nw) f.y[part][p][nw] = inner_w(set, part, p, nw);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // to[mt] += (weighted c's part)^T b, columns nw
    __device__ __forceinline__ void update(const Frags &f, int set, int part, int nw, f32x4 (&to)[MT]) const
    {
#pragma unroll
        for (int p = 0; p < KG; ++p) {
            const u32x4 y = DEEP ? f.y[part][p][nw] : inner_w(set, part, p, nw);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) to[mt] = M::mul(DEEP ? f.x[p][mt] : inner_b(set, p, mt), y, to[mt]);
            if constexpr (!DEEP) __builtin_amdgcn_sched_barrier(0);
        }
    }
    __device__ __forceinline__ void move_on(const Frags &f, int set, float hi, float lo)
    {
#pragma unroll
        for (int nw = 0; nw < NW; ++nw)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[nw][mt][i] = fmaf(S[nw][mt][i], hi, S[nw][mt][i] * lo);
#pragma unroll
        for (int nw = 0; nw < NW; ++nw) {
            if constexpr (F16) {
                // parts after the first are stored 2^11, 2^22 times larger and added up on their own, the smallest first
                f32x4 R[MT];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) R[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int part = PARTS - 1; part > 0; --part) {
                    update(f, set, part, nw, R);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) R[mt] *= 0x1p-11f;
                }
                update(f, set, 0, nw, R);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) S[nw][mt] += R[mt];
            } else {
#pragma unroll
                for (int part = 0; part < PARTS; ++part) update(f, set, part, nw, S[nw]);
            }
        }
    }
    __device__ __forceinline__ void store_last() const
    {
        float *last = nullptr;
        int64_t li = wk.si, lj = wk.sj;
        float mul = 1.f;
        if (!OUT) {
            last = args.seg + args.seg_walk[job] + ((int64_t)(b * args.H + h) * args.segments + seg) * da * dc;
            li = dc; lj = 1;
        } else if (args.segments == 1 && wk.last) {
            last = wk.last + state_at;
            mul = wk.last_mul * (wk.last_decays && length > 0 ? exp2f(l2) : 1.f);
        }
        if (!last) return;
        int place = m0 + 4 * g4, column = n0 + c0 + l16;
        asm("" : "+v"(place), "+v"(column));    // (or what state_setup computed of them is kept in registers all the way)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nw = 0; nw < NW; ++nw)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int m = place + 16 * mt + i, n = column + 16 * nw;
                    if (m < da && n < dc) last[m * li + n * lj] = S[nw][mt][i] * mul;
                }
    }
    template <int PARITY> __device__ __forceinline__ void state_turn(int chunk, int chunks, Fetch &next)
    {
        constexpr int SET = SETS == 2 ? PARITY : 0, OTHER = SETS == 2 ? PARITY ^ 1 : 0;
        Frags f;
        gather(f, SET);
        if constexpr (JOINT && SETS == 2) supply<PARITY>(chunk, next);
        const bool last = chunk + 1 == chunks;
        move_on(f, SET, last ? last_hi : chunk == 0 ? first_hi : chunk_hi, last ? last_lo : chunk == 0 ? first_lo : chunk_lo);
        if constexpr (SETS == 1) {
            __syncthreads();
            if constexpr (JOINT) supply<PARITY>(chunk, next);
        }
        publish(OTHER);
        __syncthreads();
    }
    __device__ __forceinline__ void state_walk(int t)
    {
        if constexpr (JOINT) fetch_setup(t);
        state_setup(t);
        if (rows > 0) {
            const int chunks = (rows + CHUNK - 1) / CHUNK;
            Fetch next;
            if constexpr (JOINT) fetch_first(next, next);
            publish(0);
            __syncthreads();
            for (int chunk = 0; chunk + 1 < chunks; chunk += 2) {
                state_turn<0>(chunk, chunks, next);
                state_turn<1>(chunk + 1, chunks, next);
            }
            if (chunks & 1) state_turn<0>(chunks - 1, chunks, next);
        }
        store_last();
    }

    // ---- the output waves: rows 16 W .. 16 W + 15 of every chunk
    struct RowsA { u32x4 k[KB]; };
    float row_mul, step_mul;
    float f[4][4];              // f^(t-s) of this wave's rows (lane % 16) and of the rows of each score tile
    uint32_t oa[FULL ? 1 : KB], oo;

    Stream sa, so;
    float out_mul;

    __device__ __forceinline__ void fetch_a(RowsA &a)
    {
        const Chunk c = sa.next();
#pragma unroll
        for (int k = 0; k < KB; ++k)
            a.k[k] = load(c, FULL ? oa[0] + (uint32_t)(k * KF * sizeof(T)) : oa[FULL ? 0 : k]);
        __builtin_amdgcn_sched_barrier(0);
    }
    // The last inner block's product again, where its result holds infinities or NaN.  The block's rows of c that the causal mask hides
    // from a row are times a score of zero there, which is NaN for such an element.  So each of those counts as zero and a second
    // product tells which results see one: only these keep theirs.  (The check before it: 1 % of the forward of 2 x 8192 rows of 32
    // heads of 128, bf16 165 -> 167 us.)
    template <int W> __device__ __forceinline__ void hide(int set, const u32x4 &x, const f32x4 (&before)[2], f32x4 (&near)[2]) const
    {
        constexpr uint32_t TOP = sizeof(T) == 4 ? 0x7f800000u : F16 ? 0x7c00u : 0x7f80u, ONE_ = sizeof(T) == 4 ? 0x3f800000u : F16 ? 0x3c00u : 0x3f80u;
        const auto bit = [](uint32_t w, int j) { return (w >> 16 * j & TOP) == TOP; };
        int row = l16;
        uint32_t all = ONE_ | (sizeof(T) == 2 ? ONE_ << 16 : 0);
        asm volatile("" : "+v"(row), "+v"(all));        // (or the masks are made before the walk and kept in registers all the way)
        u32x4 seen;             // 1 where the score's row is at or before the result's
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) {
                seen[j] = row >= score_row(g4, j) ? ONE_ : 0;
            } else {
                const int i = 2 * (j & 1);
                const uint32_t own = (row >= score_row(g4, i) ? ONE_ : 0) | (row >= score_row(g4, i + 1) ? ONE_ << 16 : 0);
                seen[j] = W & 1 ? j < 2 ? all : own : j < 2 ? own : 0;
            }
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            const u32x4 xc = inner_c(set, sizeof(T) == 2 ? W / 2 : W, nt);
            u32x4 finite, rest;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = xc[j];
                if constexpr (sizeof(T) == 4) {
                    finite[j] = bit(w, 0) ? 0 : w;
                    rest[j] = bit(w, 0) ? ONE_ : 0;
                } else {
                    finite[j] = (bit(w, 0) ? 0 : w & 0xffffu) | (bit(w, 1) ? 0 : w & 0xffff0000u);
                    rest[j] = (bit(w, 0) ? ONE_ : 0) | (bit(w, 1) ? ONE_ << 16 : 0);
                }
            }
            const f32x4 without = M::mul(finite, x, before[nt]), count = M::mul(rest, seen, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i) near[nt][i] = count[i] > 0.f ? near[nt][i] : without[i];
        }
    }
    template <int W, int PARITY> __device__ __forceinline__ void out_turn(int chunk, RowsA &a)
    {
        constexpr int SET = SETS == 2 ? PARITY : 0;
        const T *const tb = lds.b[SET], *const ts = lds.s[SET];
        // Scores, transposed (rows 16 st + .. of b by this wave's rows of a), and what comes from before the chunk, transposed (the
        // state's columns 8 g4 .. + 7 by this wave's rows).  All of a block's fragments are requested before the first product: left
        // to itself the compiler keeps one or two reads ahead, and a wave then waits for LDS at every product.
        f32x4 P[W + 1], O[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int st = 0; st <= W; ++st) P[st] = f32x4{0.f, 0.f, 0.f, 0.f};
        constexpr int BLOCK = 2;
#pragma unroll
        for (int kb = 0; kb < KB; kb += BLOCK) {
            u32x4 xb[BLOCK][W + 1], xs[BLOCK][2];
#pragma unroll
            for (int k = 0; k < BLOCK; ++k) {
                const int at_k = wide_at<T, DA>(l16, 4 * (kb + k) + g4);
#pragma unroll
                for (int st = 0; st <= W; ++st) xb[k][st] = *(const u32x4 *)(tb + 16 * st * DA + at_k);
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) xs[k][nt] = *(const u32x4 *)(ts + 16 * nt * DA + at_k);
            }
            if constexpr (DEEP) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < BLOCK; ++k) {
                u32x2 up = {0, 0};
                if constexpr (F16) up = *(const u32x2 *)(range_of(SET, kb + k) + 8 * g4);
#pragma unroll
                for (int st = 0; st <= W; ++st) P[st] = M::mul(xb[k][st], a.k[kb + k], P[st]);
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    if constexpr (F16) O[nt] += M::mul(xs[k][nt], a.k[kb + k], f32x4{0.f, 0.f, 0.f, 0.f}) * ranges(up[nt]);
                    else O[nt] = M::mul(xs[k][nt], a.k[kb + k], O[nt]);
                }
            }
        }
        constexpr int GROUPS = sizeof(T) == 2 ? W / 2 + 1 : W + 1;
        u32x4 xc[GROUPS][2];
#pragma unroll
        for (int p = 0; p < GROUPS; ++p)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) xc[p][nt] = inner_c(SET, p, nt);
        if constexpr (DEEP) __builtin_amdgcn_sched_barrier(0);
        fetch_a(a);
        const float mul = row_mul * (chunk == 0 && lead == 0 ? 1.f : step_mul);
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) O[nt] *= mul;
#pragma unroll
        for (int st = 0; st < W; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) P[st][i] *= f[st][i];
#pragma unroll
        for (int i = 0; i < 4; ++i) P[W][i] = l16 >= score_row(g4, i) ? P[W][i] * f[W][i] : 0.f;
        // (f16: the scores of a row, like the state's copy, by a power of two that brings the largest to about 1)
        f32x4 near[2] = {O[0], O[1]};
        float up = 1.f;
        if constexpr (F16) {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 4 * (W + 1); ++i) top = fmaxf(top, fabsf(P[i >> 2][i & 3]));
            top = fmaxf(top, __shfl_xor(top, 16));
            const Range r = range(fmaxf(top, __shfl_xor(top, 32)));
            up = r.up;
#pragma unroll
            for (int st = 0; st <= W; ++st) P[st] *= r.down;
            near[0] = near[1] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        u32x4 x;
        f32x4 before[2];
#pragma unroll
        for (int p = 0; p < GROUPS; ++p) {
            if constexpr (sizeof(T) == 2) {
                x[0] = M::pack(P[2 * p][0], P[2 * p][1]);
                x[1] = M::pack(P[2 * p][2], P[2 * p][3]);
                x[2] = 2 * p + 1 <= W ? M::pack(P[2 * p + 1 <= W ? 2 * p + 1 : 0][0], P[2 * p + 1 <= W ? 2 * p + 1 : 0][1]) : 0;
                x[3] = 2 * p + 1 <= W ? M::pack(P[2 * p + 1 <= W ? 2 * p + 1 : 0][2], P[2 * p + 1 <= W ? 2 * p + 1 : 0][3]) : 0;
            } else {
                x = __builtin_bit_cast(u32x4, P[p]);
            }
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                before[nt] = near[nt];
                near[nt] = M::mul(xc[p][nt], x, near[nt]);
            }
        }
        float odd = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) odd = fmaf(near[i >> 2][i & 3], 0.f, odd);
        if (__builtin_expect(__ballot(odd != 0.f) != 0, 0)) hide<W>(SET, x, before, near);
        const Chunk to_rows = so.next();
        const uint32_t off = oo + to_rows.shift;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (F16 ? fmaf(near[i >> 2][i & 3], up, O[i >> 2][i & 3]) : near[i >> 2][i & 3]) * out_mul;
        if constexpr (sizeof(T) == 2) {
            win_store_aux<0>(to_rows.win, off, u32x4{M::pack(v[0], v[1]), M::pack(v[2], v[3]), M::pack(v[4], v[5]), M::pack(v[6], v[7])});
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                win_store_aux<0>(to_rows.win, FULL || n0 + 8 * g4 + 4 * j < dc ? off + 16 * j : NOWHERE,
                                 u32x4{__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3])});
        }
    }
    __device__ __forceinline__ void between() const
    {
        if constexpr (SETS == 1) __syncthreads();
        __syncthreads();
    }
    template <int W> __device__ __forceinline__ void out_walk()
    {
#pragma unroll
        for (int k = 0; k < (FULL ? 1 : KB); ++k) oa[k] = offset(wk.a, 16 * W + l16, k * KF + g4 * V, da);
        oo = offset(wk.out, 16 * W + l16, n0 + 8 * g4, dc);
        row_mul = exp2f(l2 * (16 * W + l16));
        step_mul = exp2f(l2);
#pragma unroll
        for (int st = 0; st <= W; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) f[st][i] = exp2f(l2 * (16 * (W - st) + l16 - score_row(g4, i)));
        if (rows <= 0) return;
        sa = stream(wk.a, da);
        so = stream(wk.out, dc);
        out_mul = wk.out_mul;
        const int chunks = (rows + CHUNK - 1) / CHUNK;
        RowsA even, second, &odd = DEEP ? second : even;
        // A store that is dropped after each request, as one follows each in the loop: the waits of the first turn, which are the
        // loop's too, then count alike.
        const Chunk none = {make_window(nullptr, 0), 0};
        fetch_a(even);
        win_store_aux<0>(none.win, NOWHERE, u32x4{0, 0, 0, 0});
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (DEEP) {
            fetch_a(odd);
            win_store_aux<0>(none.win, NOWHERE, u32x4{0, 0, 0, 0});
        }
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        for (int chunk = 0; chunk + 1 < chunks; chunk += 2) {
            out_turn<W, 0>(chunk, even);
            between();
            out_turn<W, 1>(chunk + 1, odd);
            between();
        }
        if (chunks & 1) {
            out_turn<W, 0>(chunks - 1, even);
            between();
        }
    }
    // rows of the segment's time span past the sequence's end
    __device__ __forceinline__ void clear_rest(int t, int threads) const
    {
        const int end = from + args.seg_rows < args.L ? from + args.seg_rows : args.L;
        T *const po = (T *)wk.out.p + b * wk.out.sb + h * wk.out.sh;
        for (int r = (from > length ? from : length) + (t >> 5); r < end; r += threads / 32)
            if (n0 + (t & 31) < dc) Elem<T>::store(po + r * wk.out.st + n0 + (t & 31), 0.f);
    }
};

// Waves 0 - 3 make the output, waves 4 - 7 move the state on, waves 8 - 11 fetch rows: a chunk's parts depend on each other only
// from chunk to chunk, so they run side by side, three waves a SIMD.  Without an output the state's waves come first.
template <typename T, int DA, bool OUT, int PARTS, bool FULL>
__global__ __launch_bounds__((Walker<T, DA, OUT, PARTS, FULL>::WAVES * 64)) void walk_kernel(Walks args, int slices)
{
    typedef Walker<T, DA, OUT, PARTS, FULL> W;
    __shared__ typename W::Lds lds;
    int64_t group;
    int slice;
    place(blockIdx.x, slices, group, slice);
    if (group >= args.groups) return;
    const int seg = (int)(group % args.segments);
    group /= args.segments;
    const int h = (int)(group % args.H);
    group /= args.H;
    const int b = (int)(group % args.bs), job = (int)(group / args.bs);
    W w(args, args.w[job], lds);
    w.b = b; w.h = h; w.seg = seg; w.job = job;
    w.da = w.wk.da; w.dc = w.wk.dc; w.n0 = slice * COLS;
    if (w.n0 >= w.dc) return;
    w.tid = threadIdx.x;
    w.lane = w.tid & 63; w.l16 = w.lane & 15; w.g4 = w.lane >> 4;
    w.wave = __builtin_amdgcn_readfirstlane(w.tid >> 6);
    int length = args.L;
    if (args.lengths) {
        length = __builtin_amdgcn_readfirstlane(args.lengths[b]);
        length = length < 0 ? 0 : length > args.L ? args.L : length;
    }
    w.length = length;
    w.from = seg * args.seg_rows;
    w.rows = length - w.from < args.seg_rows ? length - w.from : args.seg_rows;
    w.decay = clamp_decay(args.log_decay[h]);
    w.l2 = w.decay * 1.44269504f;
    w.state_at = (int64_t)(b * args.H + h) * w.da * w.dc;
    w.lead = OUT && seg == 0 && w.wk.first ? w.wk.lead : 1;
    if constexpr (OUT) {
        switch (w.wave) {
        case 0: w.template out_walk<0>(); break;
        case 1: w.template out_walk<1>(); break;
        case 2: w.template out_walk<2>(); break;
        case 3: w.template out_walk<3>(); break;
        case 4: case 5: case 6: case 7: w.state_walk(w.tid - 256); break;
        default:
            if constexpr (!W::JOINT) w.fetch_walk(w.tid - 512);
        }
        w.clear_rest(w.tid, W::WAVES * 64);
    } else if (w.wave < 4) {
        w.state_walk(w.tid);
    } else {
        w.fetch_walk(w.tid - 256);
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
    int length = args.L;
    if (args.lengths) {
        length = args.lengths[bh / args.H];
        length = length < 0 ? 0 : length > args.L ? args.L : length;
    }
    const float decay = clamp_decay(args.log_decay[bh % args.H]);
    float whole_hi, whole_lo;
    power(decay, args.seg_rows, whole_hi, whole_lo);
    const int64_t at = bh * size + (e / wk.dc) * wk.si + (e % wk.dc) * wk.sj;
    float s = wk.first ? wk.first[at] * wk.first_mul : 0.f;
    float *p = args.seg + args.seg_walk[job] + bh * args.segments * size + e;
    for (int i = 0; i < args.segments; ++i, p += size) {
        const int left = length - i * args.seg_rows, rows = left < 0 ? 0 : left < args.seg_rows ? left : args.seg_rows;
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
// multiplied with q on the way; the threads of a column add up through LDS.  ALIGNED: dv is a multiple of 4.  Bound by the state's
// bytes: 128 sequences of 64 heads of 128 x 128 in 207 us, 5.2 TB/s; one sequence of 32 heads in 5.4 us, hardly more than a launch.
template <typename T, bool ALIGNED> __global__ __launch_bounds__(THREADS) void step_kernel(Step a)
{
    __shared__ float lq[GCG_LINEAR_MAX_DIM], lk[GCG_LINEAR_MAX_DIM], f[2];
    __shared__ __align__(16) float part[4 * THREADS];           // [thread of a column][column]
    const int slices = (a.dv + a.cols - 1) / a.cols;
    const int64_t bh = blockIdx.x / slices;
    const int slice = blockIdx.x % slices, h = (int)(bh % a.H), tid = threadIdx.x;
    const int64_t b = bh / a.H;
    const T *q = (const T *)a.q + b * a.qb + h * a.qh, *k = (const T *)a.k + b * a.kb + h * a.kh, *v = (const T *)a.v + b * a.vb + h * a.vh;
    const int quads = a.cols / 4, R = THREADS / quads, col = slice * a.cols + tid % quads * 4, row0 = tid / quads;
    float vv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vv[i] = col + i < a.dv ? Elem<T>::load(v + col + i) : 0.f;
    for (int i = tid; i < a.dk; i += THREADS) {
        lq[i] = Elem<T>::load(q + i);
        lk[i] = Elem<T>::load(k + i);
    }
    // (as a sum of two floats, as in the walk: one float's rounding, the same for every token, would show after thousands of them)
    if (tid < kWave) {
        float hi, lo;
        power(clamp_decay(a.log_decay[h]), 1, hi, lo);
        if (tid == 0) { f[0] = hi; f[1] = lo; }
    }
    float *const s = a.state + bh * a.dk * a.dv + col;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    __syncthreads();
    const float hi = f[0], lo = f[1];
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
                        x[u][i] = fmaf(x[u][i], hi, fmaf(x[u][i], lo, lk[r] * vv[i]));
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
    const dim3 grid((unsigned)blocks), block(Walker<T, DA, OUT, PARTS, true>::WAVES * 64);
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

int64_t seg_rows_of(int64_t L, int segments) { return ((L + segments - 1) / segments + CHUNK - 1) / CHUNK * CHUNK; }

// Segments of a walk.  A CU takes one workgroup of a walk with an output at a time, so a launch costs (rounds of 256 workgroups) *
// (chunks of a segment), half as much again where the segments' states are made first (two of whose workgroups would fit a CU, which
// this count leaves out), and two more launches and the join, about 10 chunks.  Segments, four chunks at least, are taken where that is
// 3 % below 3/4 of the walk in one piece, and a larger number of them wherever it gains 3 % on the last one taken.
// Measured in us (bf16, 1 sequence, heads of 128): 8 heads of 131072 rows, forward, 1 segment 1961, 8 538, 16 525; backward, 1
// segment 1890, 3 1841, 6 1429, 8 1289; 16 heads of 8192 rows, forward, 1 segment 103, 4 60, 8 71; backward, 1 segment 115, 2
// 171; 8 heads of 1024 rows, forward, 1 segment 19, 2 26.
int segments_of(int64_t walks, int64_t bs, int64_t L, int H, int dc)
{
    const int64_t units = walks * bs * H * ((dc + COLS - 1) / COLS), chunks = (L + CHUNK - 1) / CHUNK;
    const auto rounds = [&](int64_t n) { return (units * n + 255) / 256; };
    int64_t best = rounds(1) * chunks * 3 / 2;
    int segments = 1;
    for (int64_t n = 2; n <= chunks / 4 && units * n <= 768; ++n) {
        const int64_t cost = rounds(n) * (seg_rows_of(L, (int)n) / CHUNK) * 3 + 20;
        if (cost * 100 < best * 97) {
            best = cost;
            segments = (int)n;
        }
    }
    return segments;
}

void plan(Walks &w, int64_t L, int dc)
{
    w.segments = segments_of(w.n, w.bs, L, w.H, dc);
    w.seg_rows = (int32_t)seg_rows_of(L, w.segments);
    w.segments = (int)((L + w.seg_rows - 1) / w.seg_rows);
    w.L = (int32_t)L;
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
