// Which of the kernels of gcg_product8.hip makes a product of 8-bit tensors, and in what parts.  On the host, from the sizes alone.
#pragma once
#include <cstdint>
#include <cstdlib>

namespace gcg {

constexpr int kTokenBlocks = 32;    // of a wave of product8_tokens_kernel, at most

// Which kernel, and in how many parts of the blocks (each a sum in fp32, joined by another kernel): what would take the least time.
// Up to 64 rows go by product8_tokens_kernel (from 12288 x 4096 with 1, 16, 64 rows 11.8, 12.7, 15.7 us, tiles of 128 in parts 14.5, 18.5, 23.2;
// 2560 x 2560 4.2, 4.4, 5.7 and 11.4 to 12.6; 4096 x 16384 15, 15, 27 and 22 to 27), and more in groups of 64 where that takes least time (256 rows
// from 4096 x 4096 10, by tiles of 128 in parts 21; 512 rows 18 and 30; 1000 x 1000 x 1000 5.7 and 9.5; 400 rows from 12288 x 4096 53, tiles of 256 x 128
// 46).  Else, in microseconds as measured: a round of 256 tiles of 256 x 256 takes 1.35 a block and 6 around them, of 256 x 128 0.85 and 5 (0.9 if half
// the card is idle), 3 and 2 once; 512 tiles of 128 x 128, two a CU, take 1.22 a block, 256 of them 0.9, and their results, in four columns at a time or
// one by one, leave at 4.2 or 1.3 TB/s (8000 x 8000 x 256 56 us, 8000 x 8001 x 256 118; tiles of 256 x 256 43 and 44); joining moves four bytes for every part of a result twice
// at 4 TB/s, and 3 for its launch.  So (tiles of 128 x 128, 256 x 128, 256 x 256) 4096 x 4096 x 4096 goes by the last (88, 63, 55), 2048 x 4096 x 4096
// by the second (48, 34, 46), 7680 x 2561 x 5003 by either of them (147, 116, 115) and 701 x 7683 x 2560 by the second (35, 23, 34).
// Where the last round of 256 x 256 tiles would leave the card half empty, the rows of the rounds before it go by those, the rest by
// 256 x 128: 7683 x 2561 x 5003 by either alone 116 and 114 us, 105 so; 5040 x 7680 x 2560 97 and 101, 91 so.
enum { TOKENS, TILE, TALL, WIDE };       // tiles of 128 x 128, 256 x 128, 256 x 256
struct Plan8 { int kernel, splits, split_steps; int64_t rest; };        // rest (WIDE): rows at the end that go by TALL
inline float estimate(int kernel, int64_t M, int64_t N, int per, int splits)
{
    const int bm = kernel == TILE ? 128 : 256, bn = kernel == WIDE ? 256 : 128;
    const int64_t items = ((M + bm - 1) / bm) * ((N + bn - 1) / bn) * splits;
    const float join = splits > 1 ? 3.f + (float)M * (float)N * (float)splits * 8.f / 4e6f : 0.f;
    if (kernel == WIDE) return (float)((items + 255) / 256) * ((float)per * 1.35f + 6.f) + 3.f + join;
    if (kernel == TALL) return (float)((items + 255) / 256) * ((float)per * (items <= 128 ? 0.9f : 0.85f) + 5.f) + 2.f + join;
    const float leave = (float)M * (float)N / (N % 4 == 0 || splits > 1 ? 2.1e6f : 0.65e6f);
    return (items <= 256 ? (float)per * 0.9f : (float)((items + 511) / 512) * (float)per * 1.22f) + 6.f + leave + join;
}
// Groups of 64 rows by product8_tokens_kernel: the rows of b for a workgroup (in sixteens) that take least time, and that time; as measured, a round
// of 256 workgroups takes 1.9 us and 0.55, 0.85, 0.95 for each block of a wave, the first one as long as b takes to arrive at 4.3 TB/s at least.
struct TokensTime { int tiles; float time; };
inline TokensTime tokens_estimate(int64_t M, int64_t N, int steps)
{
    TokensTime best = {0, 0.f};
    const float arrive = 1.8f + (float)N * (float)steps * (128.f / 4.3e6f);
    for (int tiles = 1; tiles <= 4; tiles *= 2) {
        const int64_t items = ((M + 63) / 64) * ((N + tiles * 16 - 1) / (tiles * 16));
        const float round = 1.9f + (float)((steps + 3) / 4) * (tiles == 1 ? 0.55f : tiles == 2 ? 0.85f : 0.95f);
        const float time = 0.8f + (round > arrive ? round : arrive) + (float)((items - 1) / 256) * round;
        if (best.tiles == 0 || time < best.time) best = {tiles, time};
    }
    return best;
}
// whether product8_tokens_kernel takes it: its waves have kTokenBlocks each at most
inline bool tokens(int64_t M, int steps) { return M <= 32 ? steps <= 8 * kTokenBlocks : M <= 64 && steps <= 4 * kTokenBlocks; }
inline bool takes(int kernel, int64_t M, int64_t N) { return kernel == TILE || (M >= 256 && N >= (kernel == WIDE ? 256 : 128)); }
// Whether a plan is one that the launch takes: past it the wide tiles would start before the tensor, and the tokens' kernel leave results out.
inline bool holds(const Plan8 &p, int64_t M, int64_t N, int steps)
{
    if (p.splits < 1 || (int64_t)p.splits * p.split_steps < steps || (int64_t)(p.splits - 1) * p.split_steps >= steps) return false;
    if (p.splits > 1 && (p.split_steps % 4 || p.kernel == TOKENS)) return false;
    if (p.rest && (p.kernel != WIDE || p.splits > 1 || p.rest < 256)) return false;
    switch (p.kernel) {
    case TOKENS: return M <= 32 ? tokens(M, steps) : steps <= 4 * kTokenBlocks;
    case TILE: case TALL: case WIDE: return takes(p.kernel, M - p.rest, N);
    default: return false;
    }
}
// kernel_env, parts_env: what a tuning build is told to take instead, where that holds; null otherwise
inline Plan8 plan8(int64_t M, int64_t N, int steps, const char *kernel_env, const char *parts_env)
{
    if (kernel_env) {
        const int kernel = atoi(kernel_env), told = parts_env ? atoi(parts_env) : 1, n = told < 1 || kernel == TOKENS ? 1 : told;
        const int per = kernel == TOKENS ? steps : ((steps + n - 1) / n + 3) / 4 * 4;
        const Plan8 p = {kernel, (steps + per - 1) / per, per, 0};
        return holds(p, M, N, steps) ? p : Plan8{TILE, 1, (steps + 3) / 4 * 4, 0};
    }
    if (tokens(M, steps)) return {TOKENS, 1, steps, 0};
    Plan8 best = {TILE, 1, (steps + 3) / 4 * 4, 0};
    float least = 0.f;
    for (int kernel = TILE; kernel <= WIDE; ++kernel)
        for (int n = 1; takes(kernel, M, N) && (n == 1 || (n <= 32 && steps >= 4 * n)); n *= 2) {
            const int per = ((steps + n - 1) / n + 3) / 4 * 4, splits = (steps + per - 1) / per;
            const float time = estimate(kernel, M, N, splits > 1 ? per : steps, splits);
            if (least == 0.f || time < least) {
                least = time;
                best = {kernel, splits, per, 0};
            }
        }
    if (steps <= 4 * kTokenBlocks && tokens_estimate(M, N, steps).time < least) return {TOKENS, 1, steps, 0};
    if (best.kernel == TILE || best.splits > 1 || !takes(WIDE, M, N)) return best;
    const int64_t across = (N + 255) / 256, items = (M + 255) / 256 * across;
    for (int64_t rounds = 1; rounds * 256 < items; ++rounds) {
        const int64_t rows = rounds * 256 / across * 256;
        if (rows == 0 || M - rows < 256) continue;
        const float time = estimate(WIDE, rows, N, steps, 1) + estimate(TALL, M - rows, N, steps, 1) + 2.f;
        if (time < least) {
            least = time;
            best = {WIDE, 1, best.split_steps, M - rows};
        }
    }
    return best;
}

} // namespace gcg
