// Plans of the products: which kernel, tiles, splits of K, parts of a product, workspaces, and where an operand's tile ends. Plain
// host C++ without HIP: the library's calls and the CPU tests run the same arithmetic.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace bmx {

constexpr int GK = 64;      // K of a tile (gemm16_k)
constexpr int SK_K = 128;   // columns of a step on 4-bit weights, and of skinny_k
constexpr int SL_K = 512;   // columns of a slice (slice_k)
constexpr int SL_TT = 5;    // slice_k's most tiles of 16 tokens: 80 KB of x
constexpr int QG_T = 128, QG_N = 128;      // tokens and rows of W of a workgroup (gemm_q4_k)

constexpr int64_t round_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// The tiles a product can run on: results M x N, workgroups that run at once, and what was measured of each: us a K tile of
// 64 with a workgroup on every other compute unit or fewer (alone) and with the chip full, us to begin and end.
struct Tile { int M, N, slots; double alone, full, ends; };
constexpr Tile TILES[4] = {
    {256, 256, 256, 1.60, 1.60, 6.0},      // 8 waves, 2 buffers
    {128, 128, 512, 0.64, 1.00, 3.0},      // 4 waves, 2 buffers, two on a compute unit
    {128, 64, 256, 0.34, 0.38, 3.0},       // 2 groups of 4 waves, each every other K tile, 3 buffers
    {128, 128, 256, 0.54, 0.54, 3.0},      // the same, 2 buffers
};
struct TilePlan { int tile, splits; int64_t head; double us; };   // head: rows of M that go first, on 256 x 256 tiles

// Tiles of a product with M x N results, `products` side by side, nk tiles of K: the cheapest by those times. K is split,
// the partial sums joined by a second kernel, where that saves more than the second kernel (5 us) and the sums' bytes
// (written and read at 4 TB/s) cost.
inline TilePlan plan_product(int64_t M, int64_t N, int nk, int products, bool can_split, bool grads = false)
{
    TilePlan best = {0, 1, 0, 1e30};
    if (M <= 0 || N <= 0) return {0, 1, 0, 0.0};                   // no tokens
    for (int t = 0; t < 4; ++t)
        for (int s = 1; s <= 16; ++s)
        {
            if (s > 1 && (!can_split || nk / s < 4)) break;
            const Tile& c = TILES[t];
            const int64_t b = (M + c.M - 1) / c.M * ((N + c.N - 1) / c.N) * products * s, full = b / c.slots, rest = b % c.slots;
            const int each = (nk + s - 1) / s;
            // the gradients' epilogue reads and writes 12 bytes a result: about a fourth more
            double us = full * (each * c.full + c.ends);
            if (rest) us += each * (rest <= 256 ? c.alone : c.full) + c.ends;
            if (grads) us *= 1.25;
            if (s > 1) us += 5.0 + (double)M * N * products * s * 8.0 / 4e6;
            if (us < best.us) best = {t, s, 0, us};
        }
    // Large tiles for as many rows of M as fill whole rounds of the chip, the rest on the tiles that suit it: a last round of
    // a few large tiles would cost as much as a full one (4,096 tokens through 2 x 11,008 rows, 5.4 rounds: 665 us, in two parts 630)
    const int64_t tn = (N + 255) / 256, rounds = (M + 255) / 256 * tn / 256, head = rounds * 256 / tn * 256;
    if (products == 1 && head > 0 && head < M)
    {
        const TilePlan tail = plan_product(M - head, N, nk, 1, false, grads);
        const double us = rounds * (nk * TILES[0].full + TILES[0].ends) * (grads ? 1.25 : 1.0) + tail.us + 2.0;
        if (tail.head == 0 && us < best.us) best = {tail.tile, 1, head, us};
    }
    return best;
}

// The launches of a product with M rows of A (EPI_GU: of each of `mats` = 2 matrices) that is not split: one, or the head on
// 256 x 256 tiles and the rest
struct ProductPart { int tile, from, rows; };

inline int product_parts(const TilePlan& p, int M, int mats, ProductPart (&out)[2])
{
    if (!p.head)
    {
        out[0] = {p.tile, 0, M};
        return 1;
    }
    const int head = (int)(p.head / mats);
    out[0] = {0, 0, head};
    out[1] = {p.tile, head, M - head};
    return 2;
}

// An operand's tile at row r0 (of the result's side) and column k0: bytes from the matrix's first value to the tile's, and from
// there to the matrix's end, past which loads give zeros. Along K: stored [rows][ld], K across: [K][ld]; r0 counts from the
// matrix's first row, also in the second part of a product: from a pointer moved to that part's rows the end of a matrix
// stored [K][ld] would lie as many values too far.
struct OperandSpan { int64_t first, left; };

constexpr OperandSpan operand_span(bool across, int64_t ld, int rows, int K, int r0, int k0)
{
    const int64_t first = across ? (int64_t)k0 * ld + r0 : (int64_t)r0 * ld + k0;
    return {first * 2, ((across ? K : rows) * ld - first) * 2};
}

inline int tiles_k(int K) { return (K + GK - 1) / GK; }

// EPI_GU is one product of twice the rows, but two where K is split
inline TilePlan plan_for(int N, int T, int K, int products) { return plan_product((int64_t)N * products, T, tiles_k(K), 1, true); }

inline double product_us(int N, int T, int K, int products) { return plan_for(N, T, K, products).us; }

inline size_t product_part_bytes(int N, int T, int K, int products)
{
    const TilePlan p = plan_for(N, T, K, products);
    return p.splits > 1 ? (size_t)p.splits * products * T * ((N + 7) / 8 * 8) * 4 : 0;
}

// Tiles of a backward pass's products: dh, dx, down's gradient, gate's and up's
struct BackTiles { TilePlan dh, dx, dd, dw; bool two; };       // two: dh and down's gradient in one launch, when both are wanted

// Whether down's gradient (tiles of `a` steps of K) and dh (of `b`) end sooner in one grid: the former's tiles, one a compute
// unit, start first; dh's take the other units, then all
inline bool two_at_once(int H, int I, int T, const BackTiles& p)
{
    auto over = [](int64_t n, int64_t by) { return (n + by - 1) / by; };
    const int64_t units = TILES[0].slots, it = over(I, 256), na = it * over(H, 256), nb = it * over(T, 256);
    const int64_t a = tiles_k(T), b = tiles_k(H);
    if (p.dh.tile != 0 || p.dh.head || p.dh.splits > 1 || na >= units) return false;
    const int64_t beside = (units - na) * (a / b), left = nb > beside ? nb - beside : 0;
    const int64_t steps = left ? (a > a / b * b ? a : a / b * b) + over(left, units) * b : std::max(a, over(nb, units - na) * b);
    return steps * TILES[0].full + TILES[0].ends * 2 < p.dh.us + p.dd.us;
}

inline BackTiles back_tiles(int H, int I, int T)
{
    BackTiles p;
    p.dh = plan_product(I, T, tiles_k(H), 1, true, true);
    p.dx = plan_product(H, T, 2 * tiles_k(I), 1, true);
    p.dd = plan_product(I, H, tiles_k(T), 1, false);
    p.dw = plan_product(H, I, tiles_k(T), 2, false);
    p.two = two_at_once(H, I, T, p);
    return p;
}

// ---- few tokens, and 4-bit weights --------------------------------------------------------------------------------------

// Which kernel a product of T tokens with an N x K matrix (or two, side by side) runs on: skinny_k, slice_k or one for many tokens
enum ProductPath { FEW_DIRECT, FEW_SLICES, MANY };

// skinny_k: tiles of 16 rows per workgroup (1, 2 or, in 4 bits, 4), and how long it takes. x is read once per workgroup, so more
// tiles save what x costs beside a tile of W (about 0.2 of a 4-bit tile a token, 0.05 of a 16-bit one); but the compute unit
// with the most workgroups is the last to end, so time goes up in whole rounds of the 256 units. Tiles against measurements
// (us with 1 / 2 / 4): 16 tokens, 4-bit 5120 -> 2 x 2304 13.1 / 9.0 / 11.1, 2304 -> 5120 6.7 / 5.0 / 5.9, 4096 -> 14336 17.8 /
// 11.5 / 9.7, 16-bit 2304 -> 5120 9.8 / 8.0 / 12.0, 4096 -> 2 x 2048 10.8 / 13.0; 8 tokens 5120 -> 2304 5.6 / 6.3 / 9.5; 4 tokens
// 4096 -> 11008 9.4 / 11.8. Time, planned and measured: 4-bit 4096 -> 4096 32 / 64 / 80 tokens 7.9 / 10.0 / 17.5, 7.6 / 9.6 / 16.5;
// 4096 -> 14336 48 tokens 25.0, 25.9; 16-bit block of 4096 x 2048 17 / 33 tokens 22 / 37, 22 / 38.
struct DirectPlan { int rt; double us; };

inline DirectPlan direct_plan(int N, int K, int T, int products, bool q4)
{
    const int64_t tiles = (int64_t)(N + 15) / 16 * products, tt = (T + 15) / 16;
    const double x = (T < 16 ? T : 16) * (q4 ? 0.2 : 0.05), us = (K > 1024 ? K / 1024.0 : 1.0) * (q4 ? 0.26 : 1.0);
    DirectPlan best = {1, 1e30};
    for (int rt = 1; rt <= (q4 ? 4 : 2); rt *= 2)
    {
        const double t = 2.5 + (((tiles + rt - 1) / rt * tt + 255) / 256) * (rt + x) * us;
        if (t < best.us) best = {rt, t};
    }
    return best;
}

// The form that runs: tiles of rows, x in LDS (one token on 4-bit weights of up to 8,192 columns, 16 KB)
struct FewForm { int rt; bool xl; };

inline FewForm few_form(int N, int K, int T, int products, int group)
{
    if (group && T == 1 && K <= 8192) return {1, true};
    return {direct_plan(N, K, T, products, group != 0).rt, false};
}

// slice_k and the joining kernel, fp16 and bf16 alike (us, planned and measured in both): 768 x 2048 32 tokens 6.5, 6.0 and 7.5;
// 4096 x 4096 48 tokens 13, 12.5 and 14.8; 14336 x 4096 64 tokens 31, 26 and 28
inline double slices_us(int N, int K, int T, int products)
{
    return 1.08 * (4.3 + 0.05 * T + (double)N * K * products / 1e6 * (0.13 + 0.0039 * T));
}

// 4-bit weights of the products of many tokens: codes multiplied as they are (gemm_q4_k), the weights never rounded, or each
// decoded and rounded to 16 bits first, for gemm16_k's larger tiles. By tokens alone, so that of one matrix a call of more tokens
// never keeps more digits than one of fewer: to 1,024 as they are, with groups of 32, whose scales cost gemm_q4_k the most, to
// 256. us as they are / decoded first (bf16 x): groups of 128, 4096 -> 4096 400 tokens 41 / 37, 1,024 61 / 51, 1,100 67 / 61, 2,048
// 75 / 75, 4,096 155 / 116; 4096 -> 11008 517 71 / 80, 1,024 121 / 110, 4,096 437 / 317; 5120 -> 2304 517 35 / 39, 1,024 48 / 57, 2,048
// 82 / 71; 32, 4096 -> 4096 200 34 / 35, 300 37 / 38, 400 47 / 39, 1,024 72 / 51; 4096 -> 11008 200 72 / 59, 300 85 / 70.
constexpr int q4_whole_most(int group) { return group == 32 ? 256 : 1024; }

inline double q4_many_us(int N, int K, int T, int products, int group, bool keep);

// Up to 16 tokens skinny_k: W once. Beyond, it reads W once more for every 16 tokens (from L2), against slices, which join their
// sums in a second launch, up to SL_TT tiles of tokens, and the tiled products: whichever is planned sooner. Both sides in us:
// 4-bit 768 x 2048 80 tokens 4.5 / 9.0 by slices, 2560 -> 2304 48 tokens 6.4 / 8.8, 4096 -> 11008 80 tokens bf16 30 / 33, 4096 -> 14336
// 64 tokens 32 / 28; 16-bit block of 2048 x 768 33 tokens 12.5 / 15.9 by gemm16_k, 5120 x 2304 44 / 29.
// keep: weights that 16 bits of x's type may not hold are not decoded first.
inline ProductPath product_path(int N, int K, int T, int products, int group, bool keep)
{
    if (T <= 16) return FEW_DIRECT;
    const double us = T <= 1024 ? direct_plan(N, K, T, products, group != 0).us : 1e30;
    if (!group) return us < product_us(N, T, K, products) ? FEW_DIRECT : MANY;
    // The others' two or three launches keep the host of a call outside a graph about 11 us, the one 7. A graph has no such host, but
    // its nodes' own ends: us a call / in a graph, this way and by their times alone, 4-bit 512 -> 2553 226 tokens 7.4 / 7.5, 9.8 / 9.9;
    // 4416 -> 750 30 tokens 7.0 / 7.0, 10.8 / 6.9; 256 -> 4342 149 tokens 7.1 / 6.9, 8.5 / 7.7; 5888 -> 139 23 tokens 7.9 / 7.8, 10.9 / 6.1.
    const double least = 10.0;
    if (T <= SL_TT * 16) return us < std::max(slices_us(N, K, T, products), least) ? FEW_DIRECT : FEW_SLICES;
    // (beyond 80 tokens the plan is a tenth short: 160 tokens 2304 -> 5120 19, 23.5; by gemm_q4_k 20.3). Where the other side
    // rounds the weights, its time is that of the fewest tokens for which it does: one count at which it takes over.
    const int at = keep ? T : std::min(T, q4_whole_most(group) + 1);
    return us * 1.15 < std::max(q4_many_us(N, K, at, products, group, keep), least) ? FEW_DIRECT : MANY;
}

// ---- 8-bit weights ------------------------------------------------------------------------------------------------------

// gemm8_k's tiles, as TILES, us a stage of 64 columns and the ends of a launch (130 to 2,048 tokens, 768 to 11,008 columns: within 10 %).
// Matrix units busy over a whole launch: 128 x 128 0.45, 256 x 128 0.63, 256 x 256 0.74 to 0.80; LDS 0.25 to 0.35, and a compute unit takes
// in 50 to 74 of the 120 bytes a nanosecond that L2 gives it, whatever the depth of loads: the small ones wait at each stage's barrier.
// Against every other kernel, tile and split at 152 sizes of 17 to 2,048 tokens the plan is 1 % over the best on the geometric mean, 15 %
// at the worst (200 tokens 14336 -> 256 in 14 shares 11.5 us, in 8 10.0).
constexpr int Q8_TILES = 6;
constexpr Tile TILES8[Q8_TILES] = {
    {256, 256, 256, 0.50, 0.82, 7.3},      // 8 waves, gemm8_big_k
    {128, 128, 512, 0.17, 0.50, 5.5},      // 4 waves, two on a compute unit
    {128, 64, 256, 0.13, 0.15, 4.0},       // 2 groups of 4 waves, each every other stage
    {128, 128, 256, 0.155, 0.26, 5.5},     // the same
    {256, 128, 256, 0.265, 0.467, 6.5},    // 8 waves
    {64, 64, 512, 0.081, 0.18, 3.6},       // 2 groups of 2 waves, two on a compute unit
};
constexpr int Q8_SPLIT = 5;         // the tile whose K axis can be split: it pays for few results

// us of a stage of a tile with n of its workgroups at once: alone's with few, and more the more compute units have one (128 x 128 0.163,
// 0.19, 0.206 and 0.27 with 64, 160, 192 and 256); with a second one on some, full's
inline double stage8(const Tile& c, int64_t n)
{
    const double w = (double)n / 256, one = c.slots == 256 ? c.full : c.full / 2;
    return n <= 256 ? c.alone + (one - c.alone) * w * w : c.full;
}

// Tiles of a product with M x N results and stages of 64 columns, as plan_product: the joining kernel (4.5 us) and the sums' bytes cost
// as much (130 tokens 11008 -> 256 16.2 us, split 8.5; 11008 -> 4096 18.0, in two 25), and large tiles go ahead for as many rows of M as
// fill whole rounds
inline TilePlan plan8(int64_t M, int64_t N, int stages, bool can_split, bool can_part = true)
{
    TilePlan best = {0, 1, 0, 1e30};
    if (M <= 0 || N <= 0) return {0, 1, 0, 0.0};
    for (int t = 0; t < Q8_TILES; ++t)
        for (int s = 1; s <= 16; ++s)
        {
            if (s > 1 && (!can_split || t != Q8_SPLIT || stages / s < 8)) break;
            const Tile& c = TILES8[t];
            const int64_t b = (M + c.M - 1) / c.M * ((N + c.N - 1) / c.N) * s, full = b / c.slots, rest = b % c.slots;
            const int each = (stages + s - 1) / s;
            double us = full * (each * c.full + c.ends);
            if (rest) us += each * stage8(c, rest) + c.ends;
            if (s > 1) us += 4.5 + (double)M * N * s * 8.0 / 4e6;
            if (us < best.us) best = {t, s, 0, us};
        }
    const int64_t tn = (N + 255) / 256, rounds = (M + 255) / 256 * tn / 256, head = rounds * 256 / tn * 256;
    if (can_part && head > 0 && head < M)
    {
        const TilePlan tail = plan8(M - head, N, stages, false, false);
        const double us = rounds * (stages * TILES8[0].full + TILES8[0].ends) + tail.us + 2.0;
        if (us < best.us) best = {tail.tile, 1, head, us};
    }
    return best;
}

inline TilePlan q8_plan(int N, int K, int T, int products) { return plan8((int64_t)N * products, T, (K + 63) / 64, true); }

constexpr int S8_W = 8;             // waves of a workgroup (skinny8_k)
constexpr int S8_SLOTS = 32;        // pieces of 512 values that a workgroup quantizes, one or four a wave
inline int skinny8_pieces(int T, int K) { return T * ((K + 511) / 512); }
inline bool skinny8_fused(int T, int K) { return T <= 16 && K % 8 == 0 && skinny8_pieces(T, K) <= S8_SLOTS; }

// skinny8_k, tiles of 16 rows of W per workgroup, 1 or 2 (to 80 tokens): a workgroup takes in its rows of W and the tokens; us for 1,024
// columns of 16 of them are 0.10 alone and 0.20 when every compute unit has a workgroup (of 32 rows, more of them from HBM: 0.13 and
// 0.26), and of more workgroups than units some have one more, which is the last to end. us with 1 / 2: 77 tokens 5120 -> 4608 12.7 / 9.9
// (by gemm8_k 10.6), 64 tokens 2304 -> 5120 5.9 / 5.3, 4096 -> 4096 6.7 / 7.5, 4096 -> 1536 5.3 / 6.6
constexpr int S8_MOST = 128;
struct Few8 { int rt; double us; };
inline Few8 q8_few_rows(int N, int K, int T, int products)
{
    auto us = [&](int rt) {
        const double w = (double)(((N + 15) / 16 * products + rt - 1) / rt) / 256;
        const int whole = (int)w;
        const double rounds = w > whole ? whole + 0.5 + 0.5 * (w - whole) : w, first = rt == 1 ? 0.10 : 0.13;
        return 2.6 + (rt + (T + 15) / 16) * (K / 1024.0) * first * (w <= 1.0 ? 1.0 + w : 2.0 * rounds);
    };
    const int rt = T <= 80 && us(2) < us(1) ? 2 : 1;
    return {rt, us(rt)};
}

// A product of T tokens with an N x K matrix (or two, side by side): skinny8_k to 16 tokens, to 128 where it is planned sooner than gemm8_k
// (33 tokens 5120 -> 2304 5.6 us, by gemm8_k 8.4; 96 tokens 8.1 / 10.9; 64 tokens 4096 -> 11008 12.7 / 11.0), which reads W no faster than
// HBM does
inline bool q8_few(int N, int K, int T, int products)
{
    if (T <= 16 || T > S8_MOST) return T <= 16;
    return q8_few_rows(N, K, T, products).us <= std::max(q8_plan(N, K, T, products).us, 1.0 + (double)N * K * products / 5.0e6);
}

inline int padded(int n) { return (n + 7) / 8 * 8; }
inline int slices_of(int K) { return (K + SL_K - 1) / SL_K; }

inline size_t skinny_part_bytes(int N, int K, int T, int products, int group)
{
    return product_path(N, K, T, products, group, false) == FEW_SLICES ? (size_t)products * slices_of(K) * T * padded(N) * 4 : 0;
}

// What was measured of gemm_q4_k: us a step of 128 columns with a workgroup on every other compute unit or fewer, and with
// two on each; of decoding a matrix first: bytes at 4.8 TB/s and a launch
struct Q4Plan { bool direct; int splits; double us; };

inline Q4Plan q4_plan(int N, int K, int T, int products, int group, bool keep)
{
    if (!keep && T > q4_whole_most(group))
        return {false, 1, products * ((double)N * K * 2.5 / 4.8e6 + 2.0) + product_us(N, T, K, products)};
    const int KT = (K + SK_K - 1) / SK_K;
    const int64_t tiles = (int64_t)((N + QG_N - 1) / QG_N) * ((T + QG_T - 1) / QG_T) * products;
    const double more = group == 128 ? 1.0 : group == 64 ? 1.08 : 1.35;
    Q4Plan best = {true, 1, 1e30};
    for (int s = 1; s <= 16 && (s == 1 || KT / s >= 2); ++s)
    {
        const int64_t b = tiles * s, full = b / 512, rest = b % 512;
        const int each = (KT + s - 1) / s;
        double us = full * (each * 2.3 * more + 3.0);
        if (rest) us += each * (rest <= 256 ? 1.37 : 2.3) * more + 3.0;
        if (s > 1) us += 5.0 + (double)N * T * products * s * 8.0 / 4e6;
        if (us < best.us) best = {true, s, us};
    }
    return best;
}

inline double q4_many_us(int N, int K, int T, int products, int group, bool keep) { return q4_plan(N, K, T, products, group, keep).us; }

inline size_t group_sums_bytes(int K, int T, int group) { return round_up((size_t)(round_up(K, SK_K) / group) * round_up(T, QG_T) * 4, 256); }

// part and sums of a direct product; the decoded matrices and the tiled product's partial sums of the other
inline size_t q4_many_bytes(int N, int K, int T, int products, int group, bool keep)
{
    const Q4Plan p = q4_plan(N, K, T, products, group, keep);
    if (!p.direct) return round_up((size_t)products * N * K * 2, 256) + product_part_bytes(N, T, K, products);
    return group_sums_bytes(K, T, group) + (p.splits > 1 ? (size_t)products * p.splits * T * padded(N) * 4 : 0);
}

// Workspace of a product
inline size_t product_bytes(int N, int K, int T, int products, int group, bool keep)
{
    if (product_path(N, K, T, products, group, keep) != MANY) return skinny_part_bytes(N, K, T, products, group);
    return group ? q4_many_bytes(N, K, T, products, group, keep) : product_part_bytes(N, T, K, products);
}

// Partial sums of a product in 8 bits
inline size_t q8_part_bytes(int N, int K, int T, int products)
{
    if (q8_few(N, K, T, products)) return 0;
    const TilePlan p = q8_plan(N, K, T, products);
    return p.splits > 1 ? (size_t)p.splits * products * T * padded(N) * 4 : 0;
}

}  // namespace bmx
