// Plans of the tiled products (gemm16.hpp): tiles, splits of K, parts of a product, and where an operand's tile ends. Plain host
// C++ without HIP: the library's calls and the CPU tests run the same arithmetic.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>

namespace bmx {

constexpr int GK = 64;      // K of a tile

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

}  // namespace bmx
