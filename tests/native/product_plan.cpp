// The planner and the operand spans of the tiled products (csrc/product_plan.hpp), built with g++ for the CPU tests.
#include <cstdio>
#include <string>

#include "product_plan.hpp"

using namespace bmx;

namespace {

// The largest number of bytes past an operand's end that its tiles' ranges reach, over the launches of one product; moved: as if
// A's pointer were moved to the part's rows and its rows counted from there
int64_t past_the_end(const TilePlan& p, int M, int mats, int K, int ld, bool across, bool moved)
{
    ProductPart part[2];
    const int n = p.splits == 1 ? product_parts(p, M, mats, part) : 1;
    if (p.splits > 1) part[0] = {p.tile, 0, M};
    const int64_t bytes = (int64_t)(across ? K : M) * ld * 2;
    int64_t worst = INT64_MIN;
    int next = 0;
    for (int i = 0; i < n; ++i)
    {
        const ProductPart& q = part[i];
        if (q.from != next || q.rows <= 0) return INT64_MAX;       // every row once, in order
        next = q.from + q.rows;
        const int64_t pointer = moved ? (across ? (int64_t)q.from : (int64_t)q.from * ld) * 2 : 0;
        const int bm = TILES[q.tile].M / mats, r = moved ? 0 : q.from;
        for (int m0 = 0; m0 < q.rows; m0 += bm)
            for (int k0 = 0; k0 < K; k0 += GK)
            {
                const OperandSpan s = operand_span(across, ld, r + q.rows, K, r + m0, k0);
                const int64_t at = ((int64_t)(across ? k0 : q.from + m0) * ld + (across ? q.from + m0 : k0)) * 2;
                if (pointer + s.first != at) return INT64_MAX;     // the tile's own first value
                worst = std::max(worst, pointer + s.first + s.left - bytes);
            }
    }
    return next == M ? worst : INT64_MAX;
}

// ---- the kernel instances that a call launches, as text, one a line ----
std::string number(const char* name, int v) { return std::string(" ") + name + std::to_string(v); }

// A product on gemm16_k; how: which operands lie across K, what becomes of the sums
std::string tiled(const TilePlan& p, const std::string& how, const std::string& epi)
{
    if (p.splits > 1) return "gemm16" + number("tile", p.tile) + " " + how + " part\nfinish " + epi + "\n";
    if (p.head) return "gemm16 tile0 " + how + " " + epi + " head\ngemm16" + number("tile", p.tile) + " " + how + " " + epi + " rest\n";
    return "gemm16" + number("tile", p.tile) + " " + how + " " + epi + "\n";
}

std::string product_names(int N, int K, int T, int products, int group, bool keep, const std::string& epi)
{
    const ProductPath path = product_path(N, K, T, products, group, keep);
    if (path == FEW_DIRECT)
    {
        const FewForm f = few_form(N, K, T, products, group);
        return "skinny" + number("rt", f.rt) + number("g", group) + " " + epi + (f.xl ? " xl" : T > 16 ? " tiles" : "") + "\n";
    }
    if (path == FEW_SLICES) return "slice" + number("tt", (T + 15) / 16) + number("g", group) + "\nfinish " + epi + "\n";
    if (!group) return tiled(plan_for(N, T, K, products), "along", epi);
    const Q4Plan p = q4_plan(N, K, T, products, group, keep);
    if (!p.direct) return tiled(plan_for(N, T, K, products), "along", epi) + "dequant\n";
    if (p.splits > 1) return "gemm_q4" + number("g", group) + " part\nfinish " + epi + "\n";
    return "gemm_q4" + number("g", group) + " " + epi + "\n";
}

}  // namespace

extern "C" {

// op: 0 a 4-bit product (H -> I, group), 1 / 2 a block with 16-bit (group 0) or 4-bit weights, 2 its added form, 3 the gradients
int plan_names(int op, int T, int H, int I, int group, char* out, int size)
{
    std::string s;
    if (op == 0) s = product_names(I, H, T, 1, group, false, "store");
    else if (op < 3) s = product_names(I, H, T, 2, group, false, "gu") + product_names(H, I, T, 1, group, false, op == 2 ? "add" : "store");
    else
    {
        const BackTiles b = back_tiles(H, I, T);
        if (b.two) s += "gemm16_two\n";
        // (down's gradient alone, or without it, has a launch of its own either way)
        s += tiled(b.dh, "across", "dgu") + tiled(b.dd, "both", "store") + tiled(b.dx, "across", "store") + tiled(b.dw, "both", "store");
    }
    return snprintf(out, size, "%s", s.c_str()) < size;
}

// The products of a block's passes: 0 gate and up, 1 down, 2 dh, 3 dx, 4 down's gradient, 5 gate's and up's. Returns the bytes
// past A's end; parts: of how many launches (0: K split)
int64_t plan_past_the_end(int H, int I, int T, int which, int moved, int* parts)
{
    const BackTiles b = back_tiles(H, I, T);
    const TilePlan fwd = which == 0 ? plan_for(I, T, H, 2) : plan_for(H, T, I, 1);
    const TilePlan p = which < 2 ? fwd : which == 2 ? b.dh : which == 3 ? b.dx : which == 4 ? b.dd : b.dw;
    *parts = p.splits > 1 ? 0 : p.head ? 2 : 1;
    switch (which)
    {
        case 0: return past_the_end(p, I, 2, H, H, false, moved);
        case 1: return past_the_end(p, H, 1, I, I, false, moved);
        case 2: return past_the_end(p, I, 1, H, I, true, moved);
        case 3: return past_the_end(p, H, 1, I, H, true, moved);
        case 4: return past_the_end(p, I, 1, T, I, true, moved);
        default: return past_the_end(p, H, 1, T, H, true, moved);
    }
}

// Whether a 4-bit product decodes and rounds the weights first
int plan_rounds(int N, int K, int T, int products, int group, int keep)
{
    return product_path(N, K, T, products, group, keep) == MANY && !q4_plan(N, K, T, products, group, keep).direct;
}

}  // extern "C"
