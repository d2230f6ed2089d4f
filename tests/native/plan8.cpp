// The planner of the 8-bit products (csrc/product_plan.hpp), built with g++ for the CPU tests.
#include <cstdio>
#include <string>

#include "product_plan.hpp"

using namespace bmx;

namespace {

std::string number(const char* name, int v) { return std::string(" ") + name + std::to_string(v); }

// The instances that a product launches; given: tokens as rows, else of 16 (fp32: 32) bits
std::string names(int N, int K, int T, int products, bool given, bool fp32, const std::string& epi)
{
    const bool fused = !given && skinny8_fused(T, K);
    if (q8_few(N, K, T, products))
        return "skinny8" + (fused ? std::string(fp32 ? " fp32" : " 16") + number("ns", skinny8_pieces(T, K) <= S8_W ? 1 : 4) : std::string(" codes")) +
               number("tt", (T + 15) / 16) + number("rt", fused ? 1 : q8_few_rows(N, K, T, products).rt) + " " + epi + "\n";
    const TilePlan p = q8_plan(N, K, T, products);
    if (p.splits > 1) return "gemm8" + number("tile", p.tile) + " part\nfinish8 " + epi + "\n";
    if (p.head) return "gemm8 tile0 " + epi + "\ngemm8" + number("tile", p.tile) + " " + epi + "\n";
    return "gemm8" + number("tile", p.tile) + " " + epi + "\n";
}

}  // namespace

extern "C" {

// op: 0 a product (H -> I) of x, 1 of given rows, 2 a block, 3 its added form
int plan8_names(int op, int T, int H, int I, char* out, int size)
{
    const std::string s = op < 2 ? names(I, H, T, 1, op == 1, false, "store")
                                 : names(I, H, T, 2, false, false, "gu") + names(H, I, T, 1, false, true, op == 3 ? "add" : "store");
    return snprintf(out, size, "%s", s.c_str()) < size;
}

// Rows of W that a product's launches take, each once and in order, in whole blocks of 16 but for the last: 0 when they do not
int plan8_rows(int N, int K, int T, int products)
{
    const TilePlan p = q8_plan(N, K, T, products);
    if (p.splits > 1) return N;
    ProductPart part[2];
    const int n = product_parts(p, N, products, part);
    int next = 0;
    for (int i = 0; i < n; ++i)
    {
        if (part[i].from != next || part[i].from % 16 || part[i].rows <= 0) return 0;
        next += part[i].rows;
    }
    return next;
}

int64_t plan8_part_bytes(int N, int K, int T, int products) { return (int64_t)q8_part_bytes(N, K, T, products); }
int plan8_splits(int N, int K, int T, int products) { return q8_few(N, K, T, products) ? 1 : q8_plan(N, K, T, products).splits; }

}  // extern "C"
