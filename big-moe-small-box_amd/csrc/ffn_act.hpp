// Gated activations of the feed-forward block: h = act(g, u), and dh/dg, dh/du. The functions are act_gate's (bmx_common.hpp),
// in fp32 with the hardware exp2 and reciprocal (about 1 ulp each), and in one form without branches, so that an epilogue
// over a hundred values per lane stays short:
//   a = g' f(g'),  g' = min(g, Lg),  f = sigmoid(g' (c1 + c3 g'^2));  a = f f, f = max(g', 0) for the squared relu (g' f would
//   be NaN at minus infinity)
//   h = min(a, La) (clamp(u, -Lu, Lu) + add)
// silu c1 = 1; gelu (tanh form, 1 + tanh t = 2 sigmoid(2 t)) c1 = 2 sqrt(2 / pi), c3 = 0.044715 c1; silu_oai c1 = 1.702,
// add = 1. silu_oai clamps g before the activation, the others clamp a after it; no clamp is a clamp at infinity.
// A NaN stays one through the clamps; a gradient passes at a clamp's border itself and is zero beyond it. A NaN is beyond none:
// the comparisons ask what is outside, so that a NaN's gradient is one too, not a clean zero that no check for overflow sees.
#pragma once
#include "bmx_common.hpp"

namespace bmx {

struct ActPar {
    float c1, c3, add, Lg, La, Lu;
    int relu2, limited;              // limited: some bound is finite
};

inline ActPar act_par(int act, float limit)
{
    const float inf = __builtin_huge_valf(), L = limit != 0.0f ? limit : inf, c = 2.0f * 0.797884560803f;
    const bool oai = act == BMX_ACT_SILU_OAI;
    ActPar p;
    p.c1 = act == BMX_ACT_GELU ? c : oai ? 1.702f : 1.0f;
    p.c3 = act == BMX_ACT_GELU ? 0.044715f * c : 0.0f;
    p.add = oai ? 1.0f : 0.0f;
    p.Lg = oai ? L : inf;
    p.La = oai ? inf : L;
    p.Lu = L;
    p.relu2 = act == BMX_ACT_RELU2;
    p.limited = limit != 0.0f;
    return p;
}

__device__ __forceinline__ float clamp_hi(float v, float L) { return v > L ? L : v; }
__device__ __forceinline__ float clamp_both(float v, float L) { return v > L ? L : v < -L ? -L : v; }

// f(g); the bound on g^2 keeps c3 g^2 finite (past it sigmoid is 0 or 1 for any c3 > 0)
__device__ __forceinline__ float act_f(const ActPar& p, float g)
{
    const float s = rcp_hw(1.0f + exp_hw(-g * (p.c1 + p.c3 * fminf(g * g, 1e30f))));
    return p.relu2 ? (g < 0.0f ? 0.0f : g) : s;
}

__device__ __forceinline__ float act_a(const ActPar& p, float g, float f) { return (p.relu2 ? f : g) * f; }

__device__ __forceinline__ float act_h(const ActPar& p, float g, float u)
{
    if (!p.limited) return act_a(p, g, act_f(p, g)) * (u + p.add);
    g = clamp_hi(g, p.Lg);
    return clamp_hi(act_a(p, g, act_f(p, g)), p.La) * (clamp_both(u, p.Lu) + p.add);
}

// silu without clamps by itself: act_h's value, in half its operations (an 8-bit epilogue of 128 of them a lane waits for nothing else)
__device__ __forceinline__ bool is_silu(const ActPar& p) { return !p.limited && !p.relu2 && p.c1 == 1.0f && p.c3 == 0.0f; }
__device__ __forceinline__ float silu_h(float g, float u) { return g * rcp_hw(1.0f + exp_hw(-g)) * u; }

// dh/dg and dh/du at (g, u): a' = f + g f', f' = s (1 - s) (c1 + 3 c3 g^2); 2 f for the squared relu
__device__ __forceinline__ void act_grad(const ActPar& p, float g, float u, float& hg, float& hu)
{
    const bool gout = g > p.Lg, uout = fabsf(u) > p.Lu;
    g = clamp_hi(g, p.Lg);
    const float f = act_f(p, g), a = act_a(p, g, f);
    const float da = p.relu2 ? f + f : f + g * (f * (1.0f - f) * (p.c1 + 3.0f * p.c3 * fminf(g * g, 1e30f)));
    hg = gout || a > p.La ? 0.0f : da * (clamp_both(u, p.Lu) + p.add);
    hu = uout ? 0.0f : clamp_hi(a, p.La);
}

}  // namespace bmx
