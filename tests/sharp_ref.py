"""Bounds that grow as the sums do, for the comparisons at model sizes. ffn_ref's hold for any data: each addition of a sum of K
products is off by up to a step of the sum of all magnitudes, which at K of some thousands and 16-bit results is as much as the
result itself. The data here have terms of symmetric, independent signs, and then a sum of any part of them is at most 8 sigma,
sigma^2 the sum of the terms' squares: a sum of symmetric terms over the root of its squares passes t with a probability of at
most 2 exp(-t^2 / 2) whatever the terms' sizes (Efron 1969), 3e-14 for 8. Every one of the K additions, in whichever order, is then
off by at most a step (2^-23, however the matrix units round) of 8 sigma, and errors of a factor (a value rounded before the sum)
add up to at most 8 times the root of their squares."""
import torch

from ffn_ref import ACC, HALF, TINY, act_err, act_h, check, forward, rounded

SIGMAS = 8.0
__all__ = ["product", "q4_product", "q4_whole", "symmetric_codes", "check", "forward", "rounded", "act_err", "act_h", "HALF", "TINY", "ACC"]


def product(a, b, da=0.0):
    """a b^T in 64 bits, and the bound on its error in fp32 with the values of a off by da (a tensor, or 0) before."""
    b2 = (b * b).t()
    bound = SIGMAS * a.shape[1] * ACC * ((a * a) @ b2).sqrt()
    if torch.is_tensor(da):
        bound = bound + SIGMAS * (1 + a.shape[1] * ACC) * ((da * da) @ b2).sqrt()
    return a @ b.t(), bound


def q4_whole(T, group):
    """Whether a call of T tokens keeps the weights' digits (include/bmx.h)."""
    return T <= (256 if group == 32 else 1024)


def q4_product(x, q, dt, group, da=0.0):
    """As product for a 4-bit matrix q = (W, steps) in 64 bits, steps [N, K / group] the scale of one code. To K additions come four
    operations a group. In bf16 the codes carry 128, so that the sums within a group run up to steps (128 + 15 + 128 + zero, at most
    15) times 8 root sum x^2 before the offset comes off. Many tokens: each weight rounded to dt first."""
    w, steps = q
    T, K = x.shape
    n = K + 4 * K // group
    w2 = (w * w).t()
    y, s = x @ w.t(), ((x * x) @ w2).sqrt()
    bound = SIGMAS * n * ACC * s
    if not q4_whole(T, group):
        bound = bound + SIGMAS * HALF[dt] * s + SIGMAS * TINY[dt] * x.norm(dim=1, keepdim=True)
    elif dt == torch.bfloat16:
        parts = (x * x).view(T, K // group, group).sum(2).sqrt()
        bound = bound + SIGMAS * (group + 8) * ACC * 286.0 * (parts @ steps.abs().t())
    if torch.is_tensor(da):
        bound = bound + SIGMAS * (1 + n * ACC) * ((da * da) @ w2).sqrt()
    return y, bound


def symmetric_codes(device, N, K, G, zero, scale_dt, seed):
    """((codes, scale, zero) in checkpoint order, (W, steps) in 64 bits) with codes - zero of symmetric signs."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    r = lambda lo, hi, *s: torch.randint(lo, hi, s, device=device, generator=g)
    z = r(4, 12, N, K // G) if zero else torch.full((N, K // G), 8, device=device)
    spread = lambda t: t.repeat_interleave(G, 1)
    most = torch.minimum(z, 15 - z)
    d = torch.minimum(r(0, 8, N, K), spread(most)) * (r(0, 2, N, K) * 2 - 1)
    c = (d + spread(z)).to(torch.uint8)
    scale = ((torch.rand((N, K // G), device=device, generator=g) + 0.5) / (4 * K ** 0.5)).to(scale_dt)
    w = d.double() * spread(scale.double())
    return (c[:, 0::2] | (c[:, 1::2] << 4), scale, z.to(torch.uint8) if zero else None), (w, scale.double())
