"""The root-mean-square norm and rows in 8 bits in 64 bits, and the bounds their kernels have to keep."""
import torch

import ffn_ref as R

STEP = 2.0 ** -23          # one step of an fp32 value, relative; a rounding is off by half of it
# A row's sums: a lane's chain (at most 16 values), its wave's six steps and up to 16 waves: each value passes fewer than 40
# additions. Of a sum of squares, all terms positive, that is its relative error.
CHAIN = 40 * STEP / 2
# rstd: half of the sum's, and division by H, sum with eps, root and reciprocal, each within a step
RSTD = CHAIN / 2 + 4 * STEP


def norm(v, w, eps):
    """y in 64 bits of rows v, and the bound of its error before its rounding: v w rounded, times rstd rounded."""
    y = v * w / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    return y, y.abs() * (RSTD + STEP)


def norm_grads(v, w, eps, dy, dr):
    """dv and dw in 64 bits and bounds of their errors before their roundings."""
    T, H = v.shape
    rstd = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    g = dy * w
    k = (g * v).mean(1, keepdim=True) * rstd * rstd
    # (the sum of g v cancels: its error goes by its terms; g is rounded, the sum divided, multiplied twice by rstd)
    ek = (CHAIN + STEP) * (g * v).abs().mean(1, keepdim=True) * rstd * rstd + k.abs() * (2 * RSTD + 4 * STEP)
    dv = rstd * (g - v * k)
    ev = rstd * ((g.abs() + (v * k).abs()) * (RSTD + 4 * STEP) + v.abs() * ek * (1 + 4 * STEP))
    if dr is not None:
        ev = ev + STEP * (dv.abs() + ev + dr.abs())
        dv = dv + dr
    t = dy * v * rstd
    # a column: a workgroup's rows one after the other (of 256 workgroups at least), every 64th of at most 4,096 workgroups, 64 groups
    adds = (T + 255) // 256 + 64 + 64
    return dv, ev, t.sum(0), t.abs().sum(0) * (RSTD + 2 * STEP + adds * STEP)


def quantized(v, e=0.0):
    """Rows v, known to within e (a tensor or 0), as the 8-bit form's values in 64 bits, and a bound on how far a kernel's are from
    them: where a value within its error of a border between two codes gets the other one, a step; and the scale's error. The kernel
    multiplies by 127 / top rounded (half a step of fp32, and as much for the product with magnitudes up to 127)."""
    e = e if torch.is_tensor(e) else torch.zeros_like(v)
    top, etop = v.abs().amax(1, keepdim=True), e.amax(1, keepdim=True)
    some = top > 0
    s = torch.where(some, top / 127.0, torch.ones_like(top))
    z = v / s
    rel = torch.where(some, etop / s / 127.0, torch.zeros_like(top)) + 2 * STEP
    ez = e / s + z.abs() * rel
    code = torch.round(z)
    near = ((z - torch.floor(z)) - 0.5).abs() <= ez
    assert float(ez.max()) < 0.5
    q = torch.where(some, code * s, torch.zeros_like(v))
    return q, torch.where(some, near * s * (1 + rel) + q.abs() * rel, torch.zeros_like(v))


def product(q, w, eq=0.0):
    """q W^T of 8-bit values in 64 bits and the bound of its error before its rounding, q off by eq: the sum is exact, then goes to
    fp32 and is multiplied twice. (This sum, in 64 bits, of products that are scales' multiples is itself off by half a step, 2^-53, of
    its terms per addition and product: where the whole numbers add up to 0, it is all that is left of it.)"""
    y = q @ w.t()
    e = y.abs() * 2 * STEP + (q.shape[1] + 2) * 2.0 ** -53 * (q.abs() @ w.abs().t())
    if torch.is_tensor(eq):
        e = e + (1 + 2 * STEP) * (eq @ w.abs().t())
    return y, e


def act_rel(act, g):
    """The activation's fp32 evaluation, relative to it: as ffn_ref.act_err, but that an error of the exponent z's changes
    1 / (1 + exp(-z)) by (1 - sigmoid(z)) of itself only, nothing for large z."""
    if act == 2:
        return torch.full_like(g, 4 * STEP)
    z = {0: g, 1: 2.0 * 0.797884560803 * (g + 0.044715 * g ** 3), 3: 1.702 * g}[act]
    return 12 * STEP + 4 * STEP / 2 * z.abs() * torch.sigmoid(-z)


def hidden(x8, wg, wu, act, L):
    """h = act(g, u) in 64 bits and the bound of its error in fp32: the corners of the errors of g and u, twice (as ffn_ref.forward), and
    the activation's own, which ends at the clamps."""
    (g, eg), (u, eu) = product(x8, wg), product(x8, wu)
    h = R.act_h(act, g, u, L)
    ends = [(R.act_h(act, g + a * eg, u + b * eu, L) - h).abs() for a in (-1, 1) for b in (-1, 1)]
    top = L if L else float("inf")
    gc, uc = (g.clamp(max=top) if act == 3 else g), u.clamp(-top, top)
    a = R.act_a(act, gc).abs()
    if act != 3:
        a = a.clamp(max=2 * top)
    eh = 2.0 * torch.stack(ends).amax(0) + (act_rel(act, gc) + 2 * STEP) * a * (uc.abs() + 1.0) + 2.0 ** -126 * g.abs() * (u.abs() + 1.0)
    return h, eh


def block(x8, wg, wu, wd, act, L):
    """The gated block on 8-bit rows x8 (values) and matrices in 64 bits, and the bound of its error before its rounding."""
    q, eq = quantized(*hidden(x8, wg, wu, act, L))
    return product(q, wd, eq)
