"""The gated feed-forward block in 64 bits, and the bounds its 16-bit kernels have to keep."""
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # half a step of a rounding, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}    # half a step of the smallest values
# A sum of n products in fp32: every addition is off by at most one step (2^-23, whichever way the matrix units round) of a
# partial sum that is at most the sum of the magnitudes
ACC = 2.0 ** -23


def act_err(act, g):
    """The activation's fp32 evaluation, relative to its factors: exp2, reciprocal and about ten operations around them at
    2^-23 each, and the exponent's own three roundings (half a step, 2^-24, of itself each), which exp turns into a relative
    error of that size."""
    z = g.abs() * {0: 1.0, 1: 1.6, 2: 0.0, 3: 1.71}[act] * ((1.0 + 0.0448 * g * g) if act == 1 else 1.0)
    return 12 * 2.0 ** -23 + 3 * 2.0 ** -24 * z


def act_a(act, g):
    if act == 0:
        return g * torch.sigmoid(g)
    if act == 1:
        # 0.5 (1 + tanh t) = sigmoid(2 t), which keeps its digits far below zero where 1 + tanh t cancels, in 64 bits too
        return g * torch.sigmoid(2.0 * 0.797884560803 * (g + 0.044715 * g ** 3))
    if act == 2:
        return g.clamp(min=0.0) ** 2
    return g * torch.sigmoid(1.702 * g)


def act_h(act, g, u, L):
    if act == 3:
        if L:
            g, u = g.clamp(max=L), u.clamp(-L, L)
        return (u + 1.0) * act_a(act, g)
    a = act_a(act, g)
    if L:
        a, u = a.clamp(max=L), u.clamp(-L, L)
    return a * u


def act_grads(act, g, u, L):
    g, u = g.clone().requires_grad_(), u.clone().requires_grad_()
    with torch.enable_grad():
        h = act_h(act, g, u, L)
        return torch.autograd.grad(h.sum(), (g, u))


def product(a, b, da=0.0):
    """a b^T in 64 bits, and the bound on its error in fp32 with a off by da (a tensor, or 0)."""
    bound = a.shape[1] * ACC * (a.abs() @ b.abs().t())
    if torch.is_tensor(da):
        bound = bound + (1 + a.shape[1] * ACC) * (da @ b.abs().t())
    return a @ b.t(), bound


def q4_product(x, q, dt, da=0.0):
    """As product for a 4-bit matrix q = (W, spread) in 64 bits. Calls of many tokens round each weight to dt first. Calls
    of few multiply with the codes: exactly in fp16; in bf16 with 128 + code, whose sums run up to spread =
    scale (128 + 15 + 128 + zero) per weight before the offset comes off (five more operations a group)."""
    w, spread = q
    y, bound = product(x, w, da)
    bound = bound + HALF[dt] * (1 + x.shape[1] * ACC) * (x.abs() @ w.abs().t()) + 5 * ACC * (x.abs() @ w.abs().t())
    if dt == torch.bfloat16:
        bound = bound + (x.shape[1] + 5) * ACC * (x.abs() @ spread.t())
    # a weight below the type's normal range is rounded to its smallest step
    return y, bound + TINY[dt] * x.abs().sum(1, keepdim=True)


def forward(x, wg, wu, act, L, prod=product):
    """g, u, h in 64 bits and bounds of their errors before their rounding; h's takes the activation's change over the errors
    of g and u from their four corners, twice."""
    g, eg = prod(x, wg)
    u, eu = prod(x, wu)
    h = act_h(act, g, u, L)
    ends = [(act_h(act, g + a * eg, u + b * eu, L) - h).abs() for a in (-1, 1) for b in (-1, 1)]
    # the sigmoid of z < -87.3 is below 2^-126, the smallest normal fp32 value (and exp(-z) past 88.7 is infinite, its
    # reciprocal 0): there it may come out as 0, off by less than 2^-126
    eh = (2.0 * torch.stack(ends).amax(0) + act_err(act, g) * ((u.abs() + 1.0) * act_a(act, g).abs()) +
          2.0 ** -126 * g.abs() * (u.abs() + 1.0))
    return g, u, h, eg, eu, eh


def rounded(v, e, dt):
    """Bound of v's error after a rounding to dt, v off by e before it."""
    return e + HALF[dt] * (v.abs() + e) + TINY[dt]


def check(name, got, want, bound):
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} values off, worst {float((d / bound).nan_to_num(9e9).max()):.3g} "
                                 f"times the bound at {torch.nonzero(bad)[0].tolist()}")
