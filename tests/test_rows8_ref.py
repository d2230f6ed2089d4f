"""The bounds of the 8-bit rows' comparisons (rows8_ref.py): a plain fp32 evaluation keeps them, one with a planted mistake does not."""
import pytest
import torch

import ffn_ref as R
import rows8_ref as Q


def rows(T, K, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((T, K), generator=g) * torch.exp(torch.randn(K, generator=g))


def plain8(v, top_of=None):
    top = (v if top_of is None else top_of).abs().amax(1, keepdim=True)
    return torch.round(v * (127.0 / top)), top / 127.0


@pytest.mark.parametrize("T,K", [(3, 40), (20, 513)])
def test_quantized_bound(T, K):
    v = rows(T, K, T)
    q, b = Q.quantized(v.double())
    c, s = plain8(v)
    R.check("q", c * s, q, b + q.abs() * Q.STEP)
    # truncated codes, and a scale from all but the last values, are off
    for wrong in (torch.trunc(v / s) * s, (lambda c, s: c * s)(*plain8(v, v[:, : K // 2]))):
        with pytest.raises(AssertionError):
            R.check("q", wrong, q, b + q.abs() * Q.STEP)


def test_block_bound():
    T, H, I = 6, 48, 72
    x = rows(T, H, 1)
    c, s = plain8(x)
    w = [rows(n, k, 2 + i) / k ** 0.5 for i, (n, k) in enumerate(((I, H), (I, H), (H, I)))]
    w8 = [a * b for a, b in (plain8(m) for m in w)]
    x8 = (c * s).double()
    y64, e = Q.block(x8, *(m.double() for m in w8), 0, 0.0)
    g, u = c @ w8[0].t() * s, c @ w8[1].t() * s
    h = g * torch.sigmoid(g) * u
    hc, hs = plain8(h)
    R.check("y", (hc @ w8[2].t() * hs), y64, e + K_SUM(I, h, w8[2]))
    for wrong in (h @ w8[2].t(), plain8(h.half().float())[0] @ w8[2].t() * hs * 1.01):
        with pytest.raises(AssertionError):
            R.check("y", wrong, y64, e + K_SUM(I, h, w8[2]))


def K_SUM(K, h, w):
    """What fp32 sums of K terms add to the exact ones of the kernels."""
    return K * R.ACC * (h.double().abs() @ w.double().abs().t())


def test_norm_bounds():
    v, w = rows(5, 200, 3), 1.0 + 0.1 * rows(1, 200, 4)[0]
    y64, e = Q.norm(v.double(), w.double(), 1e-6)
    R.check("y", v * w * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-6), y64, e)
    with pytest.raises(AssertionError):
        R.check("y", v * w * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-3), y64, e)
    dy, dr = rows(5, 200, 5), rows(5, 200, 6)
    dv, ev, dw, ew = Q.norm_grads(v.double(), w.double(), 1e-6, dy.double(), dr.double())
    leaves = [v.double().requires_grad_(), w.double().requires_grad_()]
    y = Q.norm(*leaves, 1e-6)[0]
    want = torch.autograd.grad((y * dy.double()).sum() + (leaves[0] * dr.double()).sum(), leaves)
    assert torch.allclose(dv, want[0], rtol=1e-12, atol=1e-12) and torch.allclose(dw, want[1], rtol=1e-12, atol=1e-12)
    assert bool((ev < 1e-4 * (dv.abs() + 10)).all()) and bool((ew < 1e-3).all())
