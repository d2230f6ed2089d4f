"""Calls whose arrays pass 2^31 values: the last tokens' results are those of the formulas, and sums over all tokens have them all."""
import pytest
import torch

import ffn_ref as R
import sharp_ref as S

pytestmark = pytest.mark.gpu


def normal(cuda, seed, *shape, dt):
    """In parts, so that no fp32 copy of all is needed."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    out = torch.empty(shape, dtype=dt, device=cuda)
    for i in range(0, shape[0], 1 << 16):
        part = out[i:i + (1 << 16)]
        part.copy_(torch.randn(part.shape, device=cuda, generator=g))
    return out


@pytest.mark.parametrize("T,H,I", [(400008, 64, 5504), (400008, 5504, 64)])
def test_block_and_its_gradients(cuda, T, H, I):
    """g, u, h and their gradients, or x, y, dy and dx, of 2.2e9 values each."""
    import bmx
    dt = torch.bfloat16
    x, dy = normal(cuda, 1, T, H, dt=dt), normal(cuda, 2, T, H, dt=dt)
    w = [(torch.randn((a, b), device=cuda, generator=torch.Generator(device=cuda).manual_seed(s)) / b ** 0.5).to(dt).requires_grad_()
         for s, (a, b) in enumerate(((I, H), (I, H), (H, I)))]
    ffn = bmx.GatedFFN(*w)
    x.requires_grad_()
    y = ffn.forward(x)
    dx, dwg, dwu, dwd = torch.autograd.grad(y, [x] + w, dy)
    x, y, w64 = x.detach(), y.detach(), [t.detach().double() for t in w]
    ends = torch.cat((torch.arange(40), torch.arange(T // 2, T // 2 + 40), torch.arange(T - 40, T))).to(cuda)
    xs, dys = x[ends].double(), dy[ends].double()
    _, _, h, _, _, eh = S.forward(xs, *w64[:2], 0, 0.0, S.product)
    y64, e = S.product(h, w64[2], S.rounded(h, eh, dt))
    S.check("y", y[ends], y64, S.rounded(y64, e, dt))
    # gradients, from products in 64 bits of the 16-bit inputs: 8 sigma of the roundings of g, u (fp32), dg and du (half a step of
    # themselves), as in the model sizes' test
    g, u = xs @ w64[0].t(), xs @ w64[1].t()
    hg, hu = R.act_grads(0, g, u, 0.0)
    dh, edh = S.product(dys, w64[2].t().contiguous())
    # slopes' change over g's and u's errors (|f''| <= 1/2, |f'| <= 1.1)
    _, eg = S.product(xs, w64[0])
    _, eu = S.product(xs, w64[1])
    slip, size = S.act_err(0, g), R.act_a(0, g).abs() + 1.0 + g.abs()
    ehg = slip * (u.abs() + 1.0) * (1.0 + size) + eg * u.abs() + 1.1 * eu
    ehu = slip * size + 1.1 * eg
    dg, du = dh * hg, dh * hu
    edg, edu = S.rounded(dg, edh * hg.abs() + dh.abs() * ehg, dt), S.rounded(du, edh * hu.abs() + dh.abs() * ehu, dt)
    a, ea = S.product(dg, w64[0].t().contiguous(), edg)
    b, eb = S.product(du, w64[1].t().contiguous(), edu)
    S.check("dx", dx[ends], a + b, S.rounded(a + b, ea + eb + 2.0 * (ea + eb), dt))
    # The weights' gradients over all tokens, by norm. A cut (half a step, 2^-24, on average) in each of 400,000 additions to a partial
    # sum of 0.7 sigma on average is 0.017, were they all of one sign; the roundings of h or dg, of the result and of g's and u's
    # sums are 0.002 each. 2^-5 is more than all together, and tokens left out from 2^31 values on 0.16.
    want = [torch.zeros_like(t, dtype=torch.float64) for t in w]
    for i in range(0, T, 1 << 15):
        xs, dys = x[i:i + (1 << 15)].double(), dy[i:i + (1 << 15)].double()
        g, u = xs @ w64[0].t(), xs @ w64[1].t()
        sg = torch.sigmoid(g)
        dh = dys @ w64[2]
        want[0] += (dh * u * (sg * (1.0 + g * (1.0 - sg)))).t() @ xs
        want[1] += (dh * g * sg).t() @ xs
        want[2] += dys.t() @ (g * sg * u)
    for name, got, ref in zip(("dgate", "dup", "ddown"), (dwg, dwu, dwd), want):
        for d in (0, 1):                             # every row and every column
            err, size = (got.double() - ref).norm(dim=d), ref.norm(dim=d)
            assert bool((err <= 2.0 ** -5 * size).all()), (name, float((err / size).max()))


@pytest.mark.parametrize("dt,sdt", [(torch.float16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, torch.float16)])
def test_4_bit_product(cuda, dt, sdt):
    """2.4e9 results of decoded weights, and of codes multiplied as they are."""
    import bmx
    T, K, N, G = 600000, 128, 4096, 64
    given, q64 = S.symmetric_codes(cuda, N, K, G, True, sdt, seed=1)
    x = normal(cuda, 3, T, K, dt=dt)
    y = bmx.ops.q4_linear(x, bmx.Q4Matrix(*given, group=G))
    for i in (0, T // 2, 524288 - 2000, T - 4000):   # row 524,288 begins at 2^31 values
        rows = slice(i, i + 4000)
        y64, e = S.q4_product(x[rows].double(), q64, dt, G)
        S.check("y", y[rows], y64, S.rounded(y64, e, dt))
