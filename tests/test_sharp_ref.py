"""What the sharp bounds tell apart, on the CPU: at the tests' own lengths a product in fp32 passes, and one that is wrong does not:
zeros, a lost step of K, tokens or rows exchanged. The mistakes are planted in the reference product."""
import pytest
import torch

import ffn_sizes as Z
import sharp_ref as S

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
# the summed lengths of every size (tokens: the weights' gradients)
LENGTHS = sorted({K for _, K, *_ in Z.LINEAR} | {n for _, H, I, *_ in Z.BLOCK4 + Z.BLOCK16 for n in (H, I)} | {T for T, *_ in Z.BLOCK16 if T > 64})


def mistakes(a, b, step):
    """Products with something wrong, as (name, result before rounding)."""
    y = a @ b.t()
    K = a.shape[1]
    yield "zeros", torch.zeros_like(y)
    if K >= 2 * step:
        lost = a.clone()
        lost[:, -step:] = 0.0
        yield "last step lost", lost @ b.t()
        twice = a.clone()
        twice[:, :step] *= 2.0
        yield "first step twice", twice @ b.t()
    yield "tokens exchanged", y[torch.tensor([1, 0] + list(range(2, y.shape[0])))]
    yield "a row of its neighbour", torch.cat((y[:, 1:2], y[:, 1:]), 1)


def expect(y64, e, dt, right, wrong):
    S.check("right", right.to(dt), y64, S.rounded(y64, e, dt))
    for name, y in wrong:
        with pytest.raises(AssertionError):
            S.check(name, y.to(dt), y64, S.rounded(y64, e, dt))


@pytest.mark.parametrize("dt", sorted(DT))
def test_products(dt):
    for K in LENGTHS:
        g = torch.Generator().manual_seed(K)
        a = torch.randn((8, K), generator=g).to(DT[dt])
        b = (torch.randn((48, K), generator=g) / K ** 0.5).to(DT[dt])
        y64, e = S.product(a.double(), b.double())
        expect(y64, e, DT[dt], a.float() @ b.float().t(), mistakes(a.double(), b.double(), 64))


@pytest.mark.parametrize("dt", sorted(DT))
def test_products_of_values_that_are_rounded_first(dt):
    """h, dg and du: the reference has them unrounded, the product rounded."""
    for K in LENGTHS:
        g = torch.Generator().manual_seed(K)
        a = torch.randn((8, K), generator=g).double()
        b = (torch.randn((48, K), generator=g) / K ** 0.5).to(DT[dt]).double()
        y64, e = S.product(a, b, S.rounded(a, 0.0 * a, DT[dt]))
        r = a.to(DT[dt])
        expect(y64, e, DT[dt], r.float() @ b.float().t(), mistakes(r.double(), b, 64))


@pytest.mark.parametrize("dt", sorted(DT))
def test_products_of_4_bit_matrices(dt):
    for T, K, _, G in Z.LINEAR + [(T, n, 0, G) for T, H, I, G in Z.BLOCK4 for n in (H, I)]:
        g = torch.Generator().manual_seed(K)
        x = torch.randn((8, K), generator=g).to(DT[dt]).double()
        _, (w, steps) = S.symmetric_codes("cpu", 48, K, G, T % 2, torch.float16, K)
        # the bound of a call of that many tokens
        y64, e = S.q4_product(x.repeat((max(T, 8) + 7) // 8, 1)[:max(T, 8)], (w, steps), DT[dt], G)
        y64, e = y64[:8], e[:8]
        v = w if S.q4_whole(T, G) else w.to(DT[dt]).double()
        expect(y64, e, DT[dt], x @ v.t(), mistakes(x, w, 128))
