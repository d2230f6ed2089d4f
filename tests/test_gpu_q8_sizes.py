"""Products and gated blocks in 8 bits at sizes that reach every kernel instance (tests/q8_sizes.py), against 64 bits."""
import pytest
import torch

import ffn_ref as R
import q8_sizes as Z
import rows8_ref as Q
from test_gpu_q8 import F32, block, check_linear, matrix, rand, values

pytestmark = pytest.mark.gpu
F16 = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("T,K,N", Z.LINEAR)
def test_linear(cuda, T, K, N):
    import bmx
    given, w = matrix(cuda, N, K, seed=N)
    q = bmx.Q8Matrix(*given)
    for dt in F16:
        x = rand(cuda, T, K, dt=dt, seed=T)
        y = bmx.ops.q8_linear(x, q)
        check_linear(x, q, w, y)
        assert torch.equal(bmx.ops.q8_linear(bmx.ops.quantize_rows(x), q), y)


@pytest.mark.parametrize("T,H,I", Z.BLOCK)
def test_gated_block(cuda, T, H, I):
    """Forward of x and of its rows, and added with and without the gate vector; the rows behind the last token stay as they are."""
    import bmx
    act, L = T % 4, 1.25 if H % 16 else 0.0
    ffn, w = block(cuda, H, I, act, L)
    for dt in F16:
        x = rand(cuda, T, H, dt=dt, seed=T)
        rows = bmx.ops.quantize_rows(x)
        y64, e = Q.block(values(rows), *w, act, L)
        y = ffn(x)
        R.check("y", y, y64, R.rounded(y64, e, dt))
        assert torch.equal(ffn(rows), y)
        vec = (torch.randn(H, device=cuda) / H ** 0.5).to(dt) if dt is F16[0] else None
        base = torch.randn((T + 2, H), device=cuda)
        out = base.clone()
        ffn.add_to(out[:T], x, vec, rows)
        s = torch.ones((T, 1), dtype=torch.float64, device=cuda) if vec is None else torch.sigmoid(x.double() @ vec.double())[:, None]
        want = base[:T].double() + s * y64
        R.check("out", out[:T], want, s * e + 2.0 ** -22 * (want.abs() + y64.abs()) + H * R.ACC * y64.abs())
        assert out.dtype is F32 and torch.equal(out[T:], base[T:])


@pytest.mark.parametrize("T,K", [((1 << 23) + 5, 3), ((1 << 20) + 37, 8)])
def test_more_rows_than_an_axis_of_a_launch_holds(cuda, T, K):
    """2^23 workgroups of 512 threads are more than 2^32 threads; the first form with rows at any boundary, the second the norm's."""
    import bmx
    x = torch.randn((T, K), device=cuda).half()
    rows = bmx.ops.quantize_rows(x)
    top = x.abs().amax(1).float()
    assert torch.equal(rows.scale, (top.double() / 127.0).float())
    want = torch.round(x.double() * 127.0 / x.abs().amax(1, keepdim=True).double())
    assert torch.equal(rows.int8().double(), want)
    if K % 8 == 0:
        norm = bmx.RMSNorm(torch.ones(K, device=cuda).half())
        y, rows, r = norm.both(x, x)
        v = r.double()
        y64 = v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt()
        # (before its rounding y is off by its sum of 8 squares and six operations, under 2^-20; fp16 numbers below 2^-14 lie 2^-24
        # apart whatever their size, which a bound relative to y64 does not hold: a rounding there is off by up to 2^-25)
        assert torch.equal(r, x + x)
        R.check("y", y, y64, R.rounded(y64, 2.0 ** -20 * y64.abs(), y.dtype))
        assert torch.equal(rows.int8().double(), torch.round(v * 127.0 / v.abs().amax(1, keepdim=True)))


def test_more_than_2_to_31_codes(cuda):
    """A matrix, and tokens, whose codes lie past 32 bits: the last rows' results are those of a matrix of them alone, bit for bit."""
    import bmx
    n, K, few = 540000, 4096, 70
    codes = torch.randint(-128, 128, (n, K), device=cuda, dtype=torch.int8)
    scale = (torch.rand(n, device=cuda) + 0.2) / 4096
    big, last = bmx.Q8Matrix(codes, scale), bmx.Q8Matrix(codes[-few:].contiguous(), scale[-few:].contiguous())
    assert torch.equal(big.int8()[-few:], codes[-few:])
    rows = bmx.Rows8(codes, scale, torch.bfloat16)
    del codes
    for T in (1, 16, 40, 130, 300):
        x = rand(cuda, T, K, dt=torch.bfloat16, seed=T)
        assert torch.equal(bmx.ops.q8_linear(x, big)[:, -few:], bmx.ops.q8_linear(x, last))
    del big
    tail = bmx.Rows8(last.int8(), last.scale, torch.bfloat16)
    for N in (8, 70, 300):
        q = bmx.Q8Matrix.quantize(torch.randn((N, K), device=cuda) / 64)
        assert torch.equal(bmx.ops.q8_linear(rows, q)[-few:], bmx.ops.q8_linear(tail, q))
