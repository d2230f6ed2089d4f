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
