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
