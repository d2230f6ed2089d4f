"""The 8-bit gated block with silu and no clamp, which the tiled kernels evaluate in a branch of their own: at the sizes that reach every
kernel instance, against 64 bits, and a token's results the same bits in calls of few tokens, which have no such branch."""
import pytest
import torch

import ffn_ref as R
import q8_sizes as Z
import rows8_ref as Q
from test_gpu_q8 import block, rand, values

pytestmark = pytest.mark.gpu
# several large tiles a workgroup, and large tiles ahead of smaller ones
MORE = [(2300, 4104, 2568), (4100, 2056, 1032), (8200, 136, 4104)]


@pytest.mark.parametrize("T,H,I", Z.BLOCK + MORE)
def test_gated_block(cuda, T, H, I):
    import bmx
    ffn, w = block(cuda, H, I)
    dt = (torch.float16, torch.bfloat16)[T % 2]
    x = rand(cuda, T, H, dt=dt, seed=T)
    rows = bmx.ops.quantize_rows(x)
    y64, e = Q.block(values(rows), *w, 0, 0.0)
    y = ffn(x)
    R.check("y", y, y64, R.rounded(y64, e, dt))
    assert torch.equal(ffn(rows), y)
    base = torch.randn((T, H), device=cuda)
    out = ffn.add_to(base.clone(), x)
    want = base.double() + y64
    R.check("out", out, want, e + 2.0 ** -22 * (want.abs() + y64.abs()))
    for n in (1, 16, 70, 300):
        if n < T:
            assert torch.equal(ffn(x[T - n:]), y[T - n:]), n
            assert torch.equal(ffn.add_to(base[T - n:].clone(), x[T - n:]), out[T - n:]), n


@pytest.mark.parametrize("act,L", [(0, 7.0), (1, 0.0), (1, 7.0), (2, 10.0), (3, 0.0), (3, 7.0)])
def test_a_tokens_result_does_not_depend_on_the_others(cuda, act, L):
    ffn, _ = block(cuda, 1032, 520, act, L)
    x = rand(cuda, 1500, 1032, dt=torch.bfloat16, seed=act)
    y = ffn(x)
    for n in (1, 16, 17, 70, 129, 300, 700):
        assert torch.equal(ffn(x[:n]), y[:n]), n
