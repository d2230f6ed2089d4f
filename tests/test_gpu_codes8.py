"""Codes of rows of 16 bits next to the borders between two codes: every pair of significands of a value and its row's largest, over the
differences of their exponents at which a code is not 0, in both kernels that quantize."""
import pytest
import torch

from test_gpu_q8 import check_quantized

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,bits", [(torch.float16, 10), (torch.bfloat16, 7)])
def test_every_pair_of_significands(cuda, dt, bits):
    """v = a 2^-d, top = b: 127 v / top is at least 2^-(11 + d) from a border that it does not lie on (2^-12 for d = 0): 2^-18.99 for
    a = 2047, b = 2031, d = 8. In 64 bits the quotient is off by 2^-53 of itself, so that the comparison knows each code."""
    import bmx
    a = torch.arange(1 << bits, 2 << bits, device=cuda).double()
    # (fp16: times 16, so that the smallest values have all their digits)
    top = a * 16.0
    v = torch.cat([top * 2.0 ** -d for d in range(10)])
    v[1::2] *= -1.0
    x = torch.cat((top[:, None], torch.where(v.abs() <= top[:, None], v, torch.zeros_like(v))), 1)
    for K in (x.shape[1], x.shape[1] // 8 * 8):             # an odd length, and a multiple of 8
        rows = x[:, x.shape[1] - K:].clone()
        rows[:, 0] = top
        assert torch.equal(rows.to(dt).double(), rows)
        check_quantized(bmx.ops.quantize_rows(rows.to(dt)), rows.to(dt))
