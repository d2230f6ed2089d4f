"""The norm's eps has to be finite as the kernels get it: in fp32."""
import pytest
import torch

from test_norm_q8_args import norm


@pytest.mark.parametrize("eps", [float("inf"), 1e39])
def test_the_library_refuses_an_infinite_eps(eps):
    """1e39 is infinite in fp32, where 1 / sqrt(mean + eps) would be 0."""
    import bmx
    d = norm(eps=eps)
    L, E = bmx.lib(), bmx._lib.BMX_ERR_ARG
    assert L.bmx_rms_norm(d, 256, None, 4, None, 1 << 20, None, None) == E and b"eps" in L.bmx_last_error()
    assert L.bmx_rms_norm_backward_workspace(d, 4) == 0 and b"eps" in L.bmx_last_error()


@pytest.mark.gpu
def test_the_class_refuses_an_infinite_eps(cuda):
    import bmx
    w = torch.ones(64, device=cuda).bfloat16()
    with pytest.raises(ValueError, match="eps"):
        bmx.RMSNorm(w, eps=1e39)
    # the largest there is: y = v w / sqrt(mean + eps) far above bfloat16's smallest
    norm = bmx.RMSNorm(w, eps=2.0 ** 127)
    x = torch.full((2, 64), 2.0 ** 10, device=cuda).bfloat16()
    want = x.double() / (x.double() ** 2 + 2.0 ** 127).sqrt()
    assert bool(((norm(x).double() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -20)).all())
