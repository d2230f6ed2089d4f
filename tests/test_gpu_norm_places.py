"""The norm in place: the sum on the residual or on x, y on x, with the bits of a call into buffers of their own."""
import pytest
import torch

from test_gpu_norm import make

pytestmark = pytest.mark.gpu
F32 = torch.float32


@pytest.mark.parametrize("T,H", [(1, 4096), (3, 136), (700, 2056), (2100, 520), (260, 8200)])
@pytest.mark.parametrize("x32,r32", [(False, False), (True, True), (True, False), (False, True)])
def test_in_place(cuda, T, H, x32, r32):
    import bmx
    dt = torch.float16
    x, res, w = make(cuda, T, H, dt, x32, r32, seed=T)
    norm = bmx.RMSNorm(w)
    y, r = norm(x, res)
    alone = norm(x)
    lib, check = bmx.lib(), bmx._lib.check
    stream = torch.cuda.current_stream().cuda_stream
    d = norm._desc(x.dtype, res.dtype)

    def call(x, res, total, out):
        check(lib.bmx_rms_norm(d, x.data_ptr(), None if res is None else res.data_ptr(), T, None if total is None else total.data_ptr(),
                               out.data_ptr(), None, stream), "bmx_rms_norm")

    out, a = torch.empty_like(y), res.clone()
    call(x, a, a, out)
    assert torch.equal(out, y) and torch.equal(a, r)
    if x.dtype == res.dtype:
        out, a = torch.empty_like(y), x.clone()
        call(a, res, a, out)
        assert torch.equal(out, y) and torch.equal(a, r)
    if not x32:
        a, total = x.clone(), torch.empty_like(res)
        call(a, res, total, a)
        assert torch.equal(a, y) and torch.equal(total, r)
        a, b = x.clone(), res.clone()
        call(a, b, b, a)
        assert torch.equal(a, y) and torch.equal(b, r)
        a = x.clone()
        call(a, None, None, a)
        assert torch.equal(a, alone)
