"""Host-side checks of the norm's and the 8-bit products' entry points: refused before any GPU work, with the reason."""
import ctypes

import pytest
import torch


def q8(**k):
    import bmx
    v = dict(N=72, K=128, codes=256, scale=256)
    v.update(k)
    return bmx._lib.Q8(*(v[n] for n, _ in bmx._lib.Q8._fields_))


@pytest.mark.parametrize("bad,text", [(dict(N=0), b"N (0)"), (dict(N=-1), b"N (-1)"), (dict(N=(1 << 24) + 1), b"2^24"), (dict(K=0), b"131071"),
                                      (dict(K=131072), b"131071"), (dict(codes=None), b"null"), (dict(scale=None), b"null"),
                                      (dict(codes=264), b"aligned"), (dict(scale=258), b"aligned")])
def test_matrix_refusals(bad, text):
    import bmx
    L, E = bmx.lib(), bmx._lib.BMX_ERR_ARG
    q = q8(**bad)
    assert L.bmx_q8_quantize(256, 0, q, None) == E and text in L.bmx_last_error()
    assert L.bmx_q8_dequant(q, 0, 256, None) == E and text in L.bmx_last_error()
    assert L.bmx_q8_pack(q, 256, None) == E and text in L.bmx_last_error()
    assert L.bmx_q8_unpack(q, 256, None) == E and text in L.bmx_last_error()
    assert L.bmx_q8_linear_workspace(q, 100) == 0 and text in L.bmx_last_error()
    assert L.bmx_q8_linear(q, 0, 256, None, 4, 256, 256, 1 << 30, None) == E and text in L.bmx_last_error()
    # as rows of a call
    w = q8(N=64, K=128)
    assert L.bmx_q8_linear(w, 0, None, q, 72, 256, 256, 1 << 30, None) == E
    ok = q8(N=128)
    for three in ((q, ok, ok), (ok, q, ok), (ok, ok, q)):
        d = bmx._lib.Ffn8Desc(0, 0, 0.0, 0, *(ctypes.pointer(m) for m in three))
        assert L.bmx_ffn8_workspace(d, 4) == 0
        assert L.bmx_ffn8_forward(d, 256, None, 4, 256, 256, 1 << 30, None) == E


def test_product_call_refusals():
    import bmx
    L, E, W = bmx.lib(), bmx._lib.BMX_ERR_ARG, bmx._lib.BMX_ERR_WORKSPACE
    q, rows = q8(), q8(N=40)
    for dt in (3, -1):
        assert L.bmx_q8_quantize(256, dt, q, None) == E and L.bmx_q8_dequant(q, dt, 256, None) == E
    assert L.bmx_q8_quantize(None, 0, q, None) == E and L.bmx_q8_quantize(257, 0, q, None) == E and L.bmx_q8_quantize(258, 2, q, None) == E
    assert L.bmx_q8_dequant(q, 0, None, None) == E and L.bmx_q8_dequant(q, 0, 264, None) == E
    assert L.bmx_q8_dequant(q8(N=1 << 24, K=131071), 0, 256, None) == E and b"too many" in L.bmx_last_error()
    assert L.bmx_q8_pack(q, None, None) == E and L.bmx_q8_unpack(q, None, None) == E
    assert L.bmx_q8_code_bytes(72, 128) == 80 * 128 and L.bmx_q8_code_bytes(1, 1) == 1024 and L.bmx_q8_code_bytes(0, 1) == 0
    lin = lambda dt=0, x=256, r=None, T=40, y=256, ws=256, n=1 << 30: L.bmx_q8_linear(q, dt, x, r, T, y, ws, n, None)
    assert lin(dt=2) == E and lin(x=None) == E and lin(r=rows) == E and lin(x=264) == E and lin(y=None) == E and lin(y=264) == E
    assert lin(T=-1) == E and lin(T=(1 << 24) + 1) == E and lin(T=0, x=None, y=None, ws=None, n=0) == 0
    assert lin(x=None, r=q8(N=41)) == E and lin(x=None, r=q8(N=40, K=120)) == E
    need = L.bmx_q8_linear_workspace(q, 40)
    assert need >= 40 * 128 and lin(n=need - 1) == W and lin(ws=None) == E and lin(ws=264) == E
    assert L.bmx_q8_linear_workspace(q, -1) == 0 and L.bmx_q8_linear_workspace(q, 0) == 0

    three = lambda a, b, c, **k: bmx._lib.Ffn8Desc(k.get("dtype", 0), k.get("act", 0), k.get("limit", 0.0), 0, *map(ctypes.pointer, (a, b, c)))
    gu, dn = q8(N=72, K=128), q8(N=128, K=72)
    good = three(gu, gu, dn)
    need = L.bmx_ffn8_workspace(good, 4)
    assert need >= 4 * 72 * 4
    for d, text in ((three(gu, dn, dn), b"[I, H]"), (three(gu, gu, gu), b"[I, H]"),
                    (three(gu, gu, dn, dtype=2), b"dtype"), (three(gu, gu, dn, act=4), b"activation"), (three(gu, gu, dn, limit=-1.0), b"act_limit"),
                    (three(gu, gu, dn, limit=float("nan")), b"act_limit"), (three(q8(N=72, K=124), q8(N=72, K=124), q8(N=124, K=72)), b"multiples of 8"),
                    (None, b"null")):
        assert L.bmx_ffn8_workspace(d, 4) == 0 and text in L.bmx_last_error()
        assert L.bmx_ffn8_forward(d, 256, None, 4, 256, 256, 1 << 30, None) == E and text in L.bmx_last_error()
        assert L.bmx_ffn8_add(d, 256, None, 4, None, 256, 256, 1 << 30, None) == E and text in L.bmx_last_error()
    r4 = q8(N=4)
    fwd = lambda x=256, r=None, T=4, y=256, ws=256, n=need: L.bmx_ffn8_forward(good, x, r, T, y, ws, n, None)
    assert fwd(x=None) == E and fwd(x=264) == E and fwd(y=None) == E and fwd(y=264) == E and fwd(ws=None) == E and fwd(ws=264) == E
    assert fwd(n=need - 1) == W and fwd(T=-1) == E and fwd(T=(1 << 24) + 1) == E and fwd(r=q8(N=5)) == E and fwd(T=0, x=None, y=None, ws=None, n=0) == 0
    add = lambda x=256, r=None, T=4, v=None, o=256, ws=256, n=need: L.bmx_ffn8_add(good, x, r, T, v, o, ws, n, None)
    assert add(x=None) == E and add(o=None) == E and add(o=264) == E and add(v=264) == E and add(x=None, r=r4, v=256) == E and add(n=need - 1) == W
    assert add(T=0, x=None, o=None, ws=None, n=0) == 0


def norm(**k):
    import bmx
    v = dict(H=64, dtype=0, x_dtype=0, residual_dtype=2, weight_dtype=0, eps=1e-6, weight=256)
    v.update(k)
    return bmx._lib.NormDesc(*(v[n] for n, _ in bmx._lib.NormDesc._fields_))


@pytest.mark.parametrize("bad,text", [(dict(H=0), b"multiple of 8"), (dict(H=60), b"multiple of 8"), (dict(H=16392), b"16384"), (dict(dtype=2), b"dtype 2"),
                                      (dict(dtype=-1), b"dtype"), (dict(x_dtype=1), b"of dtype or fp32"), (dict(residual_dtype=1), b"of dtype or fp32"),
                                      (dict(weight_dtype=3), b"of dtype or fp32"), (dict(eps=0.0), b"eps"), (dict(eps=float("nan")), b"eps"),
                                      (dict(weight=None), b"weight"), (dict(weight=264), b"weight")])
def test_norm_descriptor_refusals(bad, text):
    import bmx
    L, E = bmx.lib(), bmx._lib.BMX_ERR_ARG
    d = norm(**bad)
    assert L.bmx_rms_norm(d, 256, None, 4, None, 256, None, None) == E and text in L.bmx_last_error()
    assert L.bmx_rms_norm_backward_workspace(d, 4) == 0 and text in L.bmx_last_error()
    assert L.bmx_rms_norm_backward(d, 256, 0, 4, 256, None, 256, None, 256, 256, 1 << 30, None) == E and text in L.bmx_last_error()


def test_norm_call_refusals():
    import bmx
    L, E, W = bmx.lib(), bmx._lib.BMX_ERR_ARG, bmx._lib.BMX_ERR_WORKSPACE
    d = norm()
    rows = q8(N=4, K=64)
    fwd = lambda x=256, res=None, T=4, r=None, y=256, rows=None: L.bmx_rms_norm(d, x, res, T, r, y, rows, None)
    assert fwd(x=None) == E and fwd(x=264) == E and fwd(res=256) == E and fwd(r=256) == E and fwd(res=264, r=256) == E and fwd(res=256, r=264) == E
    assert fwd(y=None) == E and fwd(y=264) == E and fwd(T=-1) == E and fwd(T=(1 << 24) + 1) == E and fwd(T=0, x=None, y=None) == 0
    assert fwd(rows=q8(N=3, K=64)) == E and fwd(rows=q8(N=4, K=56)) == E
    need = L.bmx_rms_norm_backward_workspace(d, 1000)
    assert need >= 512 * 64 * 4 and rows.N == 4
    back = lambda v=256, s=1, T=1000, dy=256, dr=None, dx=256, ds=None, dw=256, ws=256, n=need: L.bmx_rms_norm_backward(
        d, v, s, T, dy, dr, dx, ds, dw, ws, n, None)
    assert back(v=None) == E and back(v=264) == E and back(dy=None) == E and back(dy=264) == E and back(dr=264) == E and back(dx=264) == E
    assert back(ds=264) == E and back(dw=264) == E and back(s=0, dr=256) == E and back(s=0, ds=256) == E and back(ws=None) == E and back(ws=264) == E
    assert back(n=need - 1) == W and back(T=-1) == E and back(dx=None, dw=None, ws=None, n=0) == 0
    assert back(T=0, v=None, dy=None, dw=None, ws=None, n=0) == 0


def test_host_tensors_are_refused():
    import bmx
    w = torch.ones(64, dtype=torch.float16)
    with pytest.raises(ValueError):
        bmx.RMSNorm(w)
    with pytest.raises(ValueError):
        bmx.Q8Matrix(torch.zeros((4, 64), dtype=torch.int8), torch.ones(4))
    with pytest.raises(ValueError):
        bmx.Q8Matrix.quantize(w.view(1, 64))
    with pytest.raises(ValueError):
        bmx.Rows8(torch.zeros((4, 64), dtype=torch.int8), torch.ones(4))
    with pytest.raises(ValueError):
        bmx.ops.quantize_rows(w)


def test_struct_sizes_are_the_headers():
    """The ctypes structs have the header's layout (natural alignment, 64-bit pointers)."""
    import bmx
    L = bmx._lib
    assert ctypes.sizeof(L.Q8) == 24 and L.Q8.codes.offset == 8 and L.Q8.scale.offset == 16
    assert ctypes.sizeof(L.Ffn8Desc) == 40 and L.Ffn8Desc.gate.offset == 16
    assert ctypes.sizeof(L.NormDesc) == 32 and L.NormDesc.weight.offset == 24
