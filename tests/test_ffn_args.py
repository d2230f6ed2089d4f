"""Host-side checks of the feed-forward block's entry points: refused before any GPU work, with the reason."""
import ctypes

import pytest
import torch


def desc(**k):
    import bmx
    v = dict(H=64, I=72, dtype=0, act=0, act_limit=0.0, reserved=0, gate=256, up=256, down=256)
    v.update(k)
    return bmx._lib.FfnDesc(*(v[n] for n, _ in bmx._lib.FfnDesc._fields_))


@pytest.mark.parametrize("bad,text", [(dict(H=60), b"multiples of 8"), (dict(I=0), b"multiples of 8"), (dict(I=-8), b"multiples"),
                                      (dict(H=1 << 21), b"2^20"), (dict(dtype=2), b"dtype"), (dict(act=4), b"activation"),
                                      (dict(act=-1), b"activation"), (dict(act_limit=-1.0), b"act_limit"),
                                      (dict(act_limit=float("nan")), b"act_limit"), (dict(gate=None), b"null weight"),
                                      (dict(down=264), b"aligned")])
def test_descriptor_refusals(bad, text):
    import bmx
    L, E = bmx.lib(), bmx._lib.BMX_ERR_ARG
    d = desc(**bad)
    assert L.bmx_ffn_workspace(d, 4) == 0 and text in L.bmx_last_error()
    assert L.bmx_ffn_backward_workspace(d, 4) == 0 and text in L.bmx_last_error()
    sv = bmx._lib.FfnSaved(256, 256, 256)
    assert L.bmx_ffn_forward(d, 256, 4, 256, None, 256, 1 << 30, None) == E and text in L.bmx_last_error()
    assert L.bmx_ffn_add(d, 256, 4, None, 256, 256, 1 << 30, None) == E and text in L.bmx_last_error()
    assert L.bmx_ffn_backward(d, 256, 4, sv, 256, 256, None, None, None, 256, 1 << 30, None) == E and text in L.bmx_last_error()


def test_call_refusals():
    import bmx
    L, E, W = bmx.lib(), bmx._lib.BMX_ERR_ARG, bmx._lib.BMX_ERR_WORKSPACE
    d = desc()
    need, nback = L.bmx_ffn_workspace(d, 4), L.bmx_ffn_backward_workspace(d, 4)
    assert need >= 4 * 72 * 2 and nback >= 2 * 4 * 72 * 2
    sv = bmx._lib.FfnSaved(256, 256, 256)
    fwd = lambda x=256, T=4, y=256, s=None, ws=256, n=need: L.bmx_ffn_forward(d, x, T, y, s, ws, n, None)
    assert fwd(x=None) == E and fwd(x=258) == E and fwd(y=None) == E and fwd(y=264) == E and fwd(T=-1) == E
    assert fwd(T=(1 << 24) + 1) == E and fwd(ws=None) == E and fwd(ws=260) == E and fwd(n=need - 1) == W
    assert fwd(s=bmx._lib.FfnSaved(256, None, 256)) == E and fwd(s=bmx._lib.FfnSaved(256, 264, 256)) == E
    assert fwd(T=0, x=None, y=None, ws=None, n=0) == 0
    add = lambda x=256, T=4, v=None, o=256, ws=256, n=need: L.bmx_ffn_add(d, x, T, v, o, ws, n, None)
    assert add(x=None) == E and add(o=None) == E and add(o=264) == E and add(v=258) == E and add(n=need - 1) == W
    assert add(T=0, x=None, o=None, ws=None, n=0) == 0
    back = lambda x=256, T=4, s=sv, dy=256, dx=256, g=256, u=256, w=256, ws=256, n=nback: L.bmx_ffn_backward(
        d, x, T, s, dy, dx, g, u, w, ws, n, None)
    assert back(x=None) == E and back(dy=None) == E and back(dy=264) == E and back(s=None) == E
    assert back(s=bmx._lib.FfnSaved(None, 256, 256)) == E and back(dx=260) == E and back(g=260) == E and back(u=264) == E
    assert back(w=258) == E and back(n=nback - 1) == W and back(T=-1) == E
    assert back(T=0, x=None, s=None, dy=None, dx=None, g=None, u=None, w=None, ws=None, n=0) == 0


def test_host_tensors_are_refused():
    import bmx
    w = [torch.zeros(s, dtype=torch.float16) for s in ((72, 64), (72, 64), (64, 72))]
    with pytest.raises(ValueError):
        bmx.GatedFFN(*w)
