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


def q4(**k):
    import bmx
    v = dict(N=72, K=128, group=64, scale_dtype=0, codes=256, scale=256, zero=256)
    v.update(k)
    return bmx._lib.Q4(*(v[n] for n, _ in bmx._lib.Q4._fields_))


@pytest.mark.parametrize("bad,text", [(dict(group=48), b"group"), (dict(group=0), b"group"), (dict(N=0), b"positive"), (dict(K=96), b"multiple"),
                                      (dict(K=-64), b"positive"), (dict(N=1 << 21), b"2^20"), (dict(scale_dtype=3), b"scale dtype"),
                                      (dict(codes=None), b"null"), (dict(scale=None), b"null"), (dict(codes=264), b"aligned"),
                                      (dict(zero=8), b"aligned")])
def test_q4_matrix_refusals(bad, text):
    import bmx
    L, E = bmx.lib(), bmx._lib.BMX_ERR_ARG
    q = q4(**bad)
    assert L.bmx_q4_pack(q, 256, 256, 256, None) == E and text in L.bmx_last_error()
    assert L.bmx_q4_dequant(q, 0, 256, None) == E and text in L.bmx_last_error()
    assert L.bmx_q4_linear_workspace(q, 100) == 0 and text in L.bmx_last_error()
    assert L.bmx_q4_linear(q, 0, 256, 4, 256, 256, 1 << 30, None) == E and text in L.bmx_last_error()
    ok = q4(N=128, K=128)
    for three in ((q, ok, ok), (ok, q, ok), (ok, ok, q)):
        d = bmx._lib.Ffn4Desc(0, 0, 0.0, 0, *(ctypes.pointer(m) for m in three))
        assert L.bmx_ffn4_workspace(d, 4) == 0
        assert L.bmx_ffn4_forward(d, 256, 4, 256, 256, 1 << 30, None) == E


def test_q4_call_refusals():
    import bmx
    L, E, W = bmx.lib(), bmx._lib.BMX_ERR_ARG, bmx._lib.BMX_ERR_WORKSPACE
    q = q4()
    assert L.bmx_q4_code_bytes(72, 128) == 80 * 64 and L.bmx_q4_code_bytes(1, 32) == 16 * 64 and L.bmx_q4_code_bytes(0, 32) == 0
    assert L.bmx_q4_group_count(72, 128, 64) == 80 * 2 and L.bmx_q4_group_count(1, 32, 32) == 16 * 4 and L.bmx_q4_group_count(1, 32, 31) == 0
    assert L.bmx_q4_pack(q, None, 256, 256, None) == E and L.bmx_q4_pack(q, 256, None, 256, None) == E
    assert L.bmx_q4_pack(q, 256, 256, None, None) == E and L.bmx_q4_pack(q4(zero=None), 256, 256, 256, None) == E
    assert L.bmx_q4_dequant(q, 2, 256, None) == E and L.bmx_q4_dequant(q, 0, None, None) == E and L.bmx_q4_dequant(q, 0, 264, None) == E
    lin = lambda dt=0, x=256, T=4, y=256, ws=256, n=1 << 30: L.bmx_q4_linear(q, dt, x, T, y, ws, n, None)
    assert lin(dt=2) == E and lin(x=None) == E and lin(x=264) == E and lin(y=None) == E and lin(T=-1) == E
    assert lin(T=(1 << 24) + 1) == E and lin(T=0, x=None, y=None, ws=None, n=0) == 0
    need = L.bmx_q4_linear_workspace(q, 4096)
    assert need > 0 and lin(T=4096, n=need - 1) == W and lin(T=4096, ws=None) == E and lin(T=4096, ws=264) == E
    gu, dn = q4(N=128, K=64), q4(N=64, K=128)
    three = lambda a, b, c: bmx._lib.Ffn4Desc(0, 0, 0.0, 0, ctypes.pointer(a), ctypes.pointer(b), ctypes.pointer(c))
    good = three(gu, gu, dn)
    need = L.bmx_ffn4_workspace(good, 4)
    assert need > 0
    for bad in (three(gu, dn, dn), three(gu, gu, gu), three(gu, q4(N=128, K=64, group=32), dn)):
        assert L.bmx_ffn4_workspace(bad, 4) == 0
        assert L.bmx_ffn4_forward(bad, 256, 4, 256, 256, 1 << 30, None) == E
        assert L.bmx_ffn4_add(bad, 256, 4, None, 256, 256, 1 << 30, None) == E
    assert L.bmx_ffn4_forward(good, 256, 4, 256, 256, need - 1, None) == W
    assert L.bmx_ffn4_add(good, 256, 4, 258, 256, 256, need, None) == E
    assert L.bmx_ffn4_forward(None, 256, 4, 256, 256, need, None) == E


def test_workspaces_of_any_token_count():
    """The workspace queries plan on the host: no tokens and the most of them among the counts, each at least its largest part,
    never less for more tokens of one path."""
    import bmx
    L = bmx.lib()
    for H, I in ((8, 8), (64, 72), (4096, 2048), (4096, 11008), (1 << 20, 8), (8, 1 << 20)):
        d = desc(H=H, I=I)
        for T in (0, 1, 16, 17, 80, 81, 517, 4096, 100000, 1 << 24):
            assert L.bmx_ffn_workspace(d, T) >= T * I * 2 and L.bmx_ffn_backward_workspace(d, T) >= 2 * T * I * 2
    for N, K, G in ((1, 32, 32), (77, 4096, 128), (11008, 4096, 64), (1 << 20, 128, 128)):
        q = q4(N=N, K=K, group=G)
        for T in (0, 1, 16, 17, 80, 81, 517, 4096, 1 << 24):
            assert L.bmx_q4_linear_workspace(q, T) < 1 << 45
    gu, dn = q4(N=128, K=64), q4(N=64, K=128)
    d = bmx._lib.Ffn4Desc(0, 0, 0.0, 0, ctypes.pointer(gu), ctypes.pointer(gu), ctypes.pointer(dn))
    for T in (0, 1, 16, 17, 80, 81, 517, 1 << 24):
        assert L.bmx_ffn4_workspace(d, T) >= T * 128 * 2


def matrix(N, K, group=64):
    """What GatedFFN takes of a Q4Matrix, without a device."""
    import types
    return types.SimpleNamespace(N=N, K=K, group=group, device=torch.device("cpu"), struct=q4(N=N, K=K, group=group, codes=256 * N))


def test_replaced_4_bit_matrices_reach_the_next_call():
    """The descriptor is that of the matrices and options as they are, checked as the constructor checks them."""
    import bmx
    gate, up, down = matrix(128, 64), matrix(128, 64), matrix(64, 128)
    ffn = bmx.GatedFFN(gate, up, down)
    at = lambda p: ctypes.addressof(p.contents)
    d = ffn.desc(torch.float16)
    assert at(d.gate) == ctypes.addressof(gate.struct) and ffn.desc(torch.float16) is d
    other = matrix(128, 64)
    ffn.gate = other
    d = ffn.desc(torch.float16)
    assert at(d.gate) == ctypes.addressof(other.struct) and at(d.up) == ctypes.addressof(up.struct)
    ffn.act, ffn.act_limit = bmx.ACT_GELU, 2.0
    d = ffn.desc(torch.bfloat16)
    assert (d.act, d.act_limit) == (bmx.ACT_GELU, 2.0)
    for bad in (matrix(192, 64), matrix(128, 128), matrix(128, 64, group=32), torch.zeros(128, 64)):
        ffn.gate = bad
        for _ in range(2):
            with pytest.raises(ValueError):
                ffn.desc(torch.float16)
        with pytest.raises(ValueError):
            ffn.forward(torch.zeros((1, 64), dtype=torch.float16))
        with pytest.raises(ValueError):
            ffn.add_to(torch.zeros((1, 64)), torch.zeros((1, 64), dtype=torch.float16))
    ffn.gate, ffn.act = gate, 7
    with pytest.raises(ValueError):
        ffn.desc(torch.float16)
    # all three, of other sizes
    ffn.gate, ffn.up, ffn.down, ffn.act = matrix(192, 128), matrix(192, 128), matrix(128, 192), bmx.ACT_SILU
    ffn.desc(torch.float16)
    assert (ffn.hidden_size, ffn.intermediate_size) == (128, 192)


def test_forward_mode_and_tracing_are_refused():
    """Neither would see more than the output's allocation."""
    import torch.autograd.forward_ad as fw
    from torch.fx.experimental.proxy_tensor import make_fx
    import bmx
    ffn = bmx.GatedFFN(matrix(128, 64), matrix(128, 64), matrix(64, 128))
    x, out = torch.zeros((3, 64), dtype=torch.float16), torch.zeros((3, 64))
    calls = (lambda v: ffn.forward(v), lambda v: ffn.add_to(out, v), lambda v: bmx.ops.q4_linear(v, ffn.gate))
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for f in calls:
            with pytest.raises(ValueError, match="forward-mode"):
                f(d)
        with pytest.raises(ValueError, match="forward-mode"):
            ffn.add_to(fw.make_dual(out, torch.ones_like(out)), x)
        with pytest.raises(ValueError, match="forward-mode"):
            ffn.add_to(out, x, fw.make_dual(x[0], torch.ones_like(x[0])))
    for f in calls:
        with pytest.raises(ValueError, match="forward-mode"):
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f)(x)
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x,), check_trace=False)


def test_the_added_form_has_no_gradients():
    """Where autograd records it is refused, as the 4-bit block's forward pass: a leaf would train on nothing."""
    import bmx
    ffn = bmx.GatedFFN(matrix(128, 64), matrix(128, 64), matrix(64, 128))
    x, out, vec = torch.zeros((3, 64), dtype=torch.float16), torch.zeros((3, 64)), torch.zeros(64, dtype=torch.float16)
    leaf = lambda t: t.clone().requires_grad_()
    for a in ((leaf(out), x, vec), (out, leaf(x), vec), (out, x, leaf(vec)), (out, leaf(x), None)):
        with pytest.raises(ValueError, match="no gradients"):
            ffn.add_to(*a)
