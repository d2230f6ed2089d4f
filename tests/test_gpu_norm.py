"""RMSNorm on the GPU: forward, 8-bit rows, gradients, streams and graphs, against the formulas in 64 bits with bounds from the number
of roundings (tests/rows8_ref.py)."""
import pytest
import torch

import ffn_ref as R
import rows8_ref as Q

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
F32 = torch.float32
SIZES = [(1, 8), (2, 24), (3, 512), (1, 520), (5, 1000), (4, 2048), (7, 2056), (1, 4096), (3, 4104), (2, 5120), (33, 768), (513, 136), (2, 8192),
         (3, 8200), (2, 11008), (1, 16384), (2049, 64), (2050, 2048), (2051, 2064), (2052, 5120)]


def make(cuda, T, H, dt, x32=False, r32=False, w32=False, seed=1):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    n = lambda *s: torch.randn(s, device=cuda, generator=g)
    x = (n(T, H) * torch.exp(n(H))).to(F32 if x32 else dt)
    return x, (3.0 * n(T, H)).to(F32 if r32 else dt), (1.0 + 0.3 * n(H)).to(F32 if w32 else dt)


def check_y(y, v, w, eps, dt):
    y64, e = Q.norm(v.double(), w.double(), eps)
    R.check("y", y, y64, R.rounded(y64, e, dt))
    return y64, e


def check_rows(rows, y64, e):
    """Each value at most half a scale off, the scales off by what rstd is, the largest code 127, zeros behind the row."""
    top = y64.abs().amax(1)
    scale = rows.scale.double()
    assert bool(((scale - top / 127).abs() <= top / 127 * (Q.RSTD + 4 * Q.STEP)).all())
    codes = rows.int8().double()
    assert bool((codes.abs().amax(1) == 127).all())
    R.check("rows", codes * scale[:, None], y64, scale[:, None] * (0.5 + 127 * 3 * Q.STEP) + e + y64.abs() * 3 * Q.STEP)
    b = rows.codes.view(-1, (rows.K + 63) // 64, 4, 16, 16)         # nothing but zeros behind a row: chunks of 16 columns, of 16 rows each
    assert int((b != 0).sum((1, 2, 4)).view(-1)[:rows.N].sum()) == int((codes != 0).sum())


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H", SIZES)
def test_forward(cuda, T, H, dt):
    import bmx
    dt = DT[dt]
    x, res, w = make(cuda, T, H, dt, seed=H)
    n = bmx.RMSNorm(w)
    y, r = n(x, res)
    assert torch.equal(r, (x.float() + res.float()).to(dt)) and y.dtype == dt
    check_y(y, r, w, 1e-6, dt)
    check_y(n(x), x, w, 1e-6, dt)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("x32,r32,w32", [(a, b, c) for a in (False, True) for b in (False, True) for c in (False, True)])
def test_types(cuda, x32, r32, w32, dt):
    import bmx
    for T, H in ((3, 136), (2100, 72), (2, 4104)):
        x, res, w = make(cuda, T, H, DT[dt], x32, r32, w32, seed=T)
        n = bmx.RMSNorm(w, eps=1e-5, dtype=DT[dt])
        y, rows, r = n.both(x, res)
        assert r.dtype == res.dtype and torch.equal(r, (x.float() + res.float()).to(res.dtype))
        y64, e = check_y(y, r, w, 1e-5, DT[dt])
        check_rows(rows, y64, e)
        y1, r1 = n(x, res)
        rows2, r2 = n.rows8(x, res)
        assert torch.equal(y1, y) and torch.equal(r1, r) and torch.equal(r2, r)
        assert torch.equal(rows2.int8(), rows.int8()) and torch.equal(rows2.scale, rows.scale)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H", SIZES)
def test_rows(cuda, T, H, dt):
    import bmx
    x, res, w = make(cuda, T, H, DT[dt], seed=T + H)
    n = bmx.RMSNorm(w)
    rows, r = n.rows8(x, res)
    check_rows(rows, *Q.norm(r.double(), w.double(), 1e-6))
    rows = n.rows8(x)
    check_rows(rows, *Q.norm(x.double(), w.double(), 1e-6))
    assert rows.shape == x.shape and rows.dtype == x.dtype
    # what the codes stand for
    assert torch.equal(rows.dequant(F32), rows.int8().float() * rows.scale[:, None])


def backward_check(cuda, T, H, dt, x32=False, r32=False, w32=False, residual=True, seed=3, use="both"):
    import bmx
    x, res, w = make(cuda, T, H, dt, x32, r32, w32, seed)
    g = torch.Generator(device=cuda)
    g.manual_seed(seed + 50)
    dy = torch.randn((T, H), device=cuda, generator=g).to(dt)
    dr = torch.randn((T, H), device=cuda, generator=g).to(res.dtype)
    leaves = [x, res, w] if residual else [x, w]
    for t in leaves:
        t.requires_grad_()
    n = bmx.RMSNorm(w, dtype=dt)
    if residual:
        y, r = n(x, res)
        outs, given = {"both": ((y, r), (dy, dr)), "y": ((y,), (dy,)), "r": ((r,), (dr,))}[use]
    else:
        y, r = n(x), x.detach()
        outs, given = (y,), (dy,)
    got = torch.autograd.grad(outs, leaves, given)
    assert [t.dtype for t in got] == [t.dtype for t in leaves]
    with_dr = residual and use != "y"
    dv, ev, dw, ew = Q.norm_grads(r.detach().double(), w.detach().double(), 1e-6, dy.double() * (use != "r"), dr.double() if with_dr else None)
    last = lambda v, e, t: R.rounded(v, e, t) if t in R.HALF else e + 2.0 ** -149
    for name, a in (("dx", got[0]), ("dres", got[1])) if residual else (("dx", got[0]),):
        R.check(name, a, dv, last(dv, ev, a.dtype))
    R.check("dw", got[-1], dw, last(dw, ew, w.dtype))


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H", SIZES + [(600, 4096), (1100, 520), (1030, 8200), (300, 16384), (4200, 64)])
def test_gradients(cuda, T, H, dt):
    backward_check(cuda, T, H, DT[dt], seed=T + H)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("x32,r32,w32", [(a, b, c) for a in (False, True) for b in (False, True) for c in (False, True)])
def test_gradients_of_types(cuda, x32, r32, w32, dt):
    backward_check(cuda, 21, 136, DT[dt], x32, r32, w32)
    backward_check(cuda, 21, 136, DT[dt], x32, r32, w32, residual=False)


@pytest.mark.parametrize("x32,r32,w32", [(True, False, False), (False, True, False), (False, False, True), (True, True, True)])
@pytest.mark.parametrize("T,H", [(600, 8456), (1100, 4104)])
def test_gradients_of_types_over_several_rows_a_workgroup(cuda, T, H, x32, r32, w32):
    backward_check(cuda, T, H, torch.bfloat16, x32, r32, w32)
    backward_check(cuda, T, H, torch.float16, x32, r32, w32, residual=False)


@pytest.mark.parametrize("use", ["y", "r"])
def test_gradients_of_one_output(cuda, use):
    backward_check(cuda, 37, 264, torch.float16, use=use)
    backward_check(cuda, 37, 264, torch.bfloat16, x32=True, use=use)


def test_wanted_gradients_only(cuda):
    """Each subset of the inputs gets the gradients that all of them together get."""
    import bmx
    for x32 in (False, True):
        leaves = list(make(cuda, 13, 72, torch.bfloat16, x32))
        dy, dr = (torch.randn((13, 72), device=cuda).bfloat16() for _ in range(2))
        for t in leaves:
            t.requires_grad_()
        every = torch.autograd.grad(bmx.RMSNorm(leaves[2], dtype=torch.bfloat16)(*leaves[:2]), leaves, (dy, dr))
        for mask in range(1, 8):
            for i, t in enumerate(leaves):
                t.requires_grad_(bool(mask >> i & 1))
            some = [t for t in leaves if t.requires_grad]
            got = iter(torch.autograd.grad(bmx.RMSNorm(leaves[2], dtype=torch.bfloat16)(*leaves[:2]), some, (dy, dr)))
            for i in range(3):
                if mask >> i & 1:
                    assert torch.equal(next(got), every[i]), (mask, i)


def test_gradients_against_differences(cuda):
    """fp32 x, residual and weight, y and the gradient of y in fp16: along a direction the loss changes as the gradients say. y enters the
    loss through dy, so that its formula in 64 bits is what is differenced; nothing is rounded to 16 bits, and a gradient's own roundings
    in fp32 (at most some 100 steps of 2^-23 of its terms, which are up to five times as large together) stay below 2^-14 of it."""
    import bmx
    x, res, w = make(cuda, 9, 200, torch.float16, True, True, True)
    dy = torch.randn((9, 200), device=cuda).half()
    dr = torch.randn((9, 200), device=cuda)
    leaves = [t.requires_grad_() for t in (x, res, w)]
    got = torch.autograd.grad(bmx.RMSNorm(w, dtype=torch.float16)(x, res), leaves, (dy, dr))

    def loss(x, res, w):
        v = x + res
        return float((Q.norm(v, w, 1e-6)[0] * dy.double()).sum() + (v * dr.double()).sum())

    at = [t.detach().double() for t in leaves]
    for i, t in enumerate(at):
        d = torch.randn_like(t)
        step = lambda s: [a + (s * d if j == i else 0) for j, a in enumerate(at)]
        quotient = (loss(*step(1e-5)) - loss(*step(-1e-5))) / 2e-5
        assert abs(float((got[i].double() * d).sum()) - quotient) <= 2.0 ** -14 * float(got[i].double().norm() * d.norm())


def test_one_tensor_twice(cuda):
    """x as its own residual: v = 2 x, and x gets both gradients."""
    import bmx
    x, _, w = make(cuda, 6, 64, torch.float16)
    x.requires_grad_()
    y, r = bmx.RMSNorm(w)(x, x)
    assert torch.equal(r.detach(), x.detach() * 2)
    dy = torch.randn((6, 64), device=cuda).half()
    got, = torch.autograd.grad(y, x, dy)
    one, = torch.autograd.grad(bmx.RMSNorm(w)(v := r.detach().requires_grad_()), v, dy)
    assert torch.equal(got, one + one)


def test_strides_shapes_and_no_tokens(cuda):
    import bmx
    x, res, w = make(cuda, 24, 136, torch.float16)
    n = bmx.RMSNorm(w)
    y, r = n(x, res)
    y3, r3 = n(x.view(2, 3, 4, 136), res.view(2, 3, 4, 136))
    assert y3.shape == (2, 3, 4, 136) and torch.equal(y3.view(24, 136), y) and torch.equal(r3.view(24, 136), r)
    # transposed tokens, rows of a wider tensor, a start that is not 16-byte aligned
    y4, r4 = n(x.view(4, 6, 136).transpose(0, 1), res.view(4, 6, 136).transpose(0, 1))
    assert torch.equal(y4.transpose(0, 1).reshape(24, 136), y) and torch.equal(r4.transpose(0, 1).reshape(24, 136), r)
    wide = torch.randn((24, 150), device=cuda).half()
    wide[:, 7:143] = x
    assert torch.equal(n(wide[:, 7:143], res)[0], y)
    flat = torch.empty(24 * 136 + 3, device=cuda, dtype=torch.float16)
    off = flat[3:].view(24, 136).copy_(x)
    rows, r5 = n.rows8(off, res)
    assert torch.equal(r5, r) and torch.equal(rows.int8(), n.rows8(x, res)[0].int8())
    y1 = n(x[0], res[0])[0]
    assert y1.shape == (136,) and torch.equal(y1, y[0])
    # none
    e = x[:0].requires_grad_()
    w.requires_grad_()
    ye, re = n(e, res[:0])
    assert ye.shape == re.shape == (0, 136)
    de, dw = torch.autograd.grad(ye, [e, w], torch.empty_like(ye))
    assert de.shape == (0, 136) and not bool(dw.any())
    with torch.no_grad():
        assert n.rows8(e).shape == (0, 136)


@pytest.mark.parametrize("dt", sorted(DT))
def test_zeros_infinities_and_nan(cuda, dt):
    """A row's zeros, infinities and NaN stay its own."""
    import bmx
    for T in (6, 2060):
        x, res, w = make(cuda, T, 264, DT[dt])
        clean, _ = bmx.RMSNorm(w)(x, res)
        crows, _ = bmx.RMSNorm(w).rows8(x, res)
        x[1], res[1] = 0.0, 0.0
        x[2, 5], x[3, 100], x[4, 263] = float("inf"), float("nan"), float("-inf")
        y, rows, r = bmx.RMSNorm(w).both(x, res)
        keep = [0] + list(range(5, T))
        assert torch.equal(y[keep], clean[keep]) and torch.equal(rows.int8()[keep], crows.int8()[keep]) and torch.equal(rows.scale[keep], crows.scale[keep])
        assert not bool(y[1].any()) and not bool(rows.int8()[1:5].any()) and float(rows.scale[1]) == 0.0
        v = r.float()
        want = v[2:5] * w.float() / torch.sqrt((v[2:5] ** 2).mean(1, keepdim=True) + 1e-6)
        assert torch.equal(y[2:5].isnan(), want.isnan()) and bool((y[2][:5] == 0).all()) and bool(y[2, 5].isnan()) and bool(y[3].isnan().all())
        assert bool(rows.scale[2:5].isnan().all())


def test_largest_and_smallest_values(cuda):
    """fp32 rows: squares past fp32's range make rstd 0; rows below 2^-110 are zeros in 8 bits and normal in 16."""
    import bmx
    w = torch.ones(64, device=cuda)
    n = bmx.RMSNorm(w, eps=1e-6, dtype=torch.bfloat16)
    x = torch.randn((4, 64), device=cuda)
    x[0] *= 1e25
    x[1] *= 1e-35
    x[2] *= 1e-30
    y, rows = n.both(x)
    assert not bool(y[0].any()) and float(rows.scale[0]) == 0.0
    assert not bool(rows.int8()[1].any()) and float(rows.scale[1]) == 0.0
    for i in (2, 3):
        y64, e = Q.norm(x[i:i + 1].double(), w.double(), 1e-6)
        R.check("y", y[i:i + 1], y64, R.rounded(y64, e, torch.bfloat16))
        assert int(rows.int8()[i].abs().max()) == 127


def test_streams_and_graph(cuda):
    """On another stream, two calls at once, captured and replayed with other inputs in the same places."""
    import bmx
    x, res, w = make(cuda, 300, 2048, torch.float16)
    x2, res2, _ = make(cuda, 300, 2048, torch.float16, seed=9)
    n = bmx.RMSNorm(w)
    want, want2 = n.both(x, res), n.both(x2, res2)
    same = lambda a, b: torch.equal(a[0], b[0]) and torch.equal(a[1].int8(), b[1].int8()) and torch.equal(a[1].scale, b[1].scale) and torch.equal(a[2], b[2])
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = n.both(x, res)
        with torch.cuda.stream(s2):
            b = n.both(x2, res2)
        torch.cuda.synchronize()
        assert same(a, want) and same(b, want2)
    gx, gr = x.clone(), res.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = n.both(gx, gr)
    for i in range(4):
        src = ((x, res), (x2, res2))[i % 2]
        gx.copy_(src[0])
        gr.copy_(src[1])
        g.replay()
        n.both(x2, res2)
        torch.cuda.synchronize()
        assert same(out, (want, want2)[i % 2])


def test_captured_training_step(cuda):
    """Forward and gradients in one graph, replayed between eager passes, give the eager results."""
    import bmx
    for T in (5, 700):
        x, res, w = (t.requires_grad_() for t in make(cuda, T, 1032, torch.bfloat16))
        dy, dr = (torch.randn((T, 1032), device=cuda).bfloat16() for _ in range(2))
        n = bmx.RMSNorm(w)

        def step():
            y, r = n(x, res)
            return (y, r) + torch.autograd.grad((y, r), [x, res, w], (dy, dr))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [t.detach().clone() for t in step()]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        for _ in range(3):
            for t in out:
                t.detach().fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a.detach(), b) for a, b in zip(out, want))


def test_more_than_2_to_31_values(cuda):
    """Rows whose values lie past 2^31: the last ones as they are alone."""
    import bmx
    T, H = 140000, 16384
    w = torch.randn(H, device=cuda).half()
    n = bmx.RMSNorm(w)
    x = torch.empty((T, H), device=cuda, dtype=torch.float16)
    x[-3:] = torch.randn((3, H), device=cuda).half()
    x[:-3] = 1.0
    y, rows, r = n.both(x, x)
    want, wrows, wr = n.both(x[-3:].clone(), x[-3:].clone())
    assert torch.equal(y[-3:], want) and torch.equal(rows.int8()[-3:], wrows.int8()) and torch.equal(rows.scale[-3:], wrows.scale)
    assert torch.equal(r[-3:], wr)
    del y, rows
    xg = r.requires_grad_()
    dy = x
    got, = torch.autograd.grad(n(xg), xg, dy)
    one = r.detach()[-3:].clone().requires_grad_()
    assert torch.equal(got[-3:], torch.autograd.grad(n(one), one, dy[-3:])[0])


def test_replaced_weight_and_options(cuda):
    """Weights and options replaced since the last call are checked and used."""
    import copy
    import bmx
    x, res, w = make(cuda, 4, 128, torch.float16)
    n = bmx.RMSNorm(w)
    n(x)
    n.weight = w * 2
    assert torch.equal(n(x), bmx.RMSNorm(w * 2)(x))
    n.eps = 0.5
    assert torch.equal(n(x), bmx.RMSNorm(w * 2, eps=0.5)(x))
    n.weight.data = w[:64].clone()
    with pytest.raises(ValueError):
        n(x)
    assert n(x[:, :64].contiguous()).shape == (4, 64)
    m = copy.deepcopy(n)
    n.weight.data.zero_()
    assert bool(m(x[:, :64].contiguous()).any())
    n.eps = 0.0
    with pytest.raises(ValueError, match="eps"):
        n(x[:, :64])


def test_refusals(cuda):
    import bmx
    x, res, w = make(cuda, 4, 64, torch.float16)
    for bad in (w[:60].clone(), w.cpu(), w.view(1, 64), w.long(), torch.ones(128, device=cuda).half()[::2], w[:0], torch.ones(16392, device=cuda).half()):
        with pytest.raises(ValueError):
            bmx.RMSNorm(bad)
    for kw in (dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=1e-60), dict(eps=float("inf")), dict(dtype=torch.bfloat16), dict(dtype=F32)):
        with pytest.raises(ValueError):
            bmx.RMSNorm(w, **kw)
    with pytest.raises(ValueError):
        bmx.RMSNorm(w.float())
    n = bmx.RMSNorm(w)
    for args in ((x.cpu(),), (x.bfloat16(),), (x[:, :56],), (x, res[:3]), (x, res.bfloat16()), (x, res.cpu()), (x, res.view(2, 2, 64)), (x.double(),)):
        with pytest.raises(ValueError):
            n(*args)
    x.requires_grad_()
    for f in (n.rows8, n.both):
        with pytest.raises(ValueError, match="no gradients"):
            f(x)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x.detach(), x.detach())
        with pytest.raises(ValueError, match="forward-mode"):
            n(d)
    with torch.no_grad():
        n.rows8(x)
    y, r = n(x, res)
    r.add_(1)                                          # what the backward pass needs
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y.sum(), x)
