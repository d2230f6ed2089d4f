"""GatedFFN on the GPU (16-bit weights): forward, gradients, the added form, streams, graphs and refusals, against the block
in 64 bits with bounds from the number of roundings (tests/ffn_ref.py)."""
import ctypes

import pytest
import torch

import ffn_ref as R

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = [(1, 8, 8), (2, 24, 40), (15, 64, 64), (16, 136, 72), (17, 200, 264), (33, 256, 128), (63, 128, 520), (64, 520, 136),
         (65, 1032, 328), (77, 2048, 768), (127, 72, 1000), (130, 264, 200), (257, 512, 256), (300, 1288, 1032)]


def make(cuda, T, H, I, dt, seed=1, spread=1.0):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    n = lambda *s: torch.randn(s, device=cuda, generator=g)
    x = n(T, H).to(dt)
    w = [(n(a, b) * spread / b ** 0.5).to(dt) for a, b in ((I, H), (I, H), (H, I))]
    return x, w, n(T, H).to(dt)


def check_forward(x, w, act, L, ffn, y, keep=None):
    dt = x.dtype
    g, u, h, eg, eu, eh = R.forward(x.double(), *(t.double() for t in w[:2]), act, L)
    if keep is not None:
        _, gs, us, hs = keep
        R.check("g", gs, g, eg + R.TINY[torch.bfloat16])
        R.check("u", us, u, eu + R.TINY[torch.bfloat16])
        R.check("h", hs, h, R.rounded(h, eh, dt))
    y64, ey = R.product(h, w[2].double(), R.rounded(h, eh, dt))
    R.check("y", y, y64, R.rounded(y64, ey, dt))
    return y64, ey


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I", SIZES)
def test_forward(cuda, T, H, I, dt):
    import bmx
    x, w, _ = make(cuda, T, H, I, DT[dt], seed=T)
    act = (T + H) % 4
    L = 1.25 if T % 2 else 0.0
    ffn = bmx.GatedFFN(*w, act=act, act_limit=L)
    check_forward(x, w, act, L, ffn, ffn.forward(x))


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("L", [0.0, 0.7, 7.0])
def test_activations_and_clamps(cuda, act, L, dt):
    import bmx
    for T in (5, 90):
        x, w, _ = make(cuda, T, 96, 104, DT[dt], seed=act, spread=3.0)
        ffn = bmx.GatedFFN(*w, act=act, act_limit=L)
        keep = []
        check_forward(x, w, act, L, ffn, ffn._forward(x, keep), keep)


def backward_check(cuda, T, H, I, dt, act, L, seed=3):
    """Each gradient from the saved values the forward pass left (checked above), within its roundings."""
    import bmx
    x, w, dy = make(cuda, T, H, I, dt, seed=seed)
    ffn = bmx.GatedFFN(*w, act=act, act_limit=L)
    keep = []
    check_forward(x, w, act, L, ffn, ffn._forward(x, keep), keep)
    for t in [x] + w:
        t.requires_grad_()
    y = ffn.forward(x)
    dx, dwg, dwu, dwd = torch.autograd.grad(y, [x] + w, dy)
    x, w = x.detach().double(), [t.detach().double() for t in w]
    dy = dy.double()
    _, gs, us, hs = [t.double() for t in keep]
    hg, hu = R.act_grads(act, gs, us, L)
    dh, edh = R.product(dy, w[2].t().contiguous())
    # the slopes are sums of terms that may cancel: their error goes by the terms' size
    size = R.act_a(act, gs).abs() + 1.0 + gs.abs()
    dg, du = dh * hg, dh * hu
    edg = R.rounded(dg, edh * hg.abs() + R.act_err(act, gs) * dh.abs() * (us.abs() + 1.0) * (1.0 + size), dt)
    edu = R.rounded(du, edh * hu.abs() + R.act_err(act, gs) * dh.abs() * size, dt)
    a, ea = R.product(dg, w[0].t().contiguous(), edg)
    b, eb = R.product(du, w[1].t().contiguous(), edu)
    R.check("dx", dx, a + b, R.rounded(a + b, ea + eb + R.ACC * (a.abs() + b.abs()), dt))
    for name, got, d, e in (("dgate", dwg, dg, edg), ("dup", dwu, du, edu)):
        want, ew = R.product(d.t().contiguous(), x.t().contiguous(), e.t())
        R.check(name, got, want, R.rounded(want, ew, dt))
    want, ew = R.product(dy.t().contiguous(), hs.t().contiguous())
    R.check("ddown", dwd, want, R.rounded(want, ew, dt))


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I", SIZES)
def test_gradients(cuda, T, H, I, dt):
    backward_check(cuda, T, H, I, DT[dt], (T + I) % 4, 1.25 if T % 2 else 0.0)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("act", [0, 1, 2, 3])
def test_gradients_of_activations(cuda, act, dt):
    for L in (0.0, 0.7):
        backward_check(cuda, 37, 128, 200, DT[dt], act, L, seed=act)


# the 256-row tiles: enough of them to fill the chip, ragged at both ends
@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I", [(2050, 72, 3016), (70, 2568, 2600), (4100, 3208, 264)])
def test_large_tiles(cuda, T, H, I, dt):
    backward_check(cuda, T, H, I, DT[dt], 0, 0.0)


@pytest.mark.parametrize("act,L", [(0, 0.0), (1, 2.0), (2, 0.0), (3, 2.0)])
def test_gradients_against_autograd_and_differences(cuda, act, L):
    """End to end in 64 bits. Norms: h, dg, du and the result are each off by at most half a step (2^-11) of themselves (g and
    u are kept in fp32): 16 halves are more than all together."""
    import bmx
    x, w, dy = make(cuda, 70, 96, 136, torch.float16, seed=7)
    leaves = [t.double().requires_grad_() for t in [x] + w]

    def loss(x, wg, wu, wd):
        return (R.act_h(act, x @ wg.t(), x @ wu.t(), L) @ wd.t() * dy.double()).sum()

    want = torch.autograd.grad(loss(*leaves), leaves)
    for t in [x] + w:
        t.requires_grad_()
    got = torch.autograd.grad(bmx.GatedFFN(*w, act=act, act_limit=L).forward(x), [x] + w, dy)
    g = torch.Generator(device=cuda)
    g.manual_seed(11)
    for i, (a, b) in enumerate(zip(got, want)):
        assert float((a.double() - b).norm()) <= 16 * 2.0 ** -11 * float(b.norm()), i
        # along one direction, difference quotient in 64 bits (step 1e-5: its own error is of order 1e-10)
        v = torch.randn(a.shape, device=cuda, generator=g, dtype=torch.float64)
        at = lambda s: [t.detach() + (s * v if j == i else 0) for j, t in enumerate(leaves)]
        quotient = float(loss(*at(1e-5)) - loss(*at(-1e-5))) / 2e-5
        assert abs(float((a.double() * v).sum()) - quotient) <= 16 * 2.0 ** -11 * float(b.norm() * v.norm())


def test_wanted_gradients_only(cuda):
    """Each subset of the inputs gets the gradients that all of them together get."""
    import bmx
    x, w, dy = make(cuda, 21, 64, 88, torch.bfloat16)
    leaves = [x] + w
    for t in leaves:
        t.requires_grad_()
    all_of = torch.autograd.grad(bmx.GatedFFN(*w).forward(x), leaves, dy)
    for mask in range(1, 16):
        for i, t in enumerate(leaves):
            t.requires_grad_(bool(mask >> i & 1))
        some = [t for t in leaves if t.requires_grad]
        got = iter(torch.autograd.grad(bmx.GatedFFN(*w).forward(x), some, dy))
        for i, want in enumerate(all_of):
            if mask >> i & 1:
                assert torch.equal(next(got), want), (mask, i)


def test_no_tokens(cuda):
    import bmx
    x, w, _ = make(cuda, 4, 64, 72, torch.float16)
    ffn = bmx.GatedFFN(*w)
    assert ffn.forward(x[:0]).shape == (0, 64)
    out = torch.ones((0, 64), device=cuda)
    assert ffn.add_to(out, x[:0]) is out
    empty = x[:0].clone().requires_grad_()
    for t in w:
        t.requires_grad_()
    y = ffn.forward(empty)
    grads = torch.autograd.grad(y, [empty] + w, torch.empty_like(y))
    assert grads[0].shape == (0, 64) and all(bool((g == 0).all()) for g in grads[1:])


def test_layouts_of_x(cuda):
    """Leading dimensions, strided rows, a transposed view, an odd offset, an expanded gradient: the results of the plain rows."""
    import bmx
    x, w, dy = make(cuda, 24, 64, 72, torch.float16)
    ffn = bmx.GatedFFN(*w)
    want = ffn.forward(x)
    assert torch.equal(ffn.forward(x.view(2, 3, 4, 64)).view(24, 64), want)
    wide = torch.zeros((24, 200), dtype=x.dtype, device=cuda)
    wide[:, 3:67] = x
    assert torch.equal(ffn.forward(wide[:, 3:67]), want)
    assert torch.equal(ffn.forward(x.t().contiguous().t()), want)
    odd = torch.zeros(24 * 64 + 1, dtype=x.dtype, device=cuda)
    odd[1:] = x.reshape(-1)
    assert torch.equal(ffn.forward(odd[1:].view(24, 64)), want)
    assert torch.equal(ffn.forward(x[5]), ffn.forward(x[5:6])[0])
    x.requires_grad_()
    a, = torch.autograd.grad(ffn.forward(x).sum(), x)
    b, = torch.autograd.grad(ffn.forward(x), x, torch.ones_like(x))
    assert torch.equal(a, b)
    x3 = x.detach().view(2, 12, 64).requires_grad_()
    c, = torch.autograd.grad(ffn.forward(x3), x3, dy.view(2, 12, 64))
    d, = torch.autograd.grad(ffn.forward(x), x, dy)
    assert torch.equal(c.view(24, 64), d)


@pytest.mark.parametrize("T", [3, 40, 300])
def test_nan_and_infinity_stay_in_their_rows(cuda, T):
    import bmx
    x, w, dy = make(cuda, T, 136, 200, torch.bfloat16)
    ffn = bmx.GatedFFN(*w, act_limit=2.0)
    want = ffn.forward(x)
    bad = x.clone()
    bad[T // 2, 5] = float("nan")
    bad[0, 0] = float("inf")
    y = ffn.forward(bad)
    assert bool(torch.isnan(y[T // 2]).all())
    rows = [t for t in range(T) if t not in (0, T // 2)]
    assert torch.equal(y[rows], want[rows])
    x.requires_grad_()
    bdy = dy.clone()
    bdy[T // 2, 7] = float("nan")
    a, = torch.autograd.grad(ffn.forward(x), x, dy)
    b, = torch.autograd.grad(ffn.forward(x), x, bdy)
    rows = [t for t in range(T) if t != T // 2]
    assert bool(torch.isnan(b[T // 2]).any()) and torch.equal(a[rows], b[rows])


@pytest.mark.parametrize("T", [1, 20, 100, 600])
def test_added_form_and_rows_behind(cuda, T):
    """bmx_ffn_add on a larger buffer: the rows behind the last token keep their bits; with and without the gate vector."""
    import bmx
    x, w, _ = make(cuda, T, 264, 136, torch.float16)
    ffn = bmx.GatedFFN(*w)
    g, u, h, _, _, eh = R.forward(x.double(), w[0].double(), w[1].double(), 0, 0.0)
    y64, ey = R.product(h, w[2].double(), R.rounded(h, eh, x.dtype))
    for vec in (None, (torch.randn(264, device=cuda) / 16).half()):
        base = torch.randn((T + 3, 264), device=cuda)
        out = base.clone()
        assert ffn.add_to(out[:T], x, vec).data_ptr() == out.data_ptr()
        s = torch.ones((T, 1), dtype=torch.float64, device=cuda) if vec is None else torch.sigmoid(x.double() @ vec.double())[:, None]
        want = base[:T].double() + s * y64
        # the sum's two roundings, and the gate's fp32 dot and sigmoid
        bound = s * ey + 2.0 ** -22 * (want.abs() + y64.abs()) + 264 * R.ACC * y64.abs()
        R.check("out", out[:T], want, bound)
        assert torch.equal(out[T:], base[T:])
    lib, d = bmx.lib(), ffn.desc()
    y = torch.full((T + 2, 264), 7.0, dtype=torch.float16, device=cuda)
    ws = torch.empty(lib.bmx_ffn_workspace(d, T), dtype=torch.uint8, device=cuda)
    s = torch.cuda.current_stream().cuda_stream
    bmx._lib.check(lib.bmx_ffn_forward(d, x.data_ptr(), T, y.data_ptr(), None, ws.data_ptr(), ws.numel(), s))
    assert torch.equal(y[:T], ffn.forward(x)) and bool((y[T:] == 7.0).all())
    # a workspace one byte short is refused before anything runs
    assert lib.bmx_ffn_forward(d, x.data_ptr(), T, y.data_ptr(), None, ws.data_ptr(), ws.numel() - 1, s) == bmx._lib.BMX_ERR_WORKSPACE


@pytest.mark.parametrize("T", [2, 90])
def test_streams_and_graphs(cuda, T):
    """Two calls at once on two streams, and captured forward and gradient passes replayed with new inputs between eager
    calls, give the eager results' bits."""
    import bmx
    x, w, dy = make(cuda, T, 136, 264, torch.bfloat16)
    ffn = bmx.GatedFFN(*w)
    want = ffn.forward(x)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append([ffn.forward(x) for _ in range(4)])
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(o, want) for os in outs for o in os)

    sx, sdy = x.clone().requires_grad_(), dy.clone()
    ws = [t.clone().requires_grad_() for t in w]
    gffn = bmx.GatedFFN(*ws)

    def step():
        y = gffn.forward(sx)
        return (y.detach(),) + torch.autograd.grad(y, [sx] + ws, sdy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caught = step()
    with torch.cuda.graph(graph2):
        caught2 = step()
    for k in range(4):
        with torch.no_grad():
            sx.copy_(torch.randn_like(x) * (k + 1))
            sdy.copy_(torch.randn_like(dy))
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        eager = step()
        for a, b, c in zip(caught, caught2, eager):
            assert torch.equal(a, c) and torch.equal(b, c)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", [1, 9, 300])
def test_as_a_layers_shared_expert(cuda, T, gated):
    """MoELayer(shared_ffn=...): the routed experts' output plus the block, through every call form; no table of its own
    shared expert."""
    import bmx
    H, I, E = 256, 128, 16
    tab = bmx.ExpertTable.random(H, I, E, (bmx.TF_K3,) * 3, seed=2, device=cuda)
    x, w, _ = make(cuda, T, H, 200, torch.float16)
    ffn = bmx.GatedFFN(*w)
    vec = (torch.randn(H, device=cuda) / 16).half() if gated else None
    lg = torch.randn((T, E), device=cuda).half()
    plain = bmx.MoELayer(tab, 4)
    both = bmx.MoELayer(tab, 4, shared_ffn=ffn, shared_gate=vec)
    want = ffn.add_to(plain.forward(x, lg).clone(), x, vec)
    assert torch.equal(both.forward(x, lg), want) and torch.equal(both.out_bszn, want)
    sel, rw = both.routing_fn(T, None, x, {"logits": lg})
    want = ffn.add_to(plain.run_bszN(x, sel, rw).clone(), x, vec)
    assert torch.equal(both.run_bszN(x, sel, rw), want)
    slots = bmx.ExpertSlots([tab], 8, maxj=4)
    a = bmx.MoELayer(tab, 4, shared_ffn=ffn, shared_gate=vec, slots=slots)
    got = a.forward(x, lg)
    assert float((got - want).abs().max()) < 1e-2
    with pytest.raises(ValueError):
        bmx.MoELayer(bmx.ExpertTable.random(H, I, E, (bmx.TF_K3,) * 3, shared=True, device=cuda), 4, shared_ffn=ffn)
    with pytest.raises(ValueError):
        bmx.MoELayer(tab, 4, shared_ffn=bmx.GatedFFN(*(t.bfloat16() for t in w)))


def test_refusals(cuda):
    import bmx
    x, w, dy = make(cuda, 4, 64, 72, torch.float16)
    g, u, d = w
    with pytest.raises(ValueError):
        bmx.GatedFFN(g, u, d.t())
    with pytest.raises(ValueError):
        bmx.GatedFFN(g, u[:, :56].contiguous(), d)
    with pytest.raises(ValueError):
        bmx.GatedFFN(g.float(), u.float(), d.float())
    with pytest.raises(ValueError):
        bmx.GatedFFN(g, u.bfloat16(), d)
    with pytest.raises(ValueError):
        bmx.GatedFFN(g.cpu(), u.cpu(), d.cpu())
    with pytest.raises(ValueError):
        bmx.GatedFFN(g[:, :60].contiguous(), u[:, :60].contiguous(), d[:60].contiguous())
    with pytest.raises(ValueError):
        bmx.GatedFFN(g, u, d, act=4)
    for L in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            bmx.GatedFFN(g, u, d, act_limit=L)
    ffn = bmx.GatedFFN(g, u, d)
    for bad in (x.float(), x.bfloat16(), x.cpu(), x[:, :56]):
        with pytest.raises(ValueError):
            ffn.forward(bad)
    with pytest.raises(ValueError):
        ffn.add_to(torch.zeros((4, 64), device=cuda, dtype=torch.float16), x)
    with pytest.raises(ValueError):
        ffn.add_to(torch.zeros((5, 64), device=cuda), x)
    with pytest.raises(ValueError):
        ffn.add_to(torch.zeros((4, 64), device=cuda), x, torch.zeros(64, device=cuda))
    # a weight changed in place between the passes: autograd refuses the backward pass
    g.requires_grad_()
    y = ffn.forward(x)
    with torch.no_grad():
        u.mul_(2.0)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, g, dy)


# every tile shape and split count that the planner chooses: few and many rows against long and short K
@pytest.mark.parametrize("T,H,I", [(100, 2048, 64), (100, 64, 2048), (517, 768, 512), (700, 1032, 1160), (300, 4104, 520),
                                   (1100, 1544, 776), (90, 4096, 4096), (2050, 1024, 3848), (2050, 7696, 512)])
def test_tile_plans(cuda, T, H, I):
    backward_check(cuda, T, H, I, torch.float16, 0, 0.0)


@pytest.mark.parametrize("T,H,I", [(4100, 4104, 1032), (4100, 1032, 5200)])
def test_products_in_two_parts(cuda, T, H, I):
    """Whole rounds of large tiles and the rest on smaller ones: y and dx by rows of H, then h, dg and du by rows of I; the
    added form's sums are those that y rounds."""
    import bmx
    backward_check(cuda, T, H, I, torch.bfloat16, 0, 0.0)
    x, w, _ = make(cuda, T, H, I, torch.bfloat16)
    ffn = bmx.GatedFFN(*w)
    out = ffn.add_to(torch.zeros((T, H), device=cuda), x)
    assert torch.equal(out.to(x.dtype), ffn.forward(x))


def test_one_tensor_as_gate_and_up(cuda):
    """Its gradient is the sum of the two."""
    import bmx
    x, w, dy = make(cuda, 40, 72, 136, torch.float16)
    for t in w:
        t.requires_grad_()
    one, = torch.autograd.grad(bmx.GatedFFN(w[0], w[0], w[2]).forward(x), [w[0]], dy)
    other = w[0].detach().clone().requires_grad_()
    a, b = torch.autograd.grad(bmx.GatedFFN(w[0], other, w[2]).forward(x), [w[0], other], dy)
    assert torch.equal(one, a + b)
    both = bmx.GatedFFN(w[0], w[0], w[2]).forward(x)
    both.backward(dy)
    assert torch.equal(w[0].grad, one)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I", [(2050, 1032, 4104), (3100, 2056, 2568)])
def test_down_gradient_beside_dh(cuda, T, H, I, dt):
    """Sizes at which down's gradient and dh share a launch; each wanted alone is the same sums in the same order."""
    import bmx
    backward_check(cuda, T, H, I, DT[dt], 1, 0.0)
    x, w, dy = make(cuda, T, H, I, DT[dt])
    for t in [x] + w:
        t.requires_grad_()
    y = bmx.GatedFFN(*w).forward(x)
    all_of = torch.autograd.grad(y, [x] + w, dy, retain_graph=True)
    some = [torch.autograd.grad(bmx.GatedFFN(*w[:2], w[2].detach()).forward(x), [x] + w[:2], dy),
            torch.autograd.grad(bmx.GatedFFN(w[0].detach(), w[1].detach(), w[2]).forward(x.detach()), [w[2]], dy)]
    for got, want in zip(some[0] + some[1], all_of):
        assert torch.equal(got, want)


@pytest.mark.parametrize("T,H,I", [(100, 520, 4096), (90, 4096, 2048), (300, 1032, 2056), (700, 520, 264), (20, 5120, 2304), (40, 776, 264)])
def test_added_form_is_y_before_its_rounding(cuda, T, H, I):
    """Products with K split and not, and the kernel of few tokens: added to zeros and rounded, the sums are y."""
    import bmx
    x, w, _ = make(cuda, T, H, I, torch.bfloat16)
    ffn = bmx.GatedFFN(*w)
    y = ffn.forward(x)
    assert torch.equal(ffn.add_to(torch.zeros((T, H), device=cuda), x).to(x.dtype), y)
    check_forward(x, w, 0, 0.0, ffn, y)
