"""GatedFFN where values are not finite: what NaN and infinite activations give, in the result and in the gradients."""
import pytest
import torch

import ffn_ref as R

pytestmark = pytest.mark.gpu


def tensors(cuda, T, H, I, dt=torch.bfloat16, seed=1):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    n = lambda *s: torch.randn(s, device=cuda, generator=g)
    return n(T, H).to(dt), [(n(a, b) / b ** 0.5).to(dt) for a, b in ((I, H), (I, H), (H, I))], n(T, H).to(dt)


def gradients(ffn, x, g, u, h, dy):
    """dx, dgate, dup, ddown of bmx_ffn_backward from the saved values given."""
    import bmx
    lib, d, T = bmx.lib(), ffn.desc(), x.shape[0]
    ws = torch.empty(lib.bmx_ffn_backward_workspace(d, T), dtype=torch.uint8, device=x.device)
    out = [torch.empty_like(t) for t in (x, ffn.gate, ffn.up, ffn.down)]
    bmx._lib.check(lib.bmx_ffn_backward(d, x.data_ptr(), T, bmx._lib.FfnSaved(g.data_ptr(), u.data_ptr(), h.data_ptr()),
                                        dy.data_ptr(), *(o.data_ptr() for o in out), ws.data_ptr(), ws.numel(),
                                        torch.cuda.current_stream().cuda_stream))
    return out


# the gradient epilogue behind whole sums, behind sums over splits of K, and in the launch shared with down's gradient
@pytest.mark.parametrize("T,H,I", [(5, 64, 72), (517, 2048, 768), (2050, 1032, 4104)])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("L", [0.0, 2.0])
def test_gradients_of_nan_activations(cuda, T, H, I, act, L):
    """g = NaN: both slopes are NaN. u = NaN: dh/dg is NaN, dh/du does not depend on u. Everything else keeps its bits."""
    import bmx
    x, w, dy = tensors(cuda, T, H, I)
    ffn = bmx.GatedFFN(*w, act=act, act_limit=L)
    keep = []
    ffn._forward(x, keep)
    _, g, u, h = keep
    t, j = T // 2, I // 3
    g[t, j] = u[t, j] = 0.5                      # inside every limit
    dx, dg, du, dd = gradients(ffn, x, g, u, h, dy)
    assert all(bool(v.isfinite().all()) for v in (dx, dg, du, dd))
    rows, units = torch.arange(T, device=cuda) != t, torch.arange(I, device=cuda) != j
    for bad in ("g", "u"):
        gb, ub = g.clone(), u.clone()
        (gb if bad == "g" else ub)[t, j] = float("nan")
        dxb, dgb, dub, ddb = gradients(ffn, x, gb, ub, h, dy)
        assert bool(dxb[t].isnan().all()) and torch.equal(dxb[rows], dx[rows])
        assert bool(dgb[j].isnan().all()) and torch.equal(dgb[units], dg[units])
        assert torch.equal(dub[units], du[units])
        assert bool(dub[j].isnan().all()) if bad == "g" else torch.equal(dub[j], du[j])
        assert torch.equal(ddb, dd)


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("L", [0.0, 2.0])
def test_nan_in_x_reaches_its_gradients(cuda, act, L):
    """A NaN in x, or in a row of a weight, is in every gradient that depends on it. (Where a clamp holds a, dh/dg is 0 whatever u
    is: those tokens' dx does not depend on up's row.)"""
    import bmx
    nan = float("nan")
    for T in (3, 90):
        x, w, dy = tensors(cuda, T, 136, 200)
        for bad in ("x", "gate", "up"):
            leaves = [v.clone() for v in [x] + w]
            if bad == "x":
                leaves[0][T // 2, 5] = nan
            else:
                leaves[1 if bad == "gate" else 2][7, 3] = nan
            for v in leaves:
                v.requires_grad_()
            y = bmx.GatedFFN(*leaves[1:], act=act, act_limit=L).forward(leaves[0])
            dx, dg, du, dd = torch.autograd.grad(y, leaves, dy)
            if bad == "x":
                assert bool(y[T // 2].isnan().all()) and bool(dx[T // 2].isnan().all())
                assert all(bool(v.isnan().all()) for v in (dg, du, dd))
            else:
                inside = torch.ones(T, dtype=torch.bool, device=cuda)
                if bad == "up" and L:
                    g = x.double() @ w[0][7].double()
                    inside = (g if act == 3 else R.act_a(act, g)) < 0.99 * L
                    assert bool(inside.any())
                assert bool(y.isnan().all()) and bool(dx[inside].isnan().all())
                assert bool(dg[7].isnan().all()) and bool(dd[:, 7].isnan().all())
                assert bool(du[7].isnan().all()) if bad == "gate" else bool(du.isfinite().all())
                assert bool(dg[8:].isfinite().all()) and bool(du[8:].isfinite().all())


@pytest.mark.parametrize("T", [3, 20, 90, 600])
def test_squared_relu_of_minus_infinity(cuda, T):
    """relu(g)^2 is 0 at g = -inf as at every other g below zero, with slopes of 0."""
    import bmx
    x, w, dy = tensors(cuda, T, 136, 200)
    x[:, 5] = 1.0
    for L in (0.0, 2.0):
        low = [v.clone() for v in w]
        low[0][7] = 0.0
        low[0][7, 5] = -1.0
        want = bmx.GatedFFN(*low, act=bmx.ACT_RELU2, act_limit=L).forward(x)
        low[0][7, 5] = float("-inf")
        ffn = bmx.GatedFFN(*low, act=bmx.ACT_RELU2, act_limit=L)
        assert torch.equal(ffn.forward(x), want) and bool(want.isfinite().all())
        keep = []
        ffn._forward(x, keep)
        _, g, u, h = keep
        assert bool((g[:, 7] == float("-inf")).all()) and bool((h[:, 7] == 0).all())
        # the slopes, with weights that are finite
        ffn = bmx.GatedFFN(*w, act=bmx.ACT_RELU2, act_limit=L)
        got = gradients(ffn, x, g, u, h, dy)
        g[:, 7] = -1.0
        for a, b in zip(got, gradients(ffn, x, g, u, h, dy)):
            assert bool(b.isfinite().all()) and torch.equal(a, b)


def test_replaced_weights(cuda):
    """Weights replaced between calls are the next call's, of whatever form; tensors that do not fit are refused before the
    kernels get their addresses, in the backward pass too. A 4-bit matrix is read-only."""
    import bmx
    x, w, dy = tensors(cuda, 5, 64, 72, torch.float16)
    _, w2, _ = tensors(cuda, 5, 64, 72, torch.float16, seed=2)
    ffn = bmx.GatedFFN(*(t.clone() for t in w))
    ffn.gate = w2[0]
    assert torch.equal(ffn.forward(x), bmx.GatedFFN(w2[0], *w[1:]).forward(x))
    ffn.up.data = w2[1]
    assert torch.equal(ffn.forward(x), bmx.GatedFFN(*w2[:2], w[2]).forward(x))
    out = torch.zeros((5, 64), device=cuda)
    for bad in (w[0].t(), w[0][:64].contiguous(), w[0].bfloat16(), w[0].cpu(), w[0].view(-1)[1:].clone()):
        ffn.up = bad
        with pytest.raises(ValueError):
            ffn.forward(x)
        with pytest.raises(ValueError):
            ffn.add_to(out, x)
    ffn.up = torch.nn.Parameter(w[1].clone())
    y = ffn.forward(x)
    ffn.up.data = w[1][:64].clone()
    with pytest.raises((ValueError, RuntimeError)):
        torch.autograd.grad(y, ffn.up, dy)
    with pytest.raises(ValueError):
        ffn.forward(x)
    q = [bmx.Q4Matrix.quantize(torch.randn(n, k, device=cuda).half(), 64) for n, k in ((128, 64), (128, 64), (64, 128), (128, 64))]
    ffn = bmx.GatedFFN(*q[:3])
    ffn.forward(x)
    ffn.gate = q[3]
    assert torch.equal(ffn.forward(x), bmx.GatedFFN(q[3], q[1], q[2]).forward(x))
    with pytest.raises(AttributeError):
        q[0].codes = q[3].codes
    with pytest.raises(AttributeError):
        q[0].N = 64


def test_forward_mode_is_refused_and_compiled_programs_call_the_kernels(cuda):
    import torch.autograd.forward_ad as fw
    import bmx
    x, w, _ = tensors(cuda, 5, 64, 72, torch.float16)
    ffn, q = bmx.GatedFFN(*w), bmx.Q4Matrix.quantize(w[0], 64)
    with fw.dual_level():
        for f in (ffn.forward, lambda v: bmx.ops.q4_linear(v, q)):
            with pytest.raises(ValueError):
                f(fw.make_dual(x, torch.ones_like(x)))
            assert f(x).shape[0] == 5                # no tangent: an ordinary call
        dual = bmx.GatedFFN(w[0], fw.make_dual(w[1], torch.ones_like(w[1])), w[2])
        with pytest.raises(ValueError):
            dual.forward(x)
        with pytest.raises(ValueError):
            dual.add_to(torch.zeros((5, 64), device=cuda), x)
    program = torch.compile(lambda v: (ffn.forward(v * 2), bmx.ops.q4_linear(v * 2, q)), backend="eager")
    for k in range(3):
        v = x + k
        for a, b in zip(program(v), (ffn.forward(v * 2), bmx.ops.q4_linear(v * 2, q))):
            assert torch.equal(a, b)


def test_the_added_form_has_no_gradients(cuda):
    """Nor has a layer that uses it: a block whose weights require grad is refused there unless autograd is off, and x is
    detached by whoever wants the layer's output alone."""
    import bmx
    x, w, _ = tensors(cuda, 5, 256, 72, torch.float16)
    plain = bmx.GatedFFN(*w)
    ffn = bmx.GatedFFN(*(torch.nn.Parameter(t.clone()) for t in w))
    tab = bmx.ExpertTable.random(256, 128, 16, (bmx.TF_K3,) * 3, seed=2, device=cuda)
    lg = torch.randn((5, 16), device=cuda).half()
    want = bmx.MoELayer(tab, 4, shared_ffn=plain).forward(x, lg)
    layer = bmx.MoELayer(tab, 4, shared_ffn=ffn)
    with pytest.raises(ValueError, match="no gradients"):
        layer.forward(x, lg)
    with torch.no_grad():
        assert torch.equal(layer.forward(x, lg), want)
    for t in (ffn.gate, ffn.up, ffn.down):
        t.requires_grad_(False)
    assert torch.equal(layer.forward(x, lg), want)
    ffn.down.requires_grad_()
    with pytest.raises(ValueError, match="no gradients"):
        ffn.add_to(torch.zeros((5, 256), device=cuda), x)


@pytest.mark.parametrize("shape", [(6,), (6, 64), (2, 3, 64), (64,)])
def test_the_result_may_be_changed_in_place(cuda, shape):
    """As any tensor that autograd records, whatever the leading dimensions: a residual added to y, then its gradients."""
    import bmx
    shape = shape if shape[-1] == 64 else (*shape, 64)
    _, w, _ = tensors(cuda, 5, 64, 72, torch.float16)
    x = torch.randn(shape, device=cuda).half().requires_grad_()
    w = [t.requires_grad_() for t in w]
    ffn, dy = bmx.GatedFFN(*w), torch.randn(shape, device=cuda).half()
    y = ffn.forward(x)
    want = torch.autograd.grad(y + x, [x] + w, dy)
    y = ffn.forward(x)
    before = y.detach().clone()
    y += x
    assert y.shape == x.shape and torch.equal(y, before + x)
    for a, b in zip(torch.autograd.grad(y, [x] + w, dy), want):
        assert torch.equal(a, b)


def test_a_layer_refuses_before_its_work(cuda):
    """A gate vector that the block cannot take is refused with the layer, a weight that requires grad before a step is taken
    on the slot table."""
    import bmx
    x, w, _ = tensors(cuda, 5, 256, 72, torch.float16)
    tab = bmx.ExpertTable.random(256, 128, 16, (bmx.TF_K3,) * 3, seed=2, device=cuda)
    ffn, odd = bmx.GatedFFN(*w), torch.zeros(257, dtype=torch.float16, device=cuda)[1:]
    for vec in (odd, odd.clone().cpu(), odd.float(), odd[:128]):
        with pytest.raises(ValueError):
            bmx.MoELayer(tab, 4, shared_ffn=ffn, shared_gate=vec)
    slots = bmx.ExpertSlots([tab], 8, maxj=4)
    layer = bmx.MoELayer(tab, 4, shared_ffn=ffn, slots=slots)
    lg = torch.randn((1, 16), device=cuda).half()
    steps = list(slots.seq)
    ffn.up.requires_grad_()
    for f in (lambda: layer.forward(x[:1], lg), lambda: layer.run_bszN(x[:1], torch.zeros((1, 4), dtype=torch.int64, device=cuda), x[:1, :4])):
        with pytest.raises(ValueError, match="no gradients"):
            f()
    assert list(slots.seq) == steps and layer.out_bszn is None
    with torch.no_grad():
        layer.forward(x[:1], lg)


def test_saved_values_elsewhere(cuda):
    """Recomputed (checkpoint), kept in host memory, used twice (retain_graph), accumulated into .grad: the plain gradients' bits."""
    import torch.utils.checkpoint as C
    import bmx
    x, w, dy = tensors(cuda, 90, 136, 264, torch.float16)
    leaves = [t.requires_grad_() for t in [x] + w]
    ffn = bmx.GatedFFN(*w)
    want = torch.autograd.grad(ffn.forward(x), leaves, dy)
    same = lambda got: all(torch.equal(a, b) for a, b in zip(got, want))
    for reentrant in (False, True):
        y = C.checkpoint(ffn.forward, x, use_reentrant=reentrant)
        y.backward(dy)
        assert same([t.grad for t in leaves])
        for t in leaves:
            t.grad = None
    with torch.autograd.graph.save_on_cpu():
        y = ffn.forward(x)
    assert same(torch.autograd.grad(y, leaves, dy))
    y = ffn.forward(x)
    assert same(torch.autograd.grad(y, leaves, dy, retain_graph=True)) and same(torch.autograd.grad(y, leaves, dy))
    # two blocks on the same weights, one behind the other
    z = bmx.GatedFFN(*w).forward(ffn.forward(x))
    a = torch.autograd.grad(z, w, dy)
    mid = ffn.forward(x)
    parts = torch.autograd.grad(ffn.forward(mid.detach().requires_grad_()), w, dy)
    m = mid.detach().requires_grad_()
    dm, = torch.autograd.grad(ffn.forward(m), m, dy)
    for got, p, q in zip(a, parts, torch.autograd.grad(mid, w, dm)):
        assert torch.equal(got, p + q)
    with torch.inference_mode():
        assert torch.equal(ffn.forward(x), mid)


def test_copies(cuda):
    """A copied block has weights of its own, also one that has been called; a 4-bit matrix takes attributes of the user's."""
    import copy
    import bmx
    x, w, _ = tensors(cuda, 5, 64, 72, torch.float16)
    ffn = bmx.GatedFFN(*w)
    want = ffn.forward(x)
    other = copy.deepcopy(ffn)
    assert torch.equal(other.forward(x), want) and other.gate.data_ptr() != ffn.gate.data_ptr()
    with torch.no_grad():
        ffn.down.zero_()
    assert torch.equal(other.forward(x), want) and not bool(ffn.forward(x).any())
    q = bmx.Q4Matrix.quantize(w[0], 64)
    q.name = "gate_proj"
    q.name = "up_proj"
    assert q.name == "up_proj"
