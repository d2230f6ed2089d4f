"""The feed-forward block and the 4-bit matrices at the sizes of ffn_sizes.py, every value against 64 bits with bounds that an output
of zeros, a lost step of K or an exchanged row does not keep (sharp_ref.py, test_sharp_ref.py): each step from what the kernels kept
of the one before. And two calls at once, on streams and in graphs, of products whose partial sums lie in workspaces."""
import pytest
import torch

import ffn_ref as R
import ffn_sizes as Z
import sharp_ref as S

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def normal(cuda, seed, *shape):
    return torch.randn(shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed))


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,K,N,G", Z.LINEAR)
def test_4_bit_products(cuda, T, K, N, G, dt):
    import bmx
    for zero, sdt in ((T % 2 == 0, torch.float16), (T % 2 == 1, torch.bfloat16)):
        given, q64 = S.symmetric_codes(cuda, N, K, G, zero, sdt, seed=T)
        x = normal(cuda, T, T, K).to(DT[dt])
        # fp16 x keeps the digits of bf16 scales at any number of tokens: a smaller bound than the one used
        y64, e = S.q4_product(x.double(), q64, DT[dt], G)
        S.check("y", bmx.ops.q4_linear(x, bmx.Q4Matrix(*given, group=G)), y64, S.rounded(y64, e, DT[dt]))


def added(ffn, x, y64, e, name):
    """The added form on zeros, and on other values with the gate vector."""
    cuda, (T, H) = x.device, x.shape
    S.check(name, ffn.add_to(torch.zeros((T, H), device=cuda), x), y64, e)
    vec = (normal(cuda, 5, H) / H ** 0.5).to(x.dtype)
    base = normal(cuda, 6, T, H)
    dot, ed = S.product(x.double(), vec.double()[None])
    s = torch.sigmoid(dot)
    want = base.double() + s * y64
    # the dot's error through the sigmoid's slope of at most a quarter, the sigmoid's own few roundings, the sum's two
    S.check(name + ", gated", ffn.add_to(base.clone(), x, vec), want, s * e + (ed / 4 + 2.0 ** -21 * s) * y64.abs() + 2.0 ** -23 * want.abs())


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I,G", Z.BLOCK4)
def test_4_bit_blocks(cuda, T, H, I, G, dt):
    """(Activations whose h is symmetric as up's product is.)"""
    import bmx
    act, L = (T + H // 32) % 3, 1.25 if T % 2 else 0.0
    mats = [S.symmetric_codes(cuda, n, k, G, z, torch.float16, seed=s) for s, (n, k, z) in enumerate(((I, H, True), (I, H, False), (H, I, True)))]
    ffn = bmx.GatedFFN(*(bmx.Q4Matrix(*m[0], group=G) for m in mats), act=act, act_limit=L)
    x = normal(cuda, T, T, H).to(DT[dt])
    prod = lambda a, q: S.q4_product(a, q, DT[dt], G)
    _, _, h, _, _, eh = S.forward(x.double(), mats[0][1], mats[1][1], act, L, prod)
    y64, e = S.q4_product(h, mats[2][1], DT[dt], G, S.rounded(h, eh, DT[dt]))
    S.check("y", ffn.forward(x), y64, S.rounded(y64, e, DT[dt]))
    added(ffn, x, y64, e, "out")


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I", Z.BLOCK16)
def test_16_bit_blocks_and_their_gradients(cuda, T, H, I, dt):
    import bmx
    dt, act, L = DT[dt], (T + I // 8) % 3, 1.25 if T % 2 else 0.0
    x, dy = normal(cuda, T, T, H).to(dt), normal(cuda, T + 1, T, H).to(dt)
    w = [(normal(cuda, s, a, b) / b ** 0.5).to(dt) for s, (a, b) in enumerate(((I, H), (I, H), (H, I)))]
    ffn = bmx.GatedFFN(*w, act=act, act_limit=L)
    keep = []
    y = ffn._forward(x, keep)
    _, g, u, h = keep
    for name, got, m in (("g", g, w[0]), ("u", u, w[1])):
        S.check(name, got, *S.product(x.double(), m.double()))
    g, u, hs = g.double(), u.double(), h.double()
    h64 = S.act_h(act, g, u, L)
    slip = S.act_err(act, g)
    S.check("h", h, h64, S.rounded(h64, slip * (u.abs() + 1.0) * R.act_a(act, g).abs() + 2.0 ** -126 * g.abs() * (u.abs() + 1.0), dt))
    y64, e = S.product(hs, w[2].double())
    S.check("y", y, y64, S.rounded(y64, e, dt))
    assert torch.equal(ffn.forward(x), y)
    added(ffn, x, y64, e, "out")
    del y64, e, h64

    leaves = [x] + w
    for t in leaves:
        t.requires_grad_()
    dx, dwg, dwu, dwd = torch.autograd.grad(ffn.forward(x), leaves, dy)
    xs, ws, dys = x.detach().double(), [t.detach().double() for t in w], dy.double()
    S.check("ddown", dwd, *weight_gradient(dys, hs, 0.0, dt))
    hg, hu = R.act_grads(act, g, u, L)
    dh, edh = S.product(dys, ws[2].t().contiguous())
    size = R.act_a(act, g).abs() + 1.0 + g.abs()
    dg, du = dh * hg, dh * hu
    edg = S.rounded(dg, edh * hg.abs() + slip * dh.abs() * (u.abs() + 1.0) * (1.0 + size), dt)
    if L:
        # An a that is the clamp's value to fp32's digits (2^-24 of itself is one rounding of g^2 in the squared relu) may be on either
        # side of it: its slope is the one or the other. With 8 million values there are such, g^2 = 1.25 (1 + 3e-8) among them.
        a = R.act_a(act, g)
        at = (a - L).abs() <= slip * a.abs()
        edg = edg + torch.where(at, (dh * R.act_grads(act, g, u.clamp(-L, L), 0.0)[0]).abs(), torch.zeros_like(dh))
    edu = S.rounded(du, edh * hu.abs() + slip * dh.abs() * size, dt)
    S.check("dgate", dwg, *weight_gradient(dg, xs, edg, dt))
    S.check("dup", dwu, *weight_gradient(du, xs, edu, dt))
    a, ea = S.product(dg, ws[0].t().contiguous(), edg)
    b, eb = S.product(du, ws[1].t().contiguous(), edu)
    # one sum of 2 I products: each half's additions go on top of the other's
    n = S.SIGMAS * I * S.ACC * (((dg * dg) @ (ws[0] * ws[0])).sqrt() + ((du * du) @ (ws[1] * ws[1])).sqrt())
    S.check("dx", dx, a + b, S.rounded(a + b, ea + eb + n, dt))


def weight_gradient(d, v, ed, dt):
    """d^T v over the tokens, and its bound."""
    y, e = S.product(d.t().contiguous(), v.t().contiguous(), ed.t().contiguous() if torch.is_tensor(ed) else 0.0)
    return y, S.rounded(y, e, dt)


def twice(calls, inputs):
    """Every call on two streams at once and in two graphs, replayed with new inputs between eager calls: the eager bits."""
    want = [c() for c in calls]
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append([c() for c in calls])
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    for o in outs:
        for a, b in zip(o, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    torch.cuda.synchronize()
    graphs, caught = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            caught.append([c() for c in calls])
    for k in range(4):
        with torch.no_grad():
            for i, t in enumerate(inputs):
                t.copy_(normal(t.device, 100 * k + i, *t.shape))
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        eager = [c() for c in calls]
        for one in caught:
            for a, b in zip(one, eager):
                assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dt", sorted(DT))
def test_4_bit_products_in_parts_at_once(cuda, dt):
    """Slices, K split with and without group sums, decoded weights: each with a workspace."""
    import bmx
    for T, K, N, G in ((39, 7360, 73, 32), (77, 4096, 4096, 32), (300, 4096, 1000, 64), (1100, 1024, 520, 128)):
        q = bmx.Q4Matrix(*S.symmetric_codes(cuda, N, K, G, True, torch.float16, seed=1)[0], group=G)
        x = normal(cuda, 1, T, K).to(DT[dt])
        twice([lambda: (bmx.ops.q4_linear(x, q),)], [x])
    for T, H, I, G in ((50, 4096, 2560, 32), (150, 4096, 1024, 32)):
        mats = [bmx.Q4Matrix(*S.symmetric_codes(cuda, n, k, G, True, torch.float16, seed=1)[0], group=G) for n, k in ((I, H), (I, H), (H, I))]
        ffn, x = bmx.GatedFFN(*mats), normal(cuda, 1, T, H).to(DT[dt])
        twice([lambda: (ffn.forward(x),), lambda: (ffn.add_to(torch.zeros((T, H), device=cuda), x),)], [x])


@pytest.mark.parametrize("T,H,I", [(33, 5120, 2304), (517, 2048, 768), (2050, 1032, 4104)])
def test_16_bit_products_in_parts_at_once(cuda, T, H, I):
    """K split in the forward and the backward pass, and down's gradient beside dh."""
    import bmx
    x, dy = normal(cuda, 1, T, H).half(), normal(cuda, 2, T, H).half()
    w = [(normal(cuda, s, a, b) / b ** 0.5).half() for s, (a, b) in enumerate(((I, H), (I, H), (H, I)))]
    plain = bmx.GatedFFN(*w)
    leaves = [t.clone().requires_grad_() for t in [x] + w]
    ffn = bmx.GatedFFN(*leaves[1:])

    def step():
        y = ffn.forward(leaves[0])
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)

    twice([step, lambda: (plain.forward(x),), lambda: (plain.add_to(torch.zeros((T, H), device=cuda), x),)], [x, leaves[0], dy])
