"""4-bit matrices with group scales on the GPU: packing, decoding, products and the gated block on them, against 64 bits with
bounds from the number of roundings (tests/ffn_ref.py)."""
import pytest
import torch

import ffn_ref as R

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def codes(cuda, N, K, G, zero, scale_dt, seed=1):
    """(codes, scale, zero) in checkpoint order and (W, spread) in 64 bits; zero: "none", "mid" or "any" (0 .. 255)."""
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    c = torch.randint(0, 16, (N, K), device=cuda, generator=g, dtype=torch.uint8)
    scale = ((torch.rand((N, K // G), device=cuda, generator=g) + 0.2) / (4 * K ** 0.5)).to(scale_dt)
    z = None
    if zero != "none":
        z = torch.randint(*((0, 16) if zero == "mid" else (0, 256)), (N, K // G), device=cuda, generator=g, dtype=torch.uint8)
    spread = lambda t: t.double().repeat_interleave(G, 1)
    z64 = 8.0 if z is None else spread(z)
    w = (c.double() - z64) * spread(scale)
    return (c[:, 0::2] | (c[:, 1::2] << 4), scale, z), (w, spread(scale) * (271.0 + z64))


def rand(cuda, *s, dt, seed):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return torch.randn(s, device=cuda, generator=g).to(dt)


@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 128), (16, 256), (17, 384), (100, 640), (31, 128 + 256), (768, 2048)])
def test_pack_and_dequant(cuda, N, K, G):
    """Every weight, with each scale type and zero-point form: one rounding of the exact value."""
    import bmx
    for i, zero in enumerate(("none", "mid", "any")):
        for sdt in DT.values():
            # K odd multiples of the group too
            k = K + (G if i and G < 128 else 0)
            given, (w, _) = codes(cuda, N, k, G, zero, sdt, seed=N + i)
            q = bmx.Q4Matrix(*given, group=G)
            for dt in DT.values():
                assert torch.equal(q.dequant(dt), w.float().to(dt)), (zero, sdt, dt)


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 2, 7, 16, 17, 32, 33, 50, 64, 65, 77, 128, 129, 200, 300])
def test_linear(cuda, T, G, dt):
    import bmx
    for N, K, zero in ((1, G, "none"), (40, 3 * G, "mid"), (77, 1024 + G, "any"), (130, 2048, "mid"), (1000, 256, "none")):
        given, q64 = codes(cuda, N, K, G, zero, DT[dt], seed=T + N)
        x = rand(cuda, T, K, dt=DT[dt], seed=T)
        y = bmx.ops.q4_linear(x, bmx.Q4Matrix(*given, group=G))
        y64, e = R.q4_product(x.double(), q64, DT[dt])
        assert y.dtype == DT[dt] and y.shape == (T, N)
        R.check(f"y {N} {K}", y, y64, R.rounded(y64, e, DT[dt]))


@pytest.mark.parametrize("T,K,N", [(1, 2048, 14336), (520, 4096, 520), (1100, 1024, 4096), (4200, 256, 1032), (8, 5120, 2304), (3, 11008, 4096), (64, 4096, 1536), (600, 512, 3016)])
def test_linear_of_model_sizes(cuda, T, K, N):
    import bmx
    given, q64 = codes(cuda, N, K, 128, "mid", torch.float16)
    for dt in DT.values():
        x = rand(cuda, T, K, dt=dt, seed=T)
        y64, e = R.q4_product(x.double(), q64, dt)
        R.check("y", bmx.ops.q4_linear(x, bmx.Q4Matrix(*given)), y64, R.rounded(y64, e, dt))


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I,G", [(1, 128, 256, 128), (2, 192, 64, 64), (5, 96, 160, 32), (16, 512, 384, 128), (17, 320, 448, 64),
                                     (33, 256, 96, 32), (64, 128, 128, 64), (65, 384, 640, 128), (81, 160, 96, 32), (200, 192, 320, 64),
                                     (520, 2048, 768, 128)])
def test_gated_block(cuda, T, H, I, G, dt):
    import bmx
    act, L = (T + H // 32) % 4, 1.25 if T % 2 else 0.0
    parts = [codes(cuda, n, k, G, z, torch.float16, seed=s) for s, (n, k, z) in enumerate(((I, H, "mid"), (I, H, "none"), (H, I, "mid")))]
    ffn = bmx.GatedFFN(*(bmx.Q4Matrix(*p[0], group=G) for p in parts), act=act, act_limit=L)
    x = rand(cuda, T, H, dt=DT[dt], seed=T)
    prod = lambda a, q: R.q4_product(a, q, DT[dt])
    g, u, h, _, _, eh = R.forward(x.double(), parts[0][1], parts[1][1], act, L, prod)
    y64, e = R.q4_product(h, parts[2][1], DT[dt], R.rounded(h, eh, DT[dt]))
    R.check("y", ffn.forward(x), y64, R.rounded(y64, e, DT[dt]))
    vec = (rand(cuda, H, dt=torch.float32, seed=3) / 16).to(DT[dt])
    base = torch.randn((T + 2, H), device=cuda)
    for v in (None, vec):
        out = base.clone()
        ffn.add_to(out[:T], x, v)
        s = torch.ones((T, 1), dtype=torch.float64, device=cuda) if v is None else torch.sigmoid(x.double() @ v.double())[:, None]
        want = base[:T].double() + s * y64
        R.check("out", out[:T], want, s * e + 2.0 ** -22 * (want.abs() + y64.abs()) + H * R.ACC * y64.abs())
        assert torch.equal(out[T:], base[T:])


def test_mixed_groups_and_layouts(cuda):
    """down may have groups of another size; leading dimensions, strided and odd-offset x; one row; no rows."""
    import bmx
    (g, _), (u, _), (d, _) = (codes(cuda, 192, 128, 32, "mid", torch.bfloat16), codes(cuda, 192, 128, 32, "none", torch.float16),
                              codes(cuda, 128, 192, 64, "any", torch.float16))
    ffn = bmx.GatedFFN(bmx.Q4Matrix(*g, group=32), bmx.Q4Matrix(*u, group=32), bmx.Q4Matrix(*d, group=64))
    x = rand(cuda, 12, 128, dt=torch.float16, seed=1)
    for f, n in ((ffn.forward, 128), (lambda v: bmx.ops.q4_linear(v, ffn.gate), 192)):
        want = f(x)
        assert torch.equal(f(x.view(3, 4, 128)).view(12, n), want)
        wide = torch.zeros((12, 300), dtype=x.dtype, device=cuda)
        wide[:, 5:133] = x
        assert torch.equal(f(wide[:, 5:133]), want)
        assert torch.equal(f(x[3]), want[3]) and f(x[:0]).shape == (0, n)
        # rows do not depend on the others of the call
        assert torch.equal(f(x[2:5]), want[2:5])
    leaf = x.clone().requires_grad_()
    with pytest.raises(ValueError):
        ffn.forward(leaf)
    with pytest.raises(ValueError):
        bmx.ops.q4_linear(leaf, ffn.gate)
    with torch.no_grad():
        assert torch.equal(ffn.forward(leaf), ffn.forward(x))


@pytest.mark.parametrize("T", [5, 100])
def test_nan_stays_in_its_row(cuda, T):
    import bmx
    for dt in DT.values():
        given, _ = codes(cuda, 200, 320, 64, "mid", torch.float16)
        q = bmx.Q4Matrix(*given, group=64)
        x = rand(cuda, T, 320, dt=dt, seed=1)
        want = bmx.ops.q4_linear(x, q)
        x[T // 2, 3] = float("nan")
        y = bmx.ops.q4_linear(x, q)
        rows = [t for t in range(T) if t != T // 2]
        assert bool(torch.isnan(y[T // 2]).all()) and torch.equal(y[rows], want[rows])


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128])
def test_quantize(cuda, G, symmetric):
    """Every weight within half a step of the stored scale (and the scale's own rounding over at most 15 codes); constant,
    zero and one-sided groups among them."""
    import bmx
    for dt in DT.values():
        w = rand(cuda, 50, 4 * G, dt=dt, seed=G)
        w[0] = 0
        w[1] = 0.5
        w[2] = w[2].abs()
        w[3] = -w[3].abs()
        q = bmx.Q4Matrix.quantize(w, G, symmetric)
        v = w.double().view(50, 4, G)
        span = v.abs().amax(2) / 7.5 if symmetric else (v.amax(2).clamp(min=0) - v.amin(2).clamp(max=0)) / 15
        # half a step, and up to 15 steps' share of the scale's rounding; symmetric: the top code is 7 steps, half a step short
        # of the bottom's 8; asymmetric: the zero point's own rounding moves the ends by up to half a step
        bound = span * (1.0 + 16 * R.HALF[dt]) + 16 * R.HALF[dt] * v.abs().amax(2)
        err = (q.dequant(dt).double() - w.double()).view(50, 4, G).abs().amax(2)
        assert bool((err <= bound).all())


@pytest.mark.parametrize("T", [3, 90])
def test_streams_and_graphs(cuda, T):
    import bmx
    given, _ = codes(cuda, 264, 256, 32, "mid", torch.float16)
    down, _ = codes(cuda, 256, 256, 32, "mid", torch.float16)
    up, _ = codes(cuda, 256, 256, 32, "mid", torch.float16, seed=5)
    q, ffn = bmx.Q4Matrix(*given, group=32), bmx.GatedFFN(*(bmx.Q4Matrix(*m, group=32) for m in (up, up, down)))
    x = rand(cuda, T, 256, dt=torch.bfloat16, seed=1)
    want = (bmx.ops.q4_linear(x, q), ffn.forward(x))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            outs.append([(bmx.ops.q4_linear(x, q), ffn.forward(x)) for _ in range(4)])
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for os in outs for o in os for a, b in zip(o, want))
    torch.cuda.synchronize()
    sx = x.clone()
    graphs, caught = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            caught.append((bmx.ops.q4_linear(sx, q), ffn.forward(sx)))
    for k in range(4):
        sx.copy_(torch.randn_like(x) * (k + 1))
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        eager = (bmx.ops.q4_linear(sx, q), ffn.forward(sx))
        for c in caught:
            assert all(torch.equal(a, b) for a, b in zip(c, eager))


@pytest.mark.parametrize("T", [1, 20, 300])
def test_layer_of_routed_and_4_bit_shared_experts(cuda, T):
    """A whole layer as it is used: routing, routed trellis experts, the 4-bit shared expert with its gate, then a 4-bit
    projection of the result."""
    import bmx
    H, E = 256, 16
    tab = bmx.ExpertTable.random(H, 128, E, (bmx.TF_K3,) * 3, seed=2, device=cuda)
    mats = [codes(cuda, n, k, 64, "mid", torch.float16, seed=i) for i, (n, k) in enumerate(((192, H), (192, H), (H, 192), (500, H)))]
    q = [bmx.Q4Matrix(*m[0], group=64) for m in mats]
    vec = (rand(cuda, H, dt=torch.float32, seed=9) / 16).half()
    ffn = bmx.GatedFFN(*q[:3])
    x, lg = rand(cuda, T, H, dt=torch.float16, seed=3), rand(cuda, T, E, dt=torch.float16, seed=4)
    routed = bmx.MoELayer(tab, 4).forward(x, lg)
    out = bmx.MoELayer(tab, 4, shared_ffn=ffn, shared_gate=vec).forward(x, lg)
    prod = lambda a, m: R.q4_product(a, m, torch.float16)
    _, _, h, _, _, eh = R.forward(x.double(), mats[0][1], mats[1][1], 0, 0.0, prod)
    y64, e = R.q4_product(h, mats[2][1], torch.float16, R.rounded(h, eh, torch.float16))
    s = torch.sigmoid(x.double() @ vec.double())[:, None]
    want = routed.double() + s * y64
    R.check("out", out, want, s * e + 2.0 ** -22 * (want.abs() + y64.abs()) + H * R.ACC * y64.abs())
    z = out.half()
    z64, ez = R.q4_product(z.double(), mats[3][1], torch.float16)
    R.check("z", bmx.ops.q4_linear(z, q[3]), z64, R.rounded(z64, ez, torch.float16))


def test_refusals(cuda):
    import bmx
    (c, s, z), _ = codes(cuda, 48, 256, 64, "mid", torch.float16)
    q = bmx.Q4Matrix(c, s, z, 64)
    for bad in (dict(group=48), dict(group=128), dict(codes=c.cpu()), dict(codes=c.int()), dict(codes=c[:, :60].contiguous()),
                dict(codes=c[:, ::2]), dict(scale=s.float()), dict(scale=s[:, :2]), dict(scale=s[:40]), dict(zero=z.int()),
                dict(zero=z[:, :3]), dict(zero=z.cpu()), dict(codes=c[:0], scale=s[:0], zero=z[:0])):
        a = dict(codes=c, scale=s, zero=z, group=64)
        a.update(bad)
        with pytest.raises(ValueError):
            bmx.Q4Matrix(**a)
    x = rand(cuda, 3, 256, dt=torch.float16, seed=1)
    for bad in (x.float(), x.cpu(), x[:, :128], x.long()):
        with pytest.raises(ValueError):
            bmx.ops.q4_linear(bad, q)
    with pytest.raises(ValueError):
        q.dequant(torch.float32)
    with pytest.raises(ValueError):
        bmx.Q4Matrix.quantize(x.float())
    with pytest.raises(ValueError):
        bmx.Q4Matrix.quantize(x[:, :100])
    down = bmx.Q4Matrix(*codes(cuda, 256, 48 + 16, 64, "mid", torch.float16)[0], group=64)
    with pytest.raises(ValueError):
        bmx.GatedFFN(q, q, down)                      # [I, H] = [48, 256] needs down [256, 48]
    other = bmx.Q4Matrix(*codes(cuda, 48, 256, 128, "mid", torch.float16)[0], group=128)
    with pytest.raises(ValueError):
        bmx.GatedFFN(q, other, down)
    with pytest.raises(ValueError):
        bmx.GatedFFN(q, q, rand(cuda, 256, 48, dt=torch.float16, seed=1))


def test_quantize_of_views_leaves_and_small_groups(cuda):
    """A transposed view and a leaf give the plain tensor's matrix; a group whose scale is below fp16's normal range keeps its
    values within that scale's own steps; no elements are refused."""
    import bmx
    w = rand(cuda, 64, 96, dt=torch.float16, seed=2)
    want = bmx.Q4Matrix.quantize(w, 32).dequant()
    assert torch.equal(bmx.Q4Matrix.quantize(w.t().contiguous().t(), 32).dequant(), want)
    assert torch.equal(bmx.Q4Matrix.quantize(w.clone().requires_grad_(), 32).dequant(), want)
    small = (w.float() * 2.0 ** -13).half()
    got = bmx.Q4Matrix.quantize(small, 32).dequant().double()
    v = small.double().view(64, 3, 32)
    span = (v.amax(2).clamp(min=0) - v.amin(2).clamp(max=0)) / 15
    # half a step, the zero point's half step, and the scale's own rounding, half of 2^-24, over up to 15 codes and in each
    # half step
    bound = span + 16 * 2.0 ** -25
    assert bool(((got - small.double()).view(64, 3, 32).abs().amax(2) <= bound).all())
    with pytest.raises(ValueError):
        bmx.Q4Matrix.quantize(w[:0], 32)


# larger matrices, whose products leave the kernel of few tokens: slices of 2 to 5 tiles of tokens, then tiles with K split and not
@pytest.mark.parametrize("T,K,N,G", [(20, 3264, 8232, 64), (30, 3200, 8232, 32), (33, 3232, 6152, 32), (40, 3200, 6150, 128),
                                     (50, 3328, 4120, 128), (64, 3200, 4120, 64), (77, 4128, 4100, 32), (77, 4096, 4120, 64),
                                     (80, 4096, 4120, 128), (81, 4128, 3080, 32), (128, 4096, 2056, 128), (129, 4160, 2056, 64),
                                     (300, 4096, 1000, 64), (200, 256, 4120, 32), (100, 320, 8232, 64), (130, 256, 6152, 128)])
def test_linear_of_larger_matrices(cuda, T, K, N, G):
    import bmx
    for dt in DT.values():
        given, q64 = codes(cuda, N, K, G, "any" if T % 2 else "none", dt, seed=T)
        x = rand(cuda, T, K, dt=dt, seed=T)
        y64, e = R.q4_product(x.double(), q64, dt)
        R.check("y", bmx.ops.q4_linear(x, bmx.Q4Matrix(*given, group=G)), y64, R.rounded(y64, e, dt))


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I,G", [(40, 4096, 4096, 64), (50, 4096, 2560, 32), (70, 4096, 4096, 128), (77, 4096, 4096, 32),
                                     (77, 4096, 2048, 64), (100, 512, 4096, 64), (100, 2560, 4096, 32), (150, 2048, 4096, 128),
                                     (150, 4096, 4096, 32), (300, 1024, 4096, 64), (300, 4096, 1024, 128), (300, 4096, 512, 128)])
def test_gated_block_of_larger_matrices(cuda, T, H, I, G, dt):
    test_gated_block(cuda, T, H, I, G, dt)
