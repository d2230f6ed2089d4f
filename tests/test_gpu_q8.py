"""8-bit matrices and rows on the GPU: quantizing, decoding, products, the gated block on them and a layer behind its norm, against the
formulas in 64 bits with bounds from the number of roundings (tests/rows8_ref.py)."""
import pytest
import torch

import ffn_ref as R
import rows8_ref as Q

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
F32 = torch.float32


def rand(cuda, *s, dt, seed, spread=0.5):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    x = torch.randn(s, device=cuda, generator=g)
    return (x * torch.exp(spread * torch.randn(s[-1], device=cuda, generator=g))).to(dt)


def matrix(cuda, N, K, seed, sdt=F32):
    """(codes, scale) over all codes, -128 among them, and W in 64 bits."""
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    c = torch.randint(-128, 128, (N, K), device=cuda, generator=g, dtype=torch.int8)
    s = ((torch.rand(N, device=cuda, generator=g) + 0.2) / (70 * K ** 0.5)).to(sdt)
    return (c, s), c.double() * s.double()[:, None]


def values(rows):
    return rows.int8().double() * rows.scale.double()[:, None]


def check_padding(rows):
    """In the blocks, zeros behind each row; and the documented order."""
    N, K = rows.N, rows.K
    b = rows.codes.view(-1, (K + 63) // 64, 4, 16, 16).transpose(2, 3)           # [16 rows][64 columns]: chunks of 16 columns, of all rows each
    flat = b.permute(0, 2, 1, 3, 4).reshape(b.shape[0] * 16, -1)
    assert torch.equal(flat[:N, :K], rows.int8()) and not bool(flat[:N, K:].any())


def check_quantized(rows, x):
    """The codes are the exact quotients' nearest whole numbers, ties to even (fp32 rows: within v inv's error, 2^-16, of a border
    either), the scales top / 127 rounded to fp32 (through 64 bits: torch divides by a number as it likes); zeros behind a row."""
    v = x.double().reshape(-1, x.shape[-1])
    top = v.abs().amax(1, keepdim=True)
    z = torch.where(top > 0, v * 127.0 / top, torch.zeros_like(v))
    codes = rows.int8()
    if x.dtype is F32:
        assert bool(((codes.double() - z).abs() <= 0.5 + 2.0 ** -16).all())
    else:
        assert torch.equal(codes, torch.round(z).to(torch.int8))
    assert torch.equal(rows.scale, (top / top.new_tensor(127.0)).float().view(-1))
    check_padding(rows)


def test_ties(cuda):
    """Halves between two codes, in rows of 16 bits where 127 / top is exact, where only top / 2 is a tie, and where top is another
    multiple of 127."""
    import bmx
    for dt, tops in ((torch.float16, (127.0, 254.0, 0.3, 1.0, 1143.0, 1905.0, 381.0, 2047.0)), (torch.bfloat16, (127.0, 0.3, 1.0, 254.0, 177.0))):
        for top in tops:
            top = float(torch.tensor(top, dtype=dt))
            n = torch.arange(-127, 127, device=cuda).double() + 0.5
            x = (n * top / 127.0).to(dt)                       # a tie where that is exact
            x = torch.cat((x, torch.tensor([top, top / 2, -top / 2, 0.0], device=cuda).to(dt), torch.arange(260, device=cuda).to(dt) * (top / 520)))
            for K in (x.numel(), x.numel() - 1):
                check_quantized(bmx.ops.quantize_rows(x[None, :K]), x[None, :K])


@pytest.mark.parametrize("dt", sorted(DT) + ["fp32"])
@pytest.mark.parametrize("T,K", [(1, 1), (3, 7), (2, 8), (5, 15), (4, 16), (3, 17), (70, 24), (1, 4096), (2, 5000), (2, 5001), (3, 11008), (2100, 40),
                                 (2100, 2048), (2100, 4104), (2, 32768), (2, 32776), (2, 131071), (1, 131064)])
def test_quantize_and_dequant(cuda, T, K, dt):
    import bmx
    dt = DT.get(dt, F32)
    x = rand(cuda, T, K, dt=dt, seed=K)
    x[-1, K // 2] = 0.0
    q = bmx.Q8Matrix.quantize(x)
    check_quantized(q, x)
    for out in (torch.float16, torch.bfloat16, F32):
        assert torch.equal(q.dequant(out), (q.int8().float() * q.scale[:, None]).to(out))
    if dt is not F32:
        r = bmx.ops.quantize_rows(x)
        assert torch.equal(r.int8(), q.int8()) and torch.equal(r.scale, q.scale) and r.dtype == dt and r.shape == (T, K)


def test_quantize_layouts_and_rows_of_no_numbers(cuda):
    import bmx
    x = rand(cuda, 6, 4, 264, dt=torch.float16, seed=1)
    q = bmx.ops.quantize_rows(x)
    assert q.shape == x.shape and q.N == 24
    check_quantized(q, x)
    for other in (x.transpose(0, 1), x[:, :, 3:250], x[1::2], x[:, :, 1:], x[0, 0], x[:, :, ::2]):
        check_quantized(bmx.ops.quantize_rows(other), other)
    for K in (264, 263):
        y = x[:, 0, :K].contiguous()
        y[1] = 0.0
        y[2, 3], y[3, 200], y[4, K - 1] = float("nan"), float("inf"), float("-inf")
        q = bmx.ops.quantize_rows(y)
        check_quantized(bmx.ops.quantize_rows(y[[0, 1, 5]]), y[[0, 1, 5]])
        assert torch.equal(q.int8()[[0, 1, 5]], bmx.ops.quantize_rows(y[[0, 1, 5]]).int8())
        assert not bool(q.int8()[1:5].any()) and bool(q.scale[2:5].isnan().all()) and float(q.scale[1]) == 0.0
        tiny = torch.full((2, K), 2.0 ** -111, device=cuda, dtype=torch.bfloat16)
        tiny[1, 5] = 2.0 ** -110
        q = bmx.ops.quantize_rows(tiny)
        assert not bool(q.int8()[0].any()) and float(q.scale[0]) == 0.0 and int(q.int8()[1, 5]) == 127
        big = torch.full((1, K), 3e38, device=cuda, dtype=torch.bfloat16)
        assert bool((bmx.ops.quantize_rows(big).int8() == 127).all())
    assert bmx.ops.quantize_rows(x[:0]).N == 0 and bmx.ops.quantize_rows(x[:0]).int8().shape == (0, 264)


@pytest.mark.parametrize("N,K", [(1, 1), (16, 64), (17, 65), (40, 15), (15, 130), (100, 4096)])
def test_given_codes(cuda, N, K):
    """Every code, in and out again, in rows and matrices; transposed and sliced ones too."""
    import bmx
    (c, s), _ = matrix(cuda, N, K, seed=N)
    odd = torch.empty(N * K + 5, dtype=torch.int8, device=cuda)[5:].view(N, K).copy_(c)
    for given in (c, c.t().contiguous().t(), torch.cat((c, c), 1)[:, :K], odd):
        for kind in (bmx.Q8Matrix, bmx.Rows8):
            q = kind(given, s)
            assert torch.equal(q.int8(), c) and torch.equal(q.scale, s)
            check_padding(q)


TOKENS = [1, 2, 3, 4, 5, 7, 15, 16, 17, 31, 33, 64, 65, 77, 128, 129, 200, 257, 300]


def check_linear(x, q, w, y, rows=None):
    import bmx
    rows = bmx.ops.quantize_rows(x) if rows is None else rows
    y64, e = Q.product(values(rows), w)
    dt = rows.dtype
    assert y.dtype == dt and y.shape == rows.shape[:-1] + (q.N,)
    R.check(f"y {q.N} {q.K}", y.reshape(rows.N, q.N), y64, R.rounded(y64, e, dt))


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T", TOKENS)
def test_linear(cuda, T, dt):
    """x given and its rows given are the same call, whatever the sizes."""
    import bmx
    for N, K in ((1, 8), (40, 136), (77, 1000), (130, 2048), (1000, 264), (33, 4104), (24, 16), (50, 1), (17, 33), (129, 515)):
        given, w = matrix(cuda, N, K, seed=T + N, sdt=(F32, DT[dt])[T % 2])
        q = bmx.Q8Matrix(*given)
        x = rand(cuda, T, K, dt=DT[dt], seed=T)
        y = bmx.ops.q8_linear(x, q)
        check_linear(x, q, w, y)
        assert torch.equal(bmx.ops.q8_linear(bmx.ops.quantize_rows(x), q), y)


@pytest.mark.parametrize("T,K,N", [(1, 4096, 14336), (1, 14336, 4096), (4, 4096, 1536), (5, 11008, 4096), (16, 5120, 2304), (20, 768, 2048),
                                   (33, 5120, 2304), (77, 4096, 4096), (150, 2304, 5120), (517, 4096, 11008), (1030, 2304, 5120), (2050, 4096, 4096),
                                   (4100, 1024, 4099), (3, 131071, 200), (300, 131064, 100)])
def test_linear_of_model_sizes(cuda, T, K, N):
    import bmx
    given, w = matrix(cuda, N, K, seed=N)
    q = bmx.Q8Matrix(*given)
    for dt in DT.values():
        x = rand(cuda, T, K, dt=dt, seed=T)
        check_linear(x, q, w, bmx.ops.q8_linear(x, q))


def test_largest_sums(cuda):
    """Every factor -128 over the longest rows: the sum is the largest that 32 bits hold."""
    import bmx
    K = 131071
    q = bmx.Q8Matrix(torch.full((40, K), -128, dtype=torch.int8, device=cuda), torch.ones(40, device=cuda))
    for T in (1, 3, 16, 40, 300):
        rows = bmx.Rows8(torch.full((T, K), -128, dtype=torch.int8, device=cuda), torch.ones(T, device=cuda) * 2.0 ** -20, torch.bfloat16)
        want = torch.tensor(128 * 128 * K * 2.0 ** -20, device=cuda).bfloat16()
        assert bool((bmx.ops.q8_linear(rows, q) == want).all())


@pytest.mark.parametrize("K,N", [(4096, 1000), (1000, 260)])
def test_a_tokens_result_does_not_depend_on_the_others(cuda, K, N):
    import bmx
    q = bmx.Q8Matrix(*matrix(cuda, N, K, seed=3)[0])
    x = rand(cuda, 1500, K, dt=torch.float16, seed=4)
    y = bmx.ops.q8_linear(x, q)
    for T in TOKENS:
        assert torch.equal(bmx.ops.q8_linear(x[:T], q), y[:T])


@pytest.mark.parametrize("T", [2, 12, 60, 300])
def test_rows_stay_apart(cuda, T):
    """A token with a NaN, an infinity or nothing but zeros, and a matrix row whose scale is NaN, change no other results."""
    import bmx
    (c, s), _ = matrix(cuda, 70, 1032, seed=1)
    s[9] = float("nan")
    q = bmx.Q8Matrix(c, s)
    x = rand(cuda, T, 1032, dt=torch.bfloat16, seed=2)
    y = bmx.ops.q8_linear(x, q)
    x[1, 77] = float("nan")
    z = bmx.ops.q8_linear(x, q)
    keep = [i for i in range(70) if i != 9]
    assert bool(z[1].isnan().all()) and bool(z[:, 9].isnan().all())
    assert torch.equal(z[0, keep], y[0, keep]) and torch.equal(z[2:, keep], y[2:, keep])
    x[1] = 0.0
    assert not bool(bmx.ops.q8_linear(x, q)[1, keep].any())


BLOCKS = [(1, 8, 8), (2, 24, 40), (4, 136, 72), (5, 200, 264), (16, 256, 128), (17, 128, 520), (33, 520, 136), (65, 1032, 328), (77, 2048, 768),
          (130, 264, 200), (300, 1288, 1032), (600, 72, 136)]


def block(cuda, H, I, act=0, L=0.0, seed=1):
    import bmx
    m = [matrix(cuda, n, k, seed + i) for i, (n, k) in enumerate(((I, H), (I, H), (H, I)))]
    return bmx.GatedFFN(*(bmx.Q8Matrix(*g) for g, _ in m), act=act, act_limit=L), [w for _, w in m]


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,H,I", BLOCKS)
def test_gated_block(cuda, T, H, I, dt):
    import bmx
    dt = DT[dt]
    act, L = (T + H) % 4, 1.25 if T % 2 else 0.0
    ffn, w = block(cuda, H, I, act, L)
    x = rand(cuda, T, H, dt=dt, seed=T)
    rows = bmx.ops.quantize_rows(x)
    y = ffn(x)
    y64, e = Q.block(values(rows), *w, act, L)
    R.check("y", y, y64, R.rounded(y64, e, dt))
    assert y.dtype == dt and torch.equal(ffn(rows), y)


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("L", [0.0, 0.7, 7.0])
def test_activations_and_clamps(cuda, act, L):
    import bmx
    for T in (3, 90):
        ffn, w = block(cuda, 96, 104, act, L, seed=act)
        x = 3.0 * rand(cuda, T, 96, dt=torch.bfloat16, seed=act)
        y64, e = Q.block(values(bmx.ops.quantize_rows(x)), *w, act, L)
        R.check("y", ffn(x), y64, R.rounded(y64, e, x.dtype))


@pytest.mark.parametrize("T,H,I", [(1, 4096, 1536), (8, 2048, 768), (16, 5120, 2304), (77, 5120, 2304), (517, 2048, 768), (1100, 4096, 2048)])
def test_gated_block_of_model_sizes(cuda, T, H, I):
    import bmx
    ffn, w = block(cuda, H, I)
    for dt in DT.values():
        x = rand(cuda, T, H, dt=dt, seed=T)
        y64, e = Q.block(values(bmx.ops.quantize_rows(x)), *w, 0, 0.0)
        R.check("y", ffn(x), y64, R.rounded(y64, e, dt))


@pytest.mark.parametrize("T,K,N", [(2100, 64, 8190), (4100, 200, 4104), (8300, 40, 8200), (16400, 1030, 2056), (4096, 2048, 4096)])
def test_many_tiles(cuda, T, K, N):
    """Several large tiles a workgroup one after the other, of fewer stages than are loaded ahead and of more, ragged at both ends; and
    the same rows in calls of few tokens."""
    import bmx
    given, w = matrix(cuda, N, K, seed=N)
    q = bmx.Q8Matrix(*given)
    x = rand(cuda, T, K, dt=torch.bfloat16, seed=T)
    y = bmx.ops.q8_linear(x, q)
    check_linear(x, q, w, y)
    for at in (0, 255, T - 300):
        assert torch.equal(bmx.ops.q8_linear(x[at:at + 300], q), y[at:at + 300])


@pytest.mark.parametrize("T,H,I", [(4100, 2056, 1032), (2300, 4104, 2568), (8200, 136, 4104)])
def test_gated_block_of_many_tiles(cuda, T, H, I):
    """Large tiles in both products: forward and added, against 64 bits, and the same as in calls of fewer tokens bit for bit."""
    import bmx
    ffn, w = block(cuda, H, I, 3, 7.0)
    x = rand(cuda, T, H, dt=torch.float16, seed=T)
    rows = bmx.ops.quantize_rows(x)
    y64, e = Q.block(values(rows), *w, 3, 7.0)
    y = ffn(x)
    R.check("y", y, y64, R.rounded(y64, e, x.dtype))
    vec = (torch.randn(H, device=cuda) / H ** 0.5).half()
    base = torch.randn((T, H), device=cuda)
    out = ffn.add_to(base.clone(), x, vec)
    s = torch.sigmoid(x.double() @ vec.double())[:, None]
    want = base.double() + s * y64
    R.check("out", out, want, s * e + 2.0 ** -22 * (want.abs() + y64.abs()) + H * R.ACC * y64.abs())
    at = T - 70
    assert torch.equal(ffn(x[at:]), y[at:]) and torch.equal(ffn.add_to(base[at:].clone(), x[at:], vec), out[at:])


@pytest.mark.parametrize("T", [1, 20, 100, 600])
def test_added_form_and_rows_behind(cuda, T):
    """add_to on a larger buffer: y before its rounding, with and without the gate vector; the rows behind the last token keep their
    bits, those of the forward pass too."""
    import bmx
    ffn, w = block(cuda, 264, 136)
    x = rand(cuda, T, 264, dt=torch.float16, seed=T)
    rows = bmx.ops.quantize_rows(x)
    y64, e = Q.block(values(rows), *w, 0, 0.0)
    for vec in (None, (torch.randn(264, device=cuda) / 16).half()):
        base = torch.randn((T + 3, 264), device=cuda)
        out, out2 = base.clone(), base.clone()
        assert ffn.add_to(out[:T], x, vec).data_ptr() == out.data_ptr()
        s = torch.ones((T, 1), dtype=torch.float64, device=cuda) if vec is None else torch.sigmoid(x.double() @ vec.double())[:, None]
        want = base[:T].double() + s * y64
        R.check("out", out[:T], want, s * e + 2.0 ** -22 * (want.abs() + y64.abs()) + 264 * R.ACC * y64.abs())
        assert torch.equal(out[T:], base[T:])
        assert torch.equal(ffn.add_to(out2[:T], x, vec, rows), out[:T])
    lib, L = bmx.lib(), bmx._lib
    s = torch.cuda.current_stream().cuda_stream
    d = ffn.desc(torch.float16)
    y = torch.full((T + 2, 264), 7.0, dtype=torch.float16, device=cuda)
    ws = torch.empty(lib.bmx_ffn8_workspace(d, T), dtype=torch.uint8, device=cuda)
    L.check(lib.bmx_ffn8_forward(d, x.data_ptr(), None, T, y.data_ptr(), ws.data_ptr(), ws.numel(), s))
    assert torch.equal(y[:T], ffn(x)) and bool((y[T:] == 7.0).all())
    q, ws = ffn.gate, torch.empty(max(1, lib.bmx_q8_linear_workspace(ffn.gate.struct, T)), dtype=torch.uint8, device=cuda)
    y = torch.full((T + 2, q.N), 7.0, dtype=torch.float16, device=cuda)
    L.check(lib.bmx_q8_linear(q.struct, 0, x.data_ptr(), None, T, y.data_ptr(), ws.data_ptr(), ws.numel(), s))
    assert torch.equal(y[:T], bmx.ops.q8_linear(x, q)) and bool((y[T:] == 7.0).all())


def test_layouts_and_no_tokens(cuda):
    import bmx
    ffn, _ = block(cuda, 136, 72)
    q = ffn.gate
    x = rand(cuda, 4, 6, 136, dt=torch.float16, seed=2)
    flat = x.view(24, 136)
    for f in (ffn, lambda a: bmx.ops.q8_linear(a, q)):
        y = f(flat)
        assert torch.equal(f(x).view(24, -1), y)
        assert torch.equal(f(x.transpose(0, 1)).transpose(0, 1).reshape(24, -1), y)
        assert torch.equal(f(bmx.ops.quantize_rows(x)).view(24, -1), y)
        wide = torch.randn((24, 150), device=cuda).half()
        wide[:, 7:143] = flat
        assert torch.equal(f(wide[:, 7:143]), y)
        assert torch.equal(f(flat[5]), y[5])
        assert f(x[:0]).shape == (0, 6, y.shape[1]) and f(bmx.ops.quantize_rows(flat[:0])).shape == (0, y.shape[1])
    with torch.no_grad():
        assert torch.equal(ffn(x.requires_grad_()).view(24, -1), ffn(flat.detach()))


@pytest.mark.parametrize("T", [1, 12, 40, 300])
def test_streams_and_graphs(cuda, T):
    """Two streams at once, and captured calls of two graphs replayed in turn with other inputs in the same places."""
    import bmx
    ffn, _ = block(cuda, 1032, 520)
    q = ffn.up
    xs = [rand(cuda, T, 1032, dt=torch.float16, seed=i) for i in range(3)]
    norm = bmx.RMSNorm(rand(cuda, 1032, dt=torch.float16, seed=8))
    run = lambda x: (bmx.ops.q8_linear(x, q), ffn(x), ffn(norm.rows8(x)))
    want = [run(x) for x in xs]
    same = lambda a, b: all(torch.equal(u, v) for u, v in zip(a, b))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(run(x))
        torch.cuda.synchronize()
        assert same(got[0], want[0]) and same(got[1], want[1])
    places, graphs, caught = [xs[0].clone(), xs[1].clone()], [], []
    for x in places:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            caught.append(run(x))
        graphs.append(g)
    for i in range(4):
        for k in (0, 1):
            places[k].copy_(xs[(i + k) % 3])
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        run(xs[2])
        torch.cuda.synchronize()
        assert same(caught[0], want[i % 3]) and same(caught[1], want[(i + 1) % 3])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", [1, 9, 300])
def test_as_a_layers_shared_expert_behind_its_norm(cuda, T, gated):
    """As it is used: an attention's output into the stream, the norm, routed and 8-bit shared experts, their fp32 output into the
    stream at the next norm, an 8-bit projection; through block() and by the single calls."""
    import bmx
    H, E = 256, 16
    tab = bmx.ExpertTable.random(H, 128, E, (bmx.TF_K3,) * 3, seed=2, device=cuda)
    ffn, w = block(cuda, H, 200)
    norm = bmx.RMSNorm((1.0 + 0.2 * rand(cuda, H, dt=F32, seed=5)).half(), eps=1e-5)
    vec = (rand(cuda, H, dt=F32, seed=6) / 16).half() if gated else None
    q, wq = matrix(cuda, 300, H, seed=7)
    q = bmx.Q8Matrix(*q)
    a, stream, lg = (rand(cuda, T, n, dt=torch.float16, seed=i) for i, n in enumerate((H, H, E)))
    z, rows, r = norm.both(a, stream)
    plain = bmx.MoELayer(tab, 4)
    layer = bmx.MoELayer(tab, 4, shared_ffn=ffn, shared_gate=vec, norm=norm)
    want = ffn.add_to(plain.forward(z, lg).clone(), z, vec, rows)
    out, r1 = layer.block(a, stream, lg)
    assert torch.equal(out, want) and torch.equal(r1, r) and torch.equal(layer.forward(z, lg, rows=rows), want)
    y64, e = Q.block(values(rows), *w, 0, 0.0)
    s = torch.sigmoid(z.double() @ vec.double())[:, None] if gated else 1.0
    want64 = plain.forward(z, lg).double() + s * y64
    R.check("out", out, want64, s * e + 2.0 ** -22 * (want64.abs() + y64.abs()) + H * R.ACC * y64.abs())
    sel, rw = layer.routing_fn(T, None, z, {"logits": lg})
    assert torch.equal(layer.run_bszN(z, sel, rw, rows=rows), ffn.add_to(plain.run_bszN(z, sel, rw).clone(), z, vec, rows))
    # without the rows the block quantizes z, which is y rounded
    assert torch.equal(layer.forward(z, lg), ffn.add_to(plain.forward(z, lg).clone(), z, vec))
    # the next norm takes the fp32 output; a layer without an 8-bit expert, and one without a residual
    n8, r2 = norm.rows8(out, r1)
    assert torch.equal(r2, (out + r1.float()).half())
    check_linear(None, q, wq, bmx.ops.q8_linear(n8, q), n8)
    o2, r3 = bmx.MoELayer(tab, 4, norm=norm).block(out, r1, lg)
    assert torch.equal(r3, r2) and torch.equal(o2, plain.forward(norm(r2), lg))
    o3, r4 = bmx.MoELayer(tab, 4, norm=norm).block(a, None, lg)
    assert r4 is a and torch.equal(o3, plain.forward(norm(a), lg))
    slots = bmx.ExpertSlots([tab], 8, maxj=4)
    o4, _ = bmx.MoELayer(tab, 4, shared_ffn=ffn, shared_gate=vec, norm=norm, slots=slots).block(a, stream, lg)
    assert float((o4 - want).abs().max()) < 1e-2


def test_a_layer_refuses_before_its_work(cuda):
    import bmx
    tab = bmx.ExpertTable.random(256, 128, 16, (bmx.TF_K3,) * 3, seed=2, device=cuda)
    ffn, _ = block(cuda, 256, 200)
    x, lg = rand(cuda, 5, 256, dt=torch.float16, seed=1), rand(cuda, 5, 16, dt=torch.float16, seed=2)
    w = torch.ones(256, device=cuda).half()
    for bad in (bmx.RMSNorm(w[:128].clone()), bmx.RMSNorm(w.bfloat16())):
        with pytest.raises(ValueError, match="norm"):
            bmx.MoELayer(tab, 4, norm=bad)
    with pytest.raises(ValueError, match="no norm"):
        bmx.MoELayer(tab, 4).block(x, None, lg)
    norm = bmx.RMSNorm(w)
    slots = bmx.ExpertSlots([tab], 8, maxj=4)
    layer = bmx.MoELayer(tab, 4, shared_ffn=ffn, norm=norm, slots=slots)
    steps, rows = list(slots.seq), bmx.ops.quantize_rows(x)
    for f in (lambda: layer.forward(x[:4], lg[:4], rows=rows), lambda: layer.block(x.view(5, 1, 256), None, lg), lambda: layer.block(x, x[:3], lg),
              lambda: layer.block(x[:0], None, lg[:0]),
              lambda: layer.block(x.bfloat16(), None, lg), lambda: layer.block(x.clone().requires_grad_(), None, lg),
              lambda: bmx.MoELayer(tab, 4, slots=slots).forward(x, lg, rows=rows)):
        with pytest.raises(ValueError):
            f()
    norm.weight = w[:128].clone()
    with pytest.raises(ValueError):
        layer.block(x[:, :128].contiguous(), None, lg)
    assert list(slots.seq) == steps and layer.out_bszn is None


def test_refusals(cuda):
    import copy
    import pickle
    import bmx
    (c, s), _ = matrix(cuda, 48, 256, seed=1)
    q = bmx.Q8Matrix(c, s)
    assert torch.equal(bmx.Q8Matrix(c, s[:, None]).scale, q.scale)
    for bad in (dict(codes=c.cpu()), dict(codes=c.int()), dict(codes=c[0]), dict(scale=s[:40]), dict(scale=s.double()), dict(scale=s.cpu()),
                dict(codes=c[:0], scale=s[:0]), dict(codes=c[:, :0]), dict(scale=s.view(1, 1, 48))):
        a = dict(codes=c, scale=s)
        a.update(bad)
        with pytest.raises(ValueError):
            bmx.Q8Matrix(**a)
    with pytest.raises(ValueError):
        bmx.Q8Matrix(torch.zeros((1, 131072), dtype=torch.int8, device=cuda), s[:1])
    for name in ("N", "K", "codes", "scale", "struct", "device"):
        with pytest.raises(AttributeError):
            setattr(q, name, None)
    for f in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError):
            f(q)
    c.zero_()
    assert bool(q.int8().any())                        # its own copy
    x = rand(cuda, 3, 256, dt=torch.float16, seed=1)
    rows = bmx.ops.quantize_rows(x)
    for bad in (x.float(), x.cpu(), x[:, :128], x.long(), bmx.ops.quantize_rows(x[:, :128])):
        with pytest.raises(ValueError):
            bmx.ops.q8_linear(bad, q)
    for bad in (x.float(), x.cpu(), x[0, 0], x[:, :0]):
        with pytest.raises(ValueError):
            bmx.ops.quantize_rows(bad)
    for bad in (x.long(), x.cpu(), x[0], x[:0]):
        with pytest.raises(ValueError):
            bmx.Q8Matrix.quantize(bad)
    with pytest.raises(ValueError):
        q.dequant(torch.float64)
    for kw in (dict(dtype=F32), dict(shape=(2, 256)), dict(shape=(256, 3))):
        with pytest.raises(ValueError):
            bmx.Rows8(rows.int8(), rows.scale, **kw)
    assert torch.equal(bmx.ops.q8_linear(bmx.Rows8(rows.int8(), rows.scale, shape=(1, 3, 256)), q)[0], bmx.ops.q8_linear(x, q))
    down = bmx.Q8Matrix(*matrix(cuda, 256, 48, seed=2)[0])
    ffn = bmx.GatedFFN(q, q, down)
    four = bmx.Q4Matrix.quantize(rand(cuda, 48, 256, dt=torch.float16, seed=3), 64)
    for three in ((q, q, q), (q, four, down), (four, q, down), (q, q, rand(cuda, 256, 48, dt=torch.float16, seed=1)),
                  tuple(bmx.Q8Matrix(*matrix(cuda, n, k, seed=1)[0]) for n, k in ((44, 256), (44, 256), (256, 44)))):
        with pytest.raises(ValueError):
            bmx.GatedFFN(*three)
    out = torch.zeros((3, 256), device=cuda)
    for bad in (lambda: ffn(x.float()), lambda: ffn(x[:, :128]), lambda: ffn(bmx.ops.quantize_rows(x[:, :128])), lambda: ffn(None),
                lambda: ffn.add_to(out, x, None, bmx.ops.quantize_rows(x[:2])), lambda: ffn.add_to(out[:2], x), lambda: ffn.add_to(out.half(), x)):
        with pytest.raises(ValueError):
            bad()
    x.requires_grad_()
    for f in (lambda: ffn(x), lambda: bmx.ops.q8_linear(x, q), lambda: bmx.ops.quantize_rows(x), lambda: ffn.add_to(out, x)):
        with pytest.raises(ValueError, match="no gradients"):
            f()
    with torch.no_grad():
        assert torch.equal(ffn(x), ffn(rows))
