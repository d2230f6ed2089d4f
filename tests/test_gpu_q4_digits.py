"""Which digits of a 4-bit matrix a product keeps: sums that fp32 holds exactly, so that nothing but y's rounding may show."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def pairs(cuda, T, N, K, G, dt, sdt, zero, low=1.0, seed=1):
    """(x, matrix, y and W in 64 bits): x is 1 at one column and -1 at another, of another group. Scales in [low, 2 low) of sdt (11 or 8
    bits), codes - zeros of 5: sums of either order, and of 128 + code before the offset comes off, take 20 bits at the most."""
    import bmx
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    r = lambda *a: torch.randint(*a, device=cuda, generator=g)
    c = r(0, 16, (N, K)).to(torch.uint8)
    s = ((torch.rand((N, K // G), device=cuda, generator=g) + 1.0) * low).to(sdt).clamp(max=2 * low)
    z = r(0, 16, (N, K // G)).to(torch.uint8) if zero else None
    at = r(0, K // G, (T,))
    to = (at + r(1, K // G, (T,))) % (K // G)
    a, b = at * G + r(0, G, (T,)), to * G + r(0, G, (T,))
    x = torch.zeros((T, K), device=cuda)
    x[torch.arange(T), a], x[torch.arange(T), b] = 1.0, -1.0
    spread = lambda t: t.double().repeat_interleave(G, 1)
    w = (c.double() - (8.0 if z is None else spread(z))) * spread(s)
    return x.to(dt), bmx.Q4Matrix(c[:, 0::2] | (c[:, 1::2] << 4), s, z, G), (w[:, a] - w[:, b]).t(), w


@pytest.mark.parametrize("dt", sorted(DT))
@pytest.mark.parametrize("T,N,K,G", [(1, 768, 2048, 128), (5, 300, 1024, 32), (16, 2304, 5120, 64), (20, 8232, 3264, 64), (77, 4096, 4096, 32),
                                     (90, 264, 512, 64), (100, 5120, 2304, 32), (200, 4096, 4096, 32), (256, 11008, 4096, 32),
                                     (300, 4096, 4096, 64), (300, 5120, 2304, 128), (400, 4096, 4096, 128), (517, 2304, 5120, 128),
                                     (900, 14336, 4096, 128), (1024, 768, 2048, 64), (1024, 4096, 11008, 128)])
def test_weights_are_not_rounded(cuda, T, N, K, G, dt):
    """To 1,024 tokens (256 with groups of 32) y is the exact sum, rounded once: rounded weights that nearly cancel would show."""
    import bmx
    x, q, y64, _ = pairs(cuda, T, N, K, G, DT[dt], torch.float16, T % 2 == 0)
    y = bmx.ops.q4_linear(x, q)
    assert torch.equal(y, y64.to(DT[dt]))
    # the matrix of rounded weights does not pass
    if T > 16:
        d = q.dequant(DT[dt]).double()
        assert not torch.equal((x.double() @ d.t()).to(DT[dt]), y)


@pytest.mark.parametrize("T", [3, 40, 300, 1100, 2100])
@pytest.mark.parametrize("low", [2.0 ** -30, 2.0 ** 20])
def test_scales_outside_the_range_of_fp16(cuda, T, low):
    """fp16 x with bf16 scales: weights that fp16 does not hold, at any number of tokens, alone and in the block."""
    import bmx
    x, q, y64, _ = pairs(cuda, T, 512, 1024, 64, torch.float16, torch.bfloat16, True, low)
    up = 2.0 ** 14 if low < 1 else 2.0 ** -14
    y = bmx.ops.q4_linear(x * up, q)
    assert torch.equal(y, (y64 * up).to(torch.float16)) and bool((y.abs() > 0).any()) and bool(y.isfinite().all())
    # the block: gate of small weights and up of large ones, h and y are fp16's again
    if low < 1:
        mats = [pairs(cuda, 1, n, k, 64, torch.float16, torch.bfloat16, True, v, seed=i)
                for i, (n, k, v) in enumerate(((256, 512, 2.0 ** -22), (256, 512, 2.0 ** 14), (512, 256, 2.0 ** 6)))]
        x = torch.randn((T, 512), device=cuda, generator=torch.Generator(device=cuda).manual_seed(2)).half() * 2.0 ** -6
        g, u = (x.double() @ m[3].t() for m in mats[:2])
        y64 = g * torch.sigmoid(g) * u @ mats[2][3].t()
        y = bmx.GatedFFN(*(m[1] for m in mats)).forward(x)
        # h is of order 2^-7, so that fp16's smallest step does not show; its rounding and y's are 2^-11 each, the sums of at most
        # 512 products 2^-23 each of themselves at the most, the activation's dozen operations 2^-23 each: 2^-9 is twice as much
        assert bool(y.isfinite().all())
        assert float((y.double() - y64).norm()) <= 2.0 ** -9 * float(y64.norm())


def test_a_matrix_of_more_than_2_32_words(cuda):
    """2^20 rows of 32,896 columns, 17 GB of codes: packed whole, and products of few and many tokens that reach every row."""
    import bmx
    N, K, G = 1 << 20, 257 * 128, 128
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    row = torch.randint(0, 256, (1009, K // 2), device=cuda, generator=g, dtype=torch.uint8)     # rows repeat every 1,009
    codes = torch.empty((N, K // 2), dtype=torch.uint8, device=cuda)
    for n in range(0, N, 1009):
        codes[n:n + 1009] = row[:min(1009, N - n)]
    scale = torch.empty((N, K // G), dtype=torch.float16, device=cuda)
    scale[:] = (1.0 + torch.arange(N, device=cuda) % 7)[:, None].half()                          # and scales every 7
    q = bmx.Q4Matrix(codes, scale, None, G)
    del codes, scale
    x = torch.zeros((100, K), device=cuda)
    at = torch.randint(0, K, (100, 4), device=cuda, generator=g)
    x.scatter_(1, at, 1.0)
    x = x.half()
    c = torch.stack((row & 15, row >> 4), 2).view(1009, K).double() - 8.0
    part = x.double() @ c.t()                                                                     # whole numbers: exact
    rows = torch.arange(N, device=cuda)
    for T in (1, 3, 20, 100):
        y = bmx.ops.q4_linear(x[:T], q)
        for t in range(T):
            assert torch.equal(y[t].double(), part[t][rows % 1009] * (1 + rows % 7))


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("G", [32, 64, 128])
@pytest.mark.parametrize("dt", sorted(DT))
def test_quantized_weights_are_within_half_a_step(cuda, G, symmetric, dt):
    """s the group's step, |s - step| <= half a rounding of it. A value whose code is in range is off by at most s / 2, whatever the
    zero point (a whole number). At the ends, up to 15 steps from the zero point's end (7.5 symmetric), the zero point's rounding or the
    missing half code takes up to s / 2 and the scale's rounding up to 15 of its own; then the decoded weight is rounded. Codes that
    are cut instead of rounded are off by up to a step."""
    import bmx
    dt = DT[dt]
    half = torch.finfo(dt).eps / 2
    w = torch.randn((200, 4 * G), device=cuda, generator=torch.Generator(device=cuda).manual_seed(G)).to(dt)
    w[0], w[1], w[2], w[3] = 0, 0.5, w[2].abs(), -w[3].abs()
    w[4, :G] *= 64.0
    v = w.double().view(200, 4, G)
    lo, hi = v.amin(2).clamp(max=0), v.amax(2).clamp(min=0)
    step = v.abs().amax(2) / 7.5 if symmetric else (hi - lo) / 15
    bound = step * (0.5 * (1 + half) + 15 * half + 2.0 ** -19) + half * v.abs().amax(2)
    q = bmx.Q4Matrix.quantize(w, G, symmetric)
    err = (q.dequant(dt).double().view(200, 4, G) - v).abs().amax(2)
    assert bool((err <= bound).all()), float((err / bound).nan_to_num().max())
    s = step.clamp(min=1e-9)[..., None]
    z = 8.0 if symmetric else (-lo[..., None] / s).round()
    cut = ((v / s + z).floor().clamp(0, 15) - z) * s
    assert bool(((cut - v).abs().amax(2) > bound)[5:].any())
