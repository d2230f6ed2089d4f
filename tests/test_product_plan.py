"""The planner of the tiled products on the CPU: its own header, built with g++ (tests/native/product_plan.cpp)."""
import ctypes
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "big-moe-small-box_amd", "csrc")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    out = str(tmp_path_factory.mktemp("plan") / "product_plan.so")
    b = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-I", CSRC, "-o", out,
                        os.path.join(HERE, "native", "product_plan.cpp")], capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-4000:]
    lib = ctypes.CDLL(out)
    lib.plan_past_the_end.restype = ctypes.c_int64
    return lib


# (H, I, T, products in two parts with A stored across K and a ragged last tile)
TWO_PARTS = [(2880, 2880, 8192, (2, 3)), (2048, 10944, 8192, (2, 4)), (2048, 10944, 16384, (4,)), (4104, 1032, 4100, (3,)), (1032, 5200, 4100, (2,))]


def past(plan, H, I, T, which, moved=0):
    parts = ctypes.c_int()
    return plan.plan_past_the_end(H, I, T, which, moved, ctypes.byref(parts)), parts.value


@pytest.mark.parametrize("H,I,T,which", TWO_PARTS)
def test_second_parts_end_where_the_matrix_ends(plan, H, I, T, which):
    """A launch's loads are cut off at the end of the matrix that they read, whichever rows of it the launch takes. (Counted from
    a pointer moved to the second part's rows, a matrix stored across K would end as many values too late.)"""
    for w in which:
        got, parts = past(plan, H, I, T, w)
        assert parts == 2 and got == 0, (w, got, parts)
        assert past(plan, H, I, T, w, moved=1)[0] > 0


def test_no_product_reads_past_its_operands(plan):
    two = 0
    for H, I in ((8, 8), (72, 264), (520, 4096), (768, 2048), (2048, 768), (2048, 10944), (2880, 2880), (4096, 2048), (4096, 11008),
                 (5120, 2304), (1032, 5200)):
        for T in (1, 17, 33, 130, 517, 1100, 2050, 4100, 8192):
            for w in range(6):
                got, parts = past(plan, H, I, T, w)
                assert got == 0, (H, I, T, w, got)
                two += parts == 2
    assert two > 20


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(139, 5888), (768, 2048), (1536, 4096), (4096, 4096), (11008, 4096), (4096, 11008), (2304, 5120), (5120, 2304)])
def test_more_tokens_never_keep_more_digits_of_a_4_bit_matrix(plan, N, K, group):
    """Weights are rounded to 16 bits from one count of tokens on, the documented one at the least, and never where 16 bits may
    not hold them."""
    K = K // group * group
    for products in (1, 2):
        counts = list(range(1, 2100)) + [2304, 3000, 4096, 4097, 5392, 8192, 1 << 16, 1 << 20]
        rounds = [plan.plan_rounds(N, K, T, products, group, 0) for T in counts]
        assert rounds == sorted(rounds) and rounds[-1] == 1
        assert not any(rounds[:256 if group == 32 else 1024])
        assert not any(plan.plan_rounds(N, K, T, products, group, 1) for T in counts[::37])


def names(plan, op, T, H, I, group=0):
    buf = ctypes.create_string_buffer(4096)
    assert plan.plan_names(op, T, H, I, group, buf, len(buf))
    return set(buf.value.decode().split("\n")) - {""}


def test_every_kernel_instance_is_compared_with_sharp_bounds(plan):
    """The sizes of ffn_sizes.py, at which test_gpu_sharp.py compares every result in both types, reach each kernel instance that
    calls of any size are planned on: skinny_k by row tiles, group, epilogue and form, slice_k, gemm_q4_k, gemm16_k by tile, operands
    and epilogue, whole, split, as head and as rest."""
    import math
    import random
    import ffn_sizes as Z
    reached = set()
    for T, K, N, G in Z.LINEAR:
        reached |= names(plan, 0, T, K, N, G)
    for T, H, I, G in Z.BLOCK4:
        reached |= names(plan, 1, T, H, I, G) | names(plan, 2, T, H, I, G)
    for T, H, I in Z.BLOCK16:
        reached |= names(plan, 1, T, H, I) | names(plan, 2, T, H, I) | names(plan, 3, T, H, I)
    rng = random.Random(3)
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    launched = set()
    for _ in range(40000):
        T = rng.choice((log(1, 16), log(17, 80), log(81, 1100), log(1100, 16384)))
        op = rng.choice((0, 1, 2, 3, 4, 5))
        if op in (0, 4, 5):
            G = rng.choice((32, 64, 128))
            launched |= names(plan, op % 3, T, G * log(1, 12288 // G), log(1, 16384) if op == 0 else G * log(1, 16384 // G), G)
        else:
            launched |= names(plan, op, T, 8 * log(1, 1100), 8 * log(1, 1376))
    assert len(launched) > 150
    assert not launched - reached, sorted(launched - reached)
