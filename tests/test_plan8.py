"""The planner of the 8-bit products on the CPU: its own header, built with g++ (tests/native/plan8.cpp)."""
import ctypes
import math
import os
import random
import shutil
import subprocess

import pytest

import q8_sizes as Z

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "big-moe-small-box_amd", "csrc")


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not found")
    out = str(tmp_path_factory.mktemp("plan8") / "plan8.so")
    b = subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-I", CSRC, "-o", out, os.path.join(HERE, "native", "plan8.cpp")],
                       capture_output=True, text=True, timeout=300)
    assert b.returncode == 0, b.stderr[-4000:]
    lib = ctypes.CDLL(out)
    lib.plan8_part_bytes.restype = ctypes.c_int64
    return lib


def names(plan, op, T, H, I):
    buf = ctypes.create_string_buffer(4096)
    assert plan.plan8_names(op, T, H, I, buf, len(buf))
    return set(buf.value.decode().split("\n")) - {""}


def logs(rng):
    return lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def test_every_kernel_instance_is_compared_with_sharp_bounds(plan):
    """skinny8_k by input, tokens, rows of W and epilogue, gemm8_k by tile and epilogue, whole and in parts along K, and finish8_k."""
    reached = set()
    for T, K, N in Z.LINEAR:
        reached |= names(plan, 0, T, K, N) | names(plan, 1, T, K, N)
    for T, H, I in Z.BLOCK:
        reached |= names(plan, 2, T, H, I) | names(plan, 3, T, H, I)
    rng = random.Random(3)
    log = logs(rng)
    launched = set()
    for _ in range(40000):
        T = rng.choice((log(1, 16), log(17, 80), log(81, 1100), log(1100, 16384)))
        op = rng.randrange(4)
        size = (log(1, 16384), log(1, 16384)) if op < 2 else (8 * log(1, 1600), 8 * log(1, 1600))
        launched |= names(plan, op, T, *size)
    assert len(launched) > 50
    assert not launched - reached, sorted(launched - reached)


def test_launches_take_each_row_once(plan):
    rng = random.Random(4)
    log = logs(rng)
    for _ in range(20000):
        T, N, K, products = log(1, 70000), log(1, 40000), log(1, 131071), rng.choice((1, 2))
        if products == 2:
            N, K = (N + 7) // 8 * 8, min(K + 7, 131064) // 8 * 8
        assert plan.plan8_rows(N, K, T, products) == N, (N, K, T, products)


def test_sums_in_parts_take_little_memory(plan):
    """Room for the sums where an axis is split, for each part and product its own, and none elsewhere."""
    rng = random.Random(5)
    log = logs(rng)
    split = 0
    for _ in range(20000):
        T, N, K, products = log(1, 70000), log(1, 40000), log(1, 131071), rng.choice((1, 2))
        n, s = plan.plan8_part_bytes(N, K, T, products), plan.plan8_splits(N, K, T, products)
        least = 0 if s == 1 else products * s * T * ((N + 7) // 8 * 8) * 4
        assert least <= n <= least + 4096, (N, K, T, products, s, n)
        split += s > 1
    assert split > 500
