"""CPU: which kernel takes a call of the 8-bit linear (rust_ascend_b200/csrc/linear_plan.h)."""
import ctypes as C
import math
import os
import random
import subprocess

import pytest

from linear_sizes import SIZES

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "rust_ascend_b200", "csrc")
SMS, PAIRS = 148, 74


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """(m, n, k[, limit]) -> the entries of linear_sizes.SIZES."""
    library = str(tmp_path_factory.mktemp("plan") / "linear_plan_host.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, "-o", library, os.path.join(HERE, "host_model", "linear_plan_host.cpp")], check=True)
    host = C.CDLL(library)

    def call(m, n, k, limit=0):
        out = (C.c_uint32 * 3)()
        pairs = max(limit // 2, 1) if limit else PAIRS
        host.host_linear_plan(m, n, k, limit or SMS, pairs, int(limit > 0), out)
        tokens, parts, rows = out
        if tokens == 0:
            return "rows", 1 if m == 1 else 2 if m == 2 else 4, rows
        if parts:
            return "few", tokens, parts
        rest = -(-n // 256) * -(-m // tokens) % pairs
        return "pairs", tokens, "halves" if rest and 2 * rest <= pairs else "whole"
    return call


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes_take_the_kernels_that_they_are_there_for(plan, size):
    assert plan(*size) == SIZES[size]


def draw(rng):
    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return log(1, 4096), log(16, 30000), 16 * log(1, 900)


def test_every_kernel_has_a_size(plan):
    """What 20000 random calls are sent to is covered by the sizes whose results are compared (test_linear_kernels_gpu)."""
    rng = random.Random(1)
    assert {plan(*draw(rng)) for _ in range(20000)} == set(SIZES.values())


def ctas(size, kernel):
    m, n, _ = size
    kind, tokens, what = kernel
    if kind == "rows":
        return -(-n // (4 * what))
    if kind == "few":
        return -(-n // 128) * -(-m // tokens) * what
    return 0        # as many as the limit allows: the launch sees to it


@pytest.mark.parametrize("limit", [1, 2, 3, 16, 20, 33, 64, 100, 147])
def test_kernels_without_a_limit_of_their_own_fit_the_sm_limit(plan, limit):
    """A kernel that cannot be capped has no more CTAs than the limit has SMs."""
    rng = random.Random(limit)
    for _ in range(3000):
        size = draw(rng)
        assert ctas(size, plan(*size, limit)) <= limit, size


@pytest.mark.parametrize("limit", [20, 64, 100])
@pytest.mark.parametrize("size", [(2048, 4096, 4096), (512, 4096, 4096), (4096, 14336, 4096), (900, 1200, 256), (1, 6144, 4096)], ids=str)
def test_calls_that_fill_the_gpu_take_pairs_under_a_limit(plan, size, limit):
    """All of these do without one.  Where even the widest tiles of the kernel for few tokens are more CTAs than the limit, only pairs are left; 48 of them
    (one token, 6144 outputs) fit 64 SMs and stay with that kernel."""
    fits = ctas(size, ("few", 128, 1)) <= limit
    assert plan(*size, limit)[0] == ("few" if fits else "pairs")
