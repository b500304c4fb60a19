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
    """(m, n, k[, sms, pairs]) -> the entries of linear_sizes.SIZES."""
    library = str(tmp_path_factory.mktemp("plan") / "linear_plan_host.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, "-o", library, os.path.join(HERE, "host_model", "linear_plan_host.cpp")], check=True)
    host = C.CDLL(library)

    def call(m, n, k, sms=SMS, pairs=PAIRS):
        out = (C.c_uint32 * 3)()
        host.host_linear_plan(m, n, k, sms, pairs, out)
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


def test_every_kernel_has_a_size(plan):
    """What 20000 random calls are sent to is covered by the sizes whose results are compared (test_linear_kernels_gpu)."""
    rng = random.Random(1)

    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    taken = {plan(log(1, 4096), log(16, 30000), 16 * log(1, 900)) for _ in range(20000)}
    assert taken == set(SIZES.values())
