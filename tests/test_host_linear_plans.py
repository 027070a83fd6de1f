"""The table of sizes that reach every kernel of the 4-bit product and the gated projection: no GPU work."""
import ctypes
import random

import pytest

import linear_plans as P
from usaf_amd import _native as N


@pytest.mark.parametrize("case", P.CASES, ids=lambda c: "-".join(map(str, c[:5])))
def test_sizes_take_their_kernels(case):
    assert P.plans(*case[:5]) == case[5]


def test_no_kernel_is_left_out():
    """Random sizes of every kind take no kernel that the table lacks."""
    known = set().union(*(P.kernels(c[0], c[4], c[5]) for c in P.CASES))
    rng = random.Random(0)

    def log(low, high):
        return int(round(low * (high / low) ** rng.random()))

    for _ in range(8000):
        call, checkpoint = rng.choice([("q4", None), ("gated4", None), ("gated4", "fp8"), ("gated16", None), ("gated16", "fp8")])
        m, n, k = log(1, 70000), log(1, 40000), log(1, 20000)
        if call != "gated16":
            k = -(-k // 128) * 128
        elif rng.random() < 0.5:
            m, n, k = -(-m // 64) * 64, -(-n // 32) * 32, -(-k // 8) * 8
        assert P.kernels(call, checkpoint, P.plans(call, m, n, k, checkpoint)) <= known, (call, m, n, k, checkpoint)


def test_refusals():
    lib, plan = N.load(), (ctypes.c_int32 * 4)()
    for bad in [(0, 64, 128, 0), (-1, 64, 128, 0), (1, 0, 128, 0), (1, 64, 1 << 23, 1)]:
        assert lib.usaf_hip_q4_linear_plan(*bad, plan) == N.USAF_ERR_INVALID
    for bad in [(0, 64, 128, 0, 0, 0), (1, 64, 128, 0, 5, 0), (1, 64, 128, 0, -1, 0), (1, 64, 128, 0, 1, 1), (1, 64, 128, 0, 2, 0)]:
        assert lib.usaf_hip_gated_plan(*bad, plan) == N.USAF_ERR_INVALID
    assert lib.usaf_hip_q4_linear_plan(1, 64, 128, 0, None) == N.USAF_ERR_INVALID
    assert lib.usaf_hip_gated_plan(1, 64, 128, 0, 0, 0, None) == N.USAF_ERR_INVALID
