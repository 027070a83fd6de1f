"""Limits of the gated projection's C entry points that its argument checks hold: no GPU work."""
import ctypes

import pytest

from usaf_amd import _native as N

LIMIT = 1 << 22  # values between two rows, as everywhere in these entry points


def _bwd(lib, m, inter, k, ldx, dx=None, dw=ctypes.c_void_p(4096), size=1 << 40):
    p = ctypes.c_void_p(4096)
    return lib.usaf_hip_gated_bwd(p, N.BF16, m, inter, k, p, None, None, None, p, p, ldx, dx, dw, p, size, None)


@pytest.mark.parametrize("m,inter,k", [(4, 32, 256), (1088, 1056, 2056)])  # x copied, x read in place
@pytest.mark.parametrize("ldx", [LIMIT + 8, 1 << 25, 1 << 31, 1 << 40])
def test_rows_too_far_apart_for_a_weight_gradient(m, inter, k, ldx):
    """Offsets of x's rows are taken in 32 bits where it is read in place."""
    lib = N.load()
    # (no workspace: a call that passes the check on ldx is still refused, for the workspace, in front of any launch)
    assert _bwd(lib, m, inter, k, ldx, size=0) == N.USAF_ERR_INVALID
    assert "ldx" in N.last_error()


@pytest.mark.parametrize("m,inter,k", [(4, 32, 256), (1088, 1056, 2056)])
def test_rows_at_the_limit_and_rows_that_nobody_reads(m, inter, k):
    lib, p = N.load(), ctypes.c_void_p(4096)
    assert _bwd(lib, m, inter, k, LIMIT, size=0) == N.USAF_ERR_INVALID
    assert "workspace" in N.last_error()
    assert _bwd(lib, m, inter, k, 1 << 40, dx=p, dw=None, size=0) == N.USAF_ERR_INVALID
    assert "workspace" in N.last_error()


def test_a_weight_gradient_of_no_rows_is_the_callers_to_clear():
    """Documented: the entry point writes nothing then, in memory of the host's here (gated_linear gives zeros)."""
    lib = N.load()
    dw = (ctypes.c_uint16 * 4096)(*([7] * 4096))
    at = ctypes.cast(dw, ctypes.c_void_p)
    assert _bwd(lib, 0, 32, 64, 64, dw=at, size=0) == N.USAF_OK
    assert list(dw) == [7] * 4096
