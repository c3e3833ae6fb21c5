"""Sizes at the end of 32 bits that the C entries have to refuse on the host: rounded up to whole blocks they would wrap around."""
import ctypes

import pytest

P = ctypes.c_void_p(64)
TOP = 2 ** 31 - 1


@pytest.mark.parametrize("size", [dict(K=TOP - 15, lda=TOP - 15), dict(N=TOP, ldy=TOP), dict(N=TOP - 200, ldy=TOP), dict(K=0x7FFF0010, lda=1 << 32)])
def test_fp8_gemm(lib, size):
    a = {**dict(lda=256, K=256, N=256, ldy=256), **size}
    assert lib.moe_fp8_gemm(P, a["lda"], P, 2, 1, P, P, None, 4, a["K"], a["N"], 1, P, a["ldy"], 0, 0, None, None) == -2
    assert b"too wide" in lib.moe_last_error()


@pytest.mark.parametrize("E", [TOP, TOP - 1, 5120])
def test_sort(lib, E):
    assert lib.moe_sort(P, 0, 4, E, P, P, P, P, P, 1 << 20, None) == -2


def test_sort_workspace(lib):
    """One group more than experts, also where their number is the largest there is."""
    assert lib.moe_sort_workspace(1000, 5119) >= 4 * 5120
    assert lib.moe_sort_workspace(1000, TOP) == 0 and lib.moe_sort_workspace(0, 8) == 0 and lib.moe_sort_workspace(1000, 0) == 0
