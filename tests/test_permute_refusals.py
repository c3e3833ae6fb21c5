"""Arguments that the sort, permute and unpermute have to refuse before the library sees them.  Runs on CPU: the library is
replaced by one that must not be reached, and the tensors pass for CUDA tensors."""
import ctypes

import pytest
import torch

from tilelang_moe_b200 import kernels, ops


class _Unreached:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture()
def no_library(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops._lib, "load", _Unreached)


def _sort(T=4, k=2, E=3, device="cpu"):
    one = torch.zeros(T * k, dtype=torch.int32, device=device)
    return kernels.MoESort(torch.zeros(E + 1, dtype=torch.int32, device=device), one, one, k)


def test_cpu_tensors_are_rejected():
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.moe_sort(torch.zeros(4, 2, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.moe_permute(torch.zeros(4, 8), _sort())
    with pytest.raises(ValueError, match="CUDA tensors only"):
        kernels.moe_unpermute(torch.zeros(8, 8), _sort())


@pytest.mark.parametrize("ids,E", [(torch.zeros(4, 2), 3), (torch.zeros(4, 2, dtype=torch.int16), 3), (torch.zeros(4, 2, 1, dtype=torch.int32), 3),
                                   (torch.zeros(4, 0, dtype=torch.int32), 3), (torch.zeros(4, 2, dtype=torch.int32), 0), (torch.zeros(4, 2, dtype=torch.int32), 5120),
                                   (torch.zeros(4, 2, dtype=torch.int32), 2 ** 33)])
def test_sort(no_library, ids, E):
    with pytest.raises(ValueError):
        kernels.moe_sort(ids, E)


@pytest.mark.parametrize("offsets,perm,row_of,k", [
    (torch.zeros(4), torch.zeros(8, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), 2),
    (torch.zeros(1, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), 2),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int64), torch.zeros(8, dtype=torch.int32), 2),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(7, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), 2),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(16, dtype=torch.int32)[::2], 2),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32), 2),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), 3),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), 0),
    (torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32, device="meta"), torch.zeros(8, dtype=torch.int32), 2)])
def test_tables(offsets, perm, row_of, k):
    with pytest.raises(ValueError):
        kernels.MoESort(offsets, perm, row_of, k)


@pytest.mark.parametrize("x", [torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(4), torch.zeros(4, 0), torch.zeros(4, 8, device="meta"),
                               torch.zeros(4, 8, dtype=torch.float64, requires_grad=True)])
def test_permute(no_library, x):
    with pytest.raises(ValueError):
        kernels.moe_permute(x, _sort())


@pytest.mark.parametrize("rows,weights", [
    (torch.zeros(7, 8), None), (torch.zeros(9, 8), None), (torch.zeros(8), None), (torch.zeros(8, 0), None),
    (torch.zeros(8, 8, dtype=torch.float64), None), (torch.zeros(8, 8, dtype=torch.uint8), None), (torch.zeros(8, 8, device="meta"), None),
    (torch.zeros(8, 8), torch.zeros(4, 2).half()), (torch.zeros(8, 8), torch.zeros(4, 3)), (torch.zeros(8, 8), torch.zeros(8)),
    (torch.zeros(8, 8), torch.zeros(4, 2, device="meta"))])
def test_unpermute(no_library, rows, weights):
    with pytest.raises(ValueError):
        kernels.moe_unpermute(rows, _sort(), weights)


def test_c_entries(lib):
    """Refused on the host, before any CUDA call."""
    p = ctypes.c_void_p(64)
    none = None
    assert lib.moe_sort(none, 0, 4, 3, p, p, p, p, p, 1 << 20, none) == -1
    assert lib.moe_sort(p, 0, 4, 0, p, p, p, p, p, 1 << 20, none) == -1
    assert lib.moe_sort(p, 0, 4, 3, p, p, none, p, p, 1 << 20, none) == -1
    assert lib.moe_sort(p, 0, 4, 3, p, p, p, p, none, 0, none) == -3
    assert lib.moe_sort(p, 0, 4, 5120, p, p, p, p, p, 1 << 20, none) == -2 and lib.moe_sort(p, 0, 4, 5119, p, p, p, p, none, 0, none) == -3
    assert lib.moe_sort(p, 0, 4, 8000, p, p, p, p, p, 1 << 20, none) == -2 and b"too large" in lib.moe_last_error()
    assert lib.moe_permute(none, 16, 16, p, p, 4, 2, p, none) == -1
    assert lib.moe_permute(p, 16, 0, p, p, 4, 2, p, none) == -1
    assert lib.moe_permute(p, -16, 16, p, p, 4, 2, p, none) == -1
    assert lib.moe_permute(p, 16, 16, p, p, 1 << 30, 2, p, none) == -2
    assert lib.moe_permute(none, 16, 16, none, none, 0, 2, none, none) == 0
    assert lib.moe_permute(p, 16, 16, p, p, 1 << 62, 8, p, none) == -2      # T * k would wrap around
    assert lib.moe_unpermute(p, 8, p, p, none, 1 << 62, 8, 8, 0, p, none) == -2
    assert lib.moe_unpermute(p, 8, p, p, none, 4, 2, 8, 3, p, none) == -1
    assert lib.moe_unpermute(p, 8, p, none, none, 4, 2, 8, 0, p, none) == -1
    assert lib.moe_unpermute_grad(p, 8, none, 8, p, p, p, 4, 2, 8, 0, p, p, none) == -1
    assert lib.moe_unpermute_grad(p, 8, none, 8, p, p, none, 4, 2, 8, 0, p, none, none) == -1
