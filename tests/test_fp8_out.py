"""Results written into a caller's tensor, as autograd has to see them.  Runs on CPU: the library is replaced by one that writes
nothing, and tensors in host memory pass for CUDA tensors."""
import contextlib

import pytest
import torch

from tilelang_moe_b200 import kernels, ops

E4M3 = torch.float8_e4m3fn


class _Library:
    calls = 0

    def moe_fp8_gemm(self, *args):
        type(self).calls += 1
        return 0


@pytest.fixture(autouse=True)
def on_host(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "status_buffer", lambda device: torch.zeros(4, dtype=torch.int32))
    monkeypatch.setattr(ops._lib, "load", _Library)
    monkeypatch.setattr(_Library, "calls", 0)


def _gemm(out):
    return kernels.fp8_gemm(torch.zeros(4, 32).to(E4M3), torch.ones(4, 1), torch.zeros(8, 32).to(E4M3), torch.ones(1, 1), out=out)


def _grouped(out):
    return kernels.fp8_grouped_gemm(torch.zeros(4, 32).to(E4M3), torch.ones(4, 1), torch.zeros(2, 8, 32).to(E4M3), torch.ones(2, 1, 1),
                                    torch.tensor([0, 1, 4]).int(), out=out)


@pytest.mark.parametrize("call", [_gemm, _grouped])
def test_a_tensor_that_autograd_has_saved(call):
    """Its backward pass has to notice, also where the result goes into a part of it."""
    for saved, part in ((torch.ones(4, 8), lambda t: t), (torch.ones(8, 16), lambda t: t[2:6, 4:12])):
        x = torch.ones_like(saved, requires_grad=True)
        y = (x * saved).sum()
        assert call(part(saved)).shape == (4, 8)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    assert _Library.calls == 2


@pytest.mark.parametrize("call", [_gemm, _grouped])
def test_a_tensor_that_requires_a_gradient(call):
    """The product has none: its values would pass for the leaf's or for a graph's that they are not of."""
    leaf = torch.ones(4, 8, requires_grad=True)
    for out in (leaf, leaf * 2):
        with pytest.raises(ValueError, match="gradient"):
            call(out)
    assert _Library.calls == 0
    with torch.no_grad():
        assert call(leaf) is leaf


def test_a_tensor_of_inference_mode():
    with torch.inference_mode():
        out = torch.ones(4, 8)
        assert _gemm(out) is out
    assert _gemm(out) is out


def test_more_experts_than_the_library_takes():
    """Refused as every other bad shape is, before the library is asked; 1024 are taken."""
    for E, taken in ((1024, True), (1025, False), (5119, False)):
        args = (torch.zeros(4, 16).to(E4M3), torch.ones(4, 1), torch.zeros(E, 1, 16).to(E4M3), torch.ones(E, 1, 1), torch.zeros(E + 1).int())
        if taken:
            kernels.fp8_grouped_gemm(*args)
        else:
            with pytest.raises(ValueError, match="1024"):
                kernels.fp8_grouped_gemm(*args)
    assert _Library.calls == 1
