"""What autograd has to see of the sort's operators.  Runs on CPU: tensors in host memory pass for CUDA tensors, and the library is
replaced by loops over that memory."""
import contextlib
import ctypes

import pytest
import torch

from tilelang_moe_b200 import kernels, ops


def _floats(address, *shape):
    n = 1
    for s in shape:
        n *= s
    return torch.frombuffer((ctypes.c_float * max(n, 1)).from_address(address), dtype=torch.float32)[:n].view(shape) if n else torch.zeros(shape)


def _ints(address, n):
    return list((ctypes.c_int32 * n).from_address(address))


class _HostLibrary:
    """fp32 and packed rows only."""

    def moe_permute(self, src, stride, row_bytes, row_of, live, T, k, dst, stream):
        H = row_bytes // 4
        assert stride == row_bytes
        x, rows = _floats(src, T, H), _floats(dst, T * k, H)
        for i, r in enumerate(_ints(row_of, T * k)):
            rows[r] = x[i // k] if r < _ints(live, 1)[0] else 0
        return 0

    def moe_unpermute(self, src, stride, row_of, live, weights, T, k, H, dtype, out, stream):
        assert stride == H and dtype == 2
        rows, y = _floats(src, T * k, H), _floats(out, T, H)
        w = _floats(weights, T * k) if weights else torch.ones(T * k)
        y.zero_()
        for i, r in enumerate(_ints(row_of, T * k)):
            if r < _ints(live, 1)[0]:
                y[i // k] += w[i] * rows[r]
        return 0

    def moe_unpermute_grad(self, gy, gy_stride, src, stride, row_of, live, weights, T, k, H, dtype, g_rows, g_w, stream):
        assert gy_stride == H and dtype == 2
        gy, w = _floats(gy, T, H), _floats(weights, T * k)
        for i, r in enumerate(_ints(row_of, T * k)):
            has = r < _ints(live, 1)[0]
            if g_rows:
                _floats(g_rows, T * k, H)[r] = w[i] * gy[i // k] if has else 0
            if g_w:
                _floats(g_w, T * k)[i] = (_floats(src, T * k, H)[r] * gy[i // k]).sum() if has else 0
        return 0


@pytest.fixture()
def on_host(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops._lib, "load", _HostLibrary)


def _sort(ids, E):
    T, k = ids.shape
    key = torch.where((ids < 0) | (ids >= E), E, ids).reshape(-1)
    perm = torch.argsort(key, stable=True)
    row_of = torch.empty_like(perm)
    row_of[perm] = torch.arange(T * k)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(key, minlength=E + 1)[:E].cumsum(0)])
    return kernels.MoESort(offsets.int(), perm.int(), row_of.int(), k)


IDS = torch.tensor([[0, 2], [1, 0], [2, -1], [1, 1]])
OTHER = torch.tensor([[2, 1], [0, 0], [-1, 1], [2, 0]])
T, K, E, H = 4, 2, 3, 5


def _loss(sort, x, w, scale):
    return kernels.moe_unpermute(kernels.moe_permute(x, sort) * scale, sort, w)


def _operands():
    g = torch.Generator().manual_seed(0)
    return (torch.randn(T, H, generator=g, requires_grad=True), torch.rand(T, K, generator=g, requires_grad=True), torch.randn(T * K, 1, generator=g),
            torch.randn(T, H, generator=g))


def _formula(ids, x, w, scale):
    s = _sort(ids, E)
    rows = x.double()[s.perm.long() // K] * scale.double()
    rows = torch.where((torch.arange(T * K) < s.offsets[-1]).unsqueeze(1), rows, 0)
    return (rows[s.row_of.long()].view(T, K, H) * w.double().unsqueeze(2)).sum(1)


def test_the_library_on_the_host_does_what_the_formula_says(on_host):
    x, w, scale, gy = _operands()
    y = _loss(_sort(IDS, E), x, w, scale)
    want = _formula(IDS, x, w, scale)
    assert torch.allclose(y.double(), want, rtol=1e-6, atol=1e-6)
    for a, b in zip(torch.autograd.grad(y, (x, w), gy), torch.autograd.grad(want, (x, w), gy.double())):
        assert torch.allclose(a, b.float(), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("table", ["offsets", "row_of"])
@pytest.mark.parametrize("call", ["permute", "unpermute", "weighted"])
def test_tables_written_again_before_the_backward_pass(on_host, call, table):
    """Gradients by the next batch's tables would be silently wrong."""
    x, w, _, gy = _operands()
    sort, new = _sort(IDS, E), _sort(OTHER, E)
    leaf, g = (x, torch.randn(T * K, H)) if call == "permute" else (torch.randn(T * K, H, requires_grad=True), gy)
    y = kernels.moe_permute(leaf, sort) if call == "permute" else kernels.moe_unpermute(leaf, sort, w if call == "weighted" else None)
    getattr(sort, table).copy_(getattr(new, table))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, g)


def test_tables_written_again_after_the_backward_pass(on_host):
    """One set of tables for batch after batch."""
    x, w, scale, gy = _operands()
    sort = _sort(IDS, E)
    for ids in (IDS, OTHER, IDS):
        for a, b in ((sort.offsets, _sort(ids, E).offsets), (sort.perm, _sort(ids, E).perm), (sort.row_of, _sort(ids, E).row_of)):
            a.copy_(b)
        got = torch.autograd.grad(_loss(sort, x, w, scale), (x, w), gy)
        for a, b in zip(got, torch.autograd.grad(_formula(ids, x, w, scale), (x, w), gy.double())):
            assert torch.allclose(a, b.float(), rtol=1e-5, atol=1e-6)


def test_tables_made_in_inference_mode(on_host):
    """Routing computed there serves a training step: such tables have no version, so the step keeps its own."""
    x, w, scale, gy = _operands()
    with torch.inference_mode():
        sort = _sort(IDS, E)
    y = _loss(sort, x, w, scale)
    with torch.inference_mode():
        sort.row_of.copy_(_sort(OTHER, E).row_of)
    for a, b in zip(torch.autograd.grad(y, (x, w), gy), torch.autograd.grad(_formula(IDS, x, w, scale), (x, w), gy.double())):
        assert torch.allclose(a, b.float(), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("call", ["permute", "rows", "weights"])
def test_forward_mode_is_refused(on_host, call, grad):
    """Without a rule for it the tangent would be lost, which reads as a derivative of zero."""
    sort = _sort(IDS, E)
    x, rows, w = torch.randn(T, H), torch.randn(T * K, H), torch.rand(T, K)
    with torch.set_grad_enabled(grad), torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))

        with pytest.raises((RuntimeError, NotImplementedError)):
            if call == "permute":
                kernels.moe_permute(dual(x), sort)
            elif call == "rows":
                kernels.moe_unpermute(dual(rows), sort, w)
            else:
                kernels.moe_unpermute(rows, sort, dual(w))
        # what has no tangent is computed there as anywhere else
        assert torch.equal(kernels.moe_unpermute(kernels.moe_permute(x, sort), sort, w).detach(), _loss(sort, x, w, 1.0).detach())
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: kernels.moe_permute(t, sort), (x,), (torch.ones_like(x),))


def test_gradients_of_gradients_are_refused(on_host):
    x, w, scale, gy = _operands()
    y = _loss(_sort(IDS, E), x, w, scale)
    gx, = torch.autograd.grad(y, x, gy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
