"""Tables of a sort over more than one step, and views of every kind, on the device."""
import pytest
import torch

from tilelang_moe_b200 import kernels

pytestmark = pytest.mark.gpu
T, K, E, H = 40, 3, 6, 72


def _inputs(cuda, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    ids = torch.randint(-1, E, (T, K), generator=g, device=cuda, dtype=torch.int32)
    return ids, torch.randn(T, H, generator=g, device=cuda), torch.rand(T, K, generator=g, device=cuda), torch.randn(T, H, generator=g, device=cuda)


def _step(sort, x, w, gy):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = kernels.moe_unpermute(kernels.moe_permute(x, sort), sort, w)
    return y, x, w, gy


def test_tables_that_serve_batch_after_batch(cuda, lib):
    """Written again between the steps they are the next batch's; between a forward and its backward pass that raises."""
    ids, *first = _inputs(cuda, 1)
    sort = kernels.moe_sort(ids, E)
    own = kernels.MoESort(sort.offsets.clone(), sort.perm.clone(), sort.row_of.clone(), K)
    for seed in (1, 2, 3):
        ids, *rest = _inputs(cuda, seed)
        new = kernels.moe_sort(ids, E)
        for a, b in ((own.offsets, new.offsets), (own.perm, new.perm), (own.row_of, new.row_of)):
            a.copy_(b)
        y, x, w, gy = _step(own, *rest)
        z, xz, wz, _ = _step(new, *rest)
        assert torch.equal(y, z)
        for a, b in zip(torch.autograd.grad(y, (x, w), gy), torch.autograd.grad(z, (xz, wz), gy)):
            assert torch.equal(a, b)
    y, x, w, gy = _step(own, *first)
    own.row_of.copy_(sort.row_of)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, (x, w), gy)


def test_tables_of_inference_mode(cuda, lib):
    ids, *rest = _inputs(cuda, 4)
    with torch.inference_mode():
        sort = kernels.moe_sort(ids, E)
    y, x, w, gy = _step(sort, *rest)
    z, xz, wz, _ = _step(kernels.moe_sort(ids, E), *rest)
    assert torch.equal(y, z)
    for a, b in zip(torch.autograd.grad(y, (x, w), gy), torch.autograd.grad(z, (xz, wz), gy)):
        assert torch.equal(a, b)


def test_conjugates_and_negatives(cuda, lib):
    ids, *_ = _inputs(cuda, 5)
    sort = kernels.moe_sort(ids, E)
    z = torch.randn(T, H, dtype=torch.complex64, device=cuda)
    assert torch.equal(kernels.moe_permute(z.conj(), sort), kernels.moe_permute(z.conj().resolve_conj(), sort))
    for one in (torch.randn(T, 1, dtype=torch.complex64, device=cuda).conj().imag, z.conj().imag):
        assert torch.equal(kernels.moe_permute(one, sort), kernels.moe_permute(one.resolve_neg(), sort))
        q, s = kernels.fp8_quantize(one)
        qr, sr = kernels.fp8_quantize(one.resolve_neg())
        assert torch.equal(q.view(torch.uint8), qr.view(torch.uint8)) and torch.equal(s, sr)


def test_forward_mode_is_refused(cuda, lib):
    ids, x, w, _ = _inputs(cuda, 6)
    sort = kernels.moe_sort(ids, E)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            kernels.moe_permute(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), sort)
        assert torch.equal(kernels.moe_unpermute(kernels.moe_permute(x, sort), sort, w), _step(sort, x, w, None)[0])


def test_a_sort_of_much_scratch_keeps_its_tables_only(cuda, lib):
    ids = torch.randint(0, 1500, (20000, 4), device=cuda, dtype=torch.int32)
    torch.cuda.synchronize(cuda)
    before = torch.cuda.memory_allocated(cuda)
    sort = kernels.moe_sort(ids, 1500)
    assert torch.cuda.memory_allocated(cuda) - before <= 4 * (1501 + 1502 + 2 * 80000) + 512
    # the scratch that has gone back is used by what comes next, in the order of the stream
    noise = [torch.full((1 << 18,), -1, dtype=torch.int32, device=cuda) for _ in range(4)]
    key = ids.reshape(-1).long()
    assert torch.equal(sort.perm.long(), torch.argsort(key, stable=True)) and len(noise) == 4
