"""Views whose memory holds something else than they stand for: conjugates and negatives that torch has not carried out.  Runs on
CPU: the library is replaced by one that looks at the memory it is given, and tensors in host memory pass for CUDA tensors."""
import contextlib
import ctypes

import pytest
import torch

from tilelang_moe_b200 import kernels, ops

E4M3 = torch.float8_e4m3fn


class _Looks:
    """What lies at the operands of the last call, by the order of the arguments that hold them."""
    seen = None

    @staticmethod
    def _floats(address, n):
        return list((ctypes.c_float * n).from_address(address))

    def moe_permute(self, src, stride, row_bytes, *rest):
        type(self).seen = [[v for t in range(2) for v in self._floats(src + t * stride, row_bytes // 4)]]
        return 0

    def moe_unpermute(self, rows, stride, row_of, live, weights, T, k, H, *rest):
        type(self).seen = [[v for r in range(T * k) for v in self._floats(rows + 4 * r * stride, H)], self._floats(weights, T * k)]
        return 0

    def moe_fp8_quantize_rows(self, x, stride, rows, K, *rest):
        type(self).seen = [[v for r in range(rows) for v in self._floats(x + 4 * r * stride, K)]]
        return 0

    def moe_fp8_silu_mul(self, gate, gs, up, us, rows, I, *rest):
        type(self).seen = [[v for r in range(rows) for v in self._floats(x + 4 * r * s, I)] for x, s in ((gate, gs), (up, us))]
        return 0

    def moe_fp8_quantize_blocks(self, w, E, N, K, *rest):
        type(self).seen = [self._floats(w, E * N * K)]
        return 0

    def moe_fp8_gemm(self, A, lda, sa, as_row, as_k, B, sb, offsets, rows, K, N, E, *rest):
        kb, nb = -(-K // 128), -(-N // 128)
        type(self).seen = [[self._floats(sa + 4 * (r * as_row + b * as_k), 1)[0] for r in range(rows) for b in range(kb)], self._floats(sb, E * nb * kb)]
        return 0


@pytest.fixture()
def look(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "_on", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "status_buffer", lambda device: torch.zeros(4, dtype=torch.int32))
    monkeypatch.setattr(ops._lib, "load", _Looks)
    return lambda: _Looks.seen


def _negative(*shape):
    """A float32 view that stands for the negative of what its memory holds."""
    t = torch.randn(*shape, dtype=torch.complex64).conj().imag
    assert t.is_neg()
    return t


def _values(t):
    return torch.view_as_real(t.resolve_conj()).reshape(-1).tolist() if t.is_complex() else (t + 0).reshape(-1).tolist()


def _sort():
    return kernels.MoESort(torch.tensor([0, 1, 2]).int(), torch.arange(2).int(), torch.arange(2).int(), 1)


@pytest.mark.parametrize("H", [1, 3])
def test_permute(look, H):
    for x in (_negative(2, H), torch.randn(2, H, dtype=torch.complex64).conj(), torch.randn(2, H, dtype=torch.complex64)):
        kernels.moe_permute(x, _sort())
        assert look() == [_values(x)]


@pytest.mark.parametrize("T", [1, 2])
@pytest.mark.parametrize("H", [1, 3])
def test_unpermute(look, T, H):
    rows, w = _negative(T, H), _negative(T, 1)
    sort = kernels.MoESort(torch.tensor([0, T]).int(), torch.arange(T).int(), torch.arange(T).int(), 1)
    kernels.moe_unpermute(rows, sort, w)
    assert look() == [_values(rows), _values(w)]


@pytest.mark.parametrize("shape", [(1, 1), (3, 1), (2, 3), (3,), (1,)])
def test_quantisers(look, shape):
    x, y = _negative(*shape), _negative(*shape)
    kernels.fp8_quantize(x)
    assert look() == [_values(x)]
    kernels.fp8_silu_mul(x, y)
    assert look() == [_values(x), _values(y)]
    if len(shape) == 2:
        kernels.fp8_quantize_blocks(x)
        assert look() == [_values(x)]


@pytest.mark.parametrize("M,N,K", [(1, 4, 16), (3, 4, 16), (2, 200, 256)])
def test_products(look, M, N, K):
    kb, nb = -(-K // 128), -(-N // 128)
    sa, sb = _negative(M, kb), _negative(nb, kb)
    a, b = torch.zeros(M, K).to(E4M3), torch.zeros(N, K).to(E4M3)
    kernels.fp8_gemm(a, sa, b, sb)
    assert look() == [_values(sa), _values(sb)]
    with pytest.raises(ValueError):
        kernels.fp8_gemm(a[:, :16], torch.ones(M, 1), b[:1, :16], torch.ones(1, 1), out=_negative(M, 1))
