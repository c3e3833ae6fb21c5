"""Arguments that the 8-bit operators have to refuse before the library sees them.  Runs on CPU: the library is replaced by
one that must not be reached, and the tensors pass for CUDA tensors."""
import ctypes

import pytest
import torch

from tilelang_moe_b200 import kernels, ops

E4M3 = torch.float8_e4m3fn


class _Unreached:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


@pytest.fixture()
def no_library(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops._lib, "load", _Unreached)


def test_cpu_tensors_are_rejected():
    x, q = torch.zeros(4, 128), torch.zeros(4, 128).to(E4M3)
    for call in (lambda: kernels.fp8_quantize(x), lambda: kernels.fp8_quantize_blocks(x), lambda: kernels.fp8_silu_mul(x, x),
                 lambda: kernels.fp8_gemm(q, torch.ones(4, 1), q, torch.ones(1, 1))):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            call()


@pytest.mark.parametrize("x", [torch.zeros(4, 128, dtype=torch.float64), torch.zeros(4, 128, dtype=torch.int32), torch.zeros(4, 0),
                               torch.zeros(())])
def test_quantize(no_library, x):
    for call in (kernels.fp8_quantize, kernels.fp8_quantize_blocks, lambda t: kernels.fp8_silu_mul(t, t)):
        with pytest.raises(ValueError):
            call(x)


def test_rows_whose_length_passes_31_bits(no_library):
    """Their length would reach the library cut to 32 bits."""
    long = torch.zeros(1).expand(2 ** 32 + 128)
    for call in (lambda: kernels.fp8_quantize(long), lambda: kernels.fp8_silu_mul(long, long), lambda: kernels.fp8_quantize_blocks(long.view(1, -1)),
                 lambda: kernels.fp8_quantize_blocks(torch.zeros(1, 1).expand(2 ** 32 + 1, 1))):
        with pytest.raises(ValueError, match="more than"):
            call()
    byte = torch.zeros(1, 1).to(E4M3)
    with pytest.raises(ValueError, match="none above"):
        kernels.fp8_gemm(byte.expand(1, 2 ** 32), torch.ones(1, 1).expand(1, 2 ** 25), byte.expand(4, 2 ** 32), torch.ones(1, 1).expand(1, 2 ** 25))


def test_blocks_need_rows(no_library):
    for x in (torch.zeros(128), torch.zeros(2, 0, 128)):
        with pytest.raises(ValueError):
            kernels.fp8_quantize_blocks(x)


@pytest.mark.parametrize("up", [torch.zeros(4, 64), torch.zeros(3, 128), torch.zeros(4, 128).half(), torch.zeros(4, 128, device="meta")])
def test_silu_mul(no_library, up):
    with pytest.raises(ValueError):
        kernels.fp8_silu_mul(torch.zeros(4, 128), up)


def _args(M=4, N=256, K=256, E=None, **changed):
    lead = () if E is None else (E,)
    args = dict(a=torch.zeros(M, K).to(E4M3), a_scale=torch.ones(M, -(-K // 128)), b=torch.zeros(*lead, N, K).to(E4M3),
                b_scale=torch.ones(*lead, -(-N // 128), -(-K // 128)))
    if E is not None:
        args["offsets"] = torch.zeros(E + 1, dtype=torch.int32)
    return {**args, **changed}


BAD = [dict(a=torch.zeros(4, 256)), dict(a=torch.zeros(4, 256).to(torch.float8_e5m2)), dict(a=torch.zeros(256).to(E4M3)),
       dict(a=torch.zeros(4, 128).to(E4M3)), dict(a_scale=torch.ones(4, 1)), dict(a_scale=torch.ones(3, 2)), dict(a_scale=torch.ones(4, 2).half()),
       dict(a_scale=torch.ones(4, 2, device="meta")), dict(out_dtype=torch.float64), dict(out_dtype=torch.float8_e4m3fn),
       dict(out=torch.zeros(4, 255)), dict(out=torch.zeros(4, 256, dtype=torch.float64)), dict(out=torch.zeros(256, 4).T),
       dict(out=torch.zeros(1, 256).expand(4, 256)), dict(out=torch.zeros(4, 256), out_dtype=torch.bfloat16), dict(out=torch.zeros(4, 256, device="meta"))]


@pytest.mark.parametrize("change", BAD + [dict(b=torch.zeros(256, 128).to(E4M3)), dict(b=torch.zeros(1, 256, 256).to(E4M3)), dict(b=torch.zeros(256, 256)),
                                          dict(b_scale=torch.ones(2, 1)), dict(b_scale=torch.ones(1, 2, 2)), dict(b_scale=torch.ones(2, 2).double())])
def test_gemm(no_library, change):
    with pytest.raises(ValueError):
        kernels.fp8_gemm(**_args(**change))


@pytest.mark.parametrize("change", BAD + [dict(b=torch.zeros(256, 256).to(E4M3)), dict(b_scale=torch.ones(2, 2)), dict(b_scale=torch.ones(4, 2, 2)),
                                          dict(offsets=None), dict(offsets=torch.zeros(3, dtype=torch.int32)),
                                          dict(offsets=torch.zeros(4, dtype=torch.int64)), dict(offsets=torch.zeros(4, dtype=torch.int32, device="meta"))])
def test_grouped_gemm(no_library, change):
    with pytest.raises(ValueError):
        kernels.fp8_grouped_gemm(**_args(E=3, **change))


@pytest.mark.parametrize("K", [8, 24, 257])
def test_inner_dimension(no_library, K):
    with pytest.raises(ValueError, match="multiple of 16"):
        kernels.fp8_gemm(**_args(K=K))


def test_c_entries(lib):
    """Refused on the host, before any CUDA call."""
    p = ctypes.c_void_p(64)

    def gemm(A=p, lda=256, as_row=2, as_k=1, B=p, offsets=None, rows=4, K=256, N=256, E=1, Y=p, ldy=256, out=0):
        return lib.moe_fp8_gemm(A, lda, p, as_row, as_k, B, p, offsets, rows, K, N, E, Y, ldy, out, 0, None, None)

    assert gemm(rows=0, A=None) == 0
    for bad in (dict(A=None), dict(B=None), dict(Y=None), dict(lda=128), dict(lda=264), dict(as_row=-1), dict(as_k=-1), dict(K=0), dict(K=24),
                dict(N=0), dict(E=0), dict(E=2), dict(ldy=255), dict(out=3), dict(rows=-1), dict(A=ctypes.c_void_p(65)), dict(B=ctypes.c_void_p(72))):
        assert gemm(**bad) == -1, bad
    assert gemm(E=1025, offsets=p) == -2 and gemm(rows=1 << 31) == -2
    assert lib.moe_fp8_quantize_rows(None, 128, 4, 128, 0, p, p, None) == -1
    assert lib.moe_fp8_quantize_rows(p, 128, 4, 0, 0, p, p, None) == -1
    assert lib.moe_fp8_quantize_rows(p, 128, 4, 128, 3, p, p, None) == -1
    assert lib.moe_fp8_quantize_rows(None, 128, 0, 128, 0, None, None, None) == 0
    assert lib.moe_fp8_silu_mul(p, 128, None, 128, 4, 128, 0, p, p, None) == -1
    assert lib.moe_fp8_quantize_blocks(None, 1, 4, 128, 0, p, p, None) == -1
    assert lib.moe_fp8_quantize_blocks(p, 1, 0, 128, 0, p, p, None) == -1
    assert lib.moe_fp8_quantize_blocks(p, 1 << 40, 128, 128, 0, p, p, None) == -2
