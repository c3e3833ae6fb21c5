"""8-bit operands (e4m3 with an fp32 scale per block of 128) and the products of them.

    q, scale = fp8_quantize(x)                  one scale per 128 elements of a row: activations
    q, scale = fp8_quantize_blocks(w)           one scale per 128 x 128: weights, laid out once
    q, scale = fp8_silu_mul(gate, up)           SiLU(gate) * up into 8 bits, between an expert's two products
    y = fp8_gemm(a, a_scale, b, b_scale)        dense: a [M, K], b [N, K]
    y = fp8_grouped_gemm(a, a_scale, b, b_scale, offsets)   rows sorted by expert (moe_sort, moe_permute): b [E, N, K]

q * scale stands for x to within half an e4m3 step.  None of these has a gradient: the results are detached.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, ops

GROUP = 128
_WIDEST = 2 ** 31 - 2 ** 16       # the library counts the elements of a row in 32 bits
_MAX_EXPERTS = 1024               # the product keeps its table of groups in shared memory
E4M3 = torch.float8_e4m3fn
_OUT_DTYPES = (None, torch.bfloat16, torch.float16, torch.float32)
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # MOE_DTYPE_* of include/moe_b200.h


def _groups(n: int) -> int:
    return (n + GROUP - 1) // GROUP


def _rows2(x: torch.Tensor) -> torch.Tensor:
    """x [..., K] as a matrix of packed rows at one non-negative stride; a copy where its strides do not allow that."""
    x = ops._carried_out(x)
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _input_type(x: torch.Tensor, least_dims: int) -> int:
    if x.dtype not in _DTYPES:
        raise ValueError("8-bit values are made from bfloat16, float16 or float32")
    if x.dim() < least_dims or x.shape[-1] < 1 or (least_dims == 2 and x.shape[-2] < 1):
        raise ValueError(f"expected at least {least_dims} dimension(s), none of the last {least_dims} empty, got {tuple(x.shape)}")
    if max(x.shape[-least_dims:]) > _WIDEST:
        raise ValueError(f"rows of more than {_WIDEST} elements: cut them into groups of {GROUP} first")
    return _DTYPES[x.dtype]


def fp8_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] -> (e4m3 [..., K], scale float32 [..., ceil(K / 128)]): the largest magnitude of each 128 becomes 448."""
    ops._need_cuda(x)
    dt = _input_type(x, 1)
    K = x.shape[-1]
    q = x.new_empty(x.shape, dtype=E4M3)
    scale = x.new_empty((*x.shape[:-1], _groups(K)), dtype=torch.float32)
    rows, dev = _rows2(x), x.device
    with ops._on(dev):
        rc = _lib.load().moe_fp8_quantize_rows(rows.data_ptr(), _stride(rows), rows.shape[0], K, dt, q.data_ptr(), scale.data_ptr(),
                                               ops._stream())
    _lib.check(rc, "moe_fp8_quantize_rows")
    ops._after(dev)
    return q, scale


def fp8_silu_mul(gate: torch.Tensor, up: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp8_quantize(silu(gate) * up), the product in fp32 and not rounded in between.  gate, up [..., I] of one type, the
    halves of one product's rows for instance."""
    ops._need_cuda(gate, up)
    dt = _input_type(gate, 1)
    if up.shape != gate.shape or up.dtype != gate.dtype or up.device != gate.device:
        raise ValueError("gate and up must have one shape and type and be on one device")
    I = gate.shape[-1]
    q = gate.new_empty(gate.shape, dtype=E4M3)
    scale = gate.new_empty((*gate.shape[:-1], _groups(I)), dtype=torch.float32)
    g, u, dev = _rows2(gate), _rows2(up), gate.device
    with ops._on(dev):
        rc = _lib.load().moe_fp8_silu_mul(g.data_ptr(), _stride(g), u.data_ptr(), _stride(u), g.shape[0], I, dt, q.data_ptr(),
                                          scale.data_ptr(), ops._stream())
    _lib.check(rc, "moe_fp8_silu_mul")
    ops._after(dev)
    return q, scale


def fp8_quantize_blocks(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """w [..., N, K] -> (e4m3 [..., N, K], scale float32 [..., ceil(N / 128), ceil(K / 128)])."""
    ops._need_cuda(w)
    dt = _input_type(w, 2)
    w = ops._carried_out(w).contiguous()
    N, K = w.shape[-2:]
    q = torch.empty(w.shape, dtype=E4M3, device=w.device)
    scale = torch.empty(*w.shape[:-2], _groups(N), _groups(K), dtype=torch.float32, device=w.device)
    with ops._on(w.device):
        rc = _lib.load().moe_fp8_quantize_blocks(ops._ptr(w), w.numel() // (N * K), N, K, dt, ops._ptr(q), ops._ptr(scale), ops._stream())
    _lib.check(rc, "moe_fp8_quantize_blocks")
    ops._after(w.device)
    return q, scale


def _product(a, a_scale, b, b_scale, E, offsets, out_dtype, out) -> torch.Tensor:
    """b [N, K] and b_scale without their leading E where offsets is None."""
    ops._need_cuda(a, a_scale, b, b_scale, offsets, out)
    if a.dtype != E4M3 or b.dtype != E4M3:
        raise ValueError("a and b must be float8_e4m3fn")
    if a.dim() != 2:
        raise ValueError("a must be [M, K]")
    M, K = a.shape
    N, K2 = b.shape[-2:]
    if K2 != K:
        raise ValueError(f"inner dimensions differ: a has K={K}, b has K={K2}")
    if K < 16 or K % 16 or N < 1 or E < 1 or max(K, N) > _WIDEST:
        raise ValueError(f"K={K} must be a positive multiple of 16, N={N} and E={E} positive, none above {_WIDEST}")
    if E > _MAX_EXPERTS:
        raise ValueError(f"E={E} exceeds the {_MAX_EXPERTS} experts of one product")
    kb, nb = _groups(K), _groups(N)
    if a_scale.dtype != torch.float32 or a_scale.shape != (M, kb):
        raise ValueError(f"a_scale must be float32 [{M}, {kb}]")
    if b_scale.dtype != torch.float32 or b_scale.shape != ((nb, kb) if offsets is None else (E, nb, kb)):
        raise ValueError(f"b_scale must be float32 [{'' if offsets is None else f'{E}, '}{nb}, {kb}]")
    dev = a.device
    for t in (a_scale, b, b_scale, offsets, out):
        if t is not None and t.device != dev:
            raise ValueError(f"all tensors must be on one device, not on {dev} and {t.device}")
    if offsets is not None:
        if offsets.dtype != torch.int32 or offsets.shape != (E + 1,):
            raise ValueError(f"offsets must be int32 [{E + 1}]")
        offsets = offsets.contiguous()
    fresh = out is None
    if fresh:
        if out_dtype not in _OUT_DTYPES:
            raise ValueError("out_dtype must be bfloat16, float16 or float32")
        out = a.new_empty((M, N), dtype=out_dtype or torch.bfloat16)
    else:
        if out.shape != (M, N) or out.dtype not in _DTYPES or (M > 0 and N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
            raise ValueError(f"out must be [{M}, {N}] in bfloat16, float16 or float32 with packed rows that do not overlap")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("out requires a gradient, and these products have none")
        if out.is_neg():
            raise ValueError("out is the negative of what its memory holds")
        if out_dtype is not None and out_dtype != out.dtype:
            raise ValueError(f"out is {out.dtype}, not {out_dtype}")
    lda = _stride(a)
    if a.stride(1) != 1 or a.data_ptr() & 15 or lda < K or lda % 16:
        a = a.clone(memory_format=torch.contiguous_format)
        lda = K
    if not b.is_contiguous() or b.data_ptr() & 15:
        b = b.clone(memory_format=torch.contiguous_format)
    a_scale, b_scale = ops._carried_out(a_scale), ops._carried_out(b_scale).contiguous()
    lib = _lib.load()
    with ops._on(dev):
        rc = lib.moe_fp8_gemm(a.data_ptr(), lda, a_scale.data_ptr(), *a_scale.stride(), b.data_ptr(), b_scale.data_ptr(),
                              ops._ptr(offsets), M, K, N, E, out.data_ptr(), N if fresh else _stride(out), _DTYPES[out.dtype], int(fresh),
                              ops.status_buffer(dev).data_ptr(), ops._stream())
    _lib.check(rc, "moe_fp8_gemm")
    if not fresh:
        torch.autograd.graph.increment_version(out)      # what autograd has saved of it is no longer there
    ops._after(dev)
    return out


def fp8_gemm(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
             out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [M, N] = (a * a_scale) @ (b * b_scale).T: a e4m3 [M, K] with a_scale float32 [M, ceil(K / 128)] (fp8_quantize), b e4m3
    [N, K] with b_scale float32 [ceil(N / 128), ceil(K / 128)] (fp8_quantize_blocks); K a multiple of 16.  Accumulated in
    fp32, rounded once to out_dtype: bfloat16 (the default), float16 or float32."""
    if b.dim() != 2:
        raise ValueError("b must be [N, K]")
    return _product(a, a_scale, b, b_scale, 1, None, out_dtype, out)


def fp8_grouped_gemm(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor, offsets: torch.Tensor,
                     out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[r] = fp8_gemm with b[e] for the rows offsets[e] .. offsets[e + 1] - 1 of every expert e: b e4m3 [E, N, K] with b_scale
    float32 [E, ceil(N / 128), ceil(K / 128)], offsets int32 [E + 1] on the device (no host synchronisation); E at most 1024, where
    moe_sort takes 5119.  Rows of no expert (behind offsets[E]) are zero in a new tensor and left as they were in ``out``."""
    if offsets is None or b.dim() != 3:
        raise ValueError("b must be [E, N, K] and offsets int32 [E + 1]")
    return _product(a, a_scale, b, b_scale, b.shape[0], offsets, out_dtype, out)
