"""Tokens sorted by expert and back, differentiable.

    sort = moe_sort(ids, n_experts)                  tables of T tokens with k entries each, no host synchronisation
    rows = moe_permute(x, sort)                      [T*k, H]: a copy of its token's row for every entry, by expert
    y    = moe_unpermute(rows_out, sort, weights)    [T, H]: the k rows of a token, weighed and added up

Rows sort.offsets[e] .. sort.offsets[e+1] - 1 belong to expert e.  An id outside [0, n_experts) marks an entry without an
expert (a padded token, an entry over an expert's capacity): its row lies behind offsets[n_experts], holds zeros, and adds
nothing; its gradients are zero.  Results and gradients are computed without atomics, in a fixed order.  Gradients are those of
the backward pass; forward mode is refused.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib, ops

_MAX_EXPERTS = 5119        # groups that the library's counting kernel has shared memory for, but the one of no expert
# Bytes of scratch that a sort may keep beside its tables.  An allocation of its own costs a call 1.9 of 15 us, which counts in a step
# of few tokens; a training step's scratch (16000 entries of 256 experts: 125 KB) would double what lives until the backward pass.
_SCRATCH_KEPT = 64 * 1024
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}   # MOE_DTYPE_* of include/moe_b200.h


@dataclass(frozen=True, eq=False)
class MoESort:
    """Tables of one routing: contiguous int32 tensors on one device, usable by any number of permutes and unpermutes.  A backward
    pass reads offsets and row_of again: it raises where they have been written to in between."""
    offsets: torch.Tensor    # [E + 1]: first row of every expert; offsets[E] rows hold an entry
    perm: torch.Tensor       # [T * k]: entry t * k + j at each sorted row
    row_of: torch.Tensor     # [T * k]: sorted row of each entry
    k: int                   # entries per token

    def __post_init__(self):
        offsets, perm, row_of = self.offsets, self.perm, self.row_of
        if not (offsets.dtype is perm.dtype is row_of.dtype is torch.int32 and offsets.dim() == perm.dim() == row_of.dim() == 1
                and offsets.is_contiguous() and perm.is_contiguous() and row_of.is_contiguous() and offsets.numel() > 1):
            raise ValueError("offsets, perm and row_of must be contiguous int32 vectors, offsets of two entries at least")
        n = row_of.numel()
        if self.k < 1 or n % self.k or perm.numel() != n:
            raise ValueError(f"perm and row_of must have {self.k} entries for each token")
        if not (offsets.device == perm.device == row_of.device):
            raise ValueError("the tables of a sort must be on one device")

    @classmethod
    def _of(cls, offsets, perm, row_of, k) -> "MoESort":
        """Tables that moe_sort has just laid out: as they should be without looking."""
        s = object.__new__(cls)
        s.__dict__.update(offsets=offsets, perm=perm, row_of=row_of, k=k)
        return s

    @property
    def n_experts(self) -> int:
        return self.offsets.numel() - 1

    @property
    def tokens(self) -> int:
        return self.row_of.numel() // self.k


def moe_sort(topk_ids: torch.Tensor, n_experts: int) -> MoESort:
    """Stable sort of the entries of topk_ids [T, k] (or [T]; int32 or int64) by expert."""
    ops._need_cuda(topk_ids)
    if topk_ids.dtype not in (torch.int64, torch.int32):
        raise ValueError("expert ids must be int64 or int32")
    if topk_ids.dim() not in (1, 2) or (topk_ids.dim() == 2 and topk_ids.shape[1] < 1):
        raise ValueError("expert ids must be [T] or [T, k]")
    if not 1 <= n_experts <= _MAX_EXPERTS:
        raise ValueError(f"n_experts={n_experts} must be in [1, {_MAX_EXPERTS}]")
    ids = topk_ids.contiguous()
    n, dev = ids.numel(), ids.device
    lib = _lib.load()
    # One allocation: counts [E + 1], offsets [E + 2], perm [n], row_of [n], and the scratch of the call where that is little.  More of
    # it goes when the call returns: the tables live until the backward pass.
    need = lib.moe_sort_workspace(n, n_experts)
    with_tables = (need + 3) // 4 if need <= _SCRATCH_KEPT else 0
    buf = torch.empty(2 * n_experts + 3 + 2 * n + with_tables, dtype=torch.int32, device=dev)
    _, offsets, _, perm, row_of, ws = buf.split_with_sizes((n_experts + 1, n_experts + 1, 1, n, n, with_tables))
    if need > _SCRATCH_KEPT:
        ws = torch.empty((need + 3) // 4, dtype=torch.int32, device=dev)
    with ops._on(dev):
        rc = lib.moe_sort(ids.data_ptr(), int(ids.dtype == torch.int64), n, n_experts, buf.data_ptr(), offsets.data_ptr(),
                          perm.data_ptr(), row_of.data_ptr(), ws.data_ptr(), need, ops._stream())
    _lib.check(rc, "moe_sort")
    ops._after(dev)
    return MoESort._of(offsets, perm, row_of, ids.shape[1] if ids.dim() == 2 else 1)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with packed rows at any non-negative stride."""
    t = ops._carried_out(t)
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _live(sort: MoESort) -> int:
    """Address of offsets[E]: the rows that hold an entry."""
    return sort.offsets.data_ptr() + 4 * (sort.offsets.numel() - 1)


def _permute(x: torch.Tensor, sort: MoESort) -> torch.Tensor:
    x = _rows(x)
    T, H = x.shape
    k, w, dev = sort.k, x.element_size(), x.device
    out = x.new_empty((T * k, H))
    with ops._on(dev):
        rc = _lib.load().moe_permute(x.data_ptr(), _stride(x) * w, H * w, sort.row_of.data_ptr(), _live(sort), T, k, out.data_ptr(),
                                     ops._stream())
    _lib.check(rc, "moe_permute")
    ops._after(dev)
    return out


def _unpermute(rows: torch.Tensor, sort: MoESort, weights: Optional[torch.Tensor]) -> torch.Tensor:
    rows = _rows(rows)
    n, H = rows.shape
    k, dev = sort.k, rows.device
    T = n // k
    out = rows.new_empty((T, H))
    with ops._on(dev):
        rc = _lib.load().moe_unpermute(rows.data_ptr(), _stride(rows), sort.row_of.data_ptr(), _live(sort), ops._ptr(weights), T, k, H,
                                       _DTYPES[rows.dtype], out.data_ptr(), ops._stream())
    _lib.check(rc, "moe_unpermute")
    ops._after(dev)
    return out


def _unpermute_grad(gy: torch.Tensor, rows: Optional[torch.Tensor], sort: MoESort, weights: torch.Tensor, want_rows: bool,
                    want_weights: bool):
    gy = _rows(gy)
    T, H = gy.shape
    k, dev = sort.k, gy.device
    g_rows = gy.new_empty((T * k, H)) if want_rows else None
    g_w = weights.new_empty((T, k)) if want_weights else None
    with ops._on(dev):
        rc = _lib.load().moe_unpermute_grad(gy.data_ptr(), _stride(gy), ops._ptr(rows), 0 if rows is None else _stride(rows),
                                            sort.row_of.data_ptr(), _live(sort), weights.data_ptr(), T, k, H, _DTYPES[gy.dtype],
                                            ops._ptr(g_rows), ops._ptr(g_w), ops._stream())
    _lib.check(rc, "moe_unpermute_grad")
    ops._after(dev)
    return g_rows, g_w


def _keep(ctx, sort: MoESort, *others) -> None:
    """Saves what the backward pass reads of the tables, under autograd's eyes: written again before it, they raise there.
    Tables of inference mode cannot be watched: of those the step keeps a copy."""
    tables = (t.clone() if t.is_inference() else t for t in (sort.offsets, sort.row_of))
    ctx.k = sort.k
    ctx.save_for_backward(*tables, *others)


def _kept(ctx):
    offsets, row_of, *others = ctx.saved_tensors
    return (MoESort._of(offsets, None, row_of, ctx.k), *others)


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, sort):
        _keep(ctx, sort)
        return _permute(x, sort)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        sort, = _kept(ctx)
        return _unpermute(g, sort, None), None


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, sort):
        rows = _rows(rows)
        # the rows are only kept where the weights' gradient needs them
        _keep(ctx, sort, rows if weights is not None and ctx.needs_input_grad[1] else None, weights)
        return _unpermute(rows, sort, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gy):
        sort, rows, weights = _kept(ctx)
        if weights is None:
            return _permute(gy, sort), None, None
        return (*_unpermute_grad(gy, rows, sort, weights, ctx.needs_input_grad[0], ctx.needs_input_grad[1]), None)


def _forward_mode() -> bool:
    """Inside a forward-mode level a tensor may carry a tangent.  There the calls go through autograd, which refuses those that do:
    past it the tangent would be lost without a word."""
    return forward_ad._current_level >= 0


def moe_permute(x: torch.Tensor, sort: MoESort) -> torch.Tensor:
    """Rows of x [T, H] at their entries' places: [T*k, H] of x's type.  Any element type; floating types of 16 and 32 bits
    have a gradient, others (8-bit values beside their scales, say) are copied."""
    ops._need_cuda(x)
    if x.dim() != 2 or x.shape[1] < 1 or x.shape[0] * sort.k != sort.row_of.numel():
        raise ValueError(f"x must be [{sort.tokens}, H], one row for each token of the sort")
    if x.device != sort.row_of.device:
        raise ValueError(f"x is on {x.device}, the sort's tables on {sort.row_of.device}")
    if x.is_conj():
        x = x.resolve_conj()
    backward = x.requires_grad and torch.is_grad_enabled()
    if backward and x.dtype not in _DTYPES:
        raise ValueError("the gradient of moe_permute is computed in bfloat16, float16 or float32")
    return _Permute.apply(x, sort) if backward or _forward_mode() else _permute(x, sort)


def moe_unpermute(rows: torch.Tensor, sort: MoESort, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[t] = sum over the entries of token t of weights[t, j] * its row: [T, H] of the rows' type (bfloat16, float16 or
    float32), summed in fp32 in slot order and rounded once.  weights: float32 [T, k]; 1 where not given."""
    ops._need_cuda(rows, weights)
    if rows.dtype not in _DTYPES:
        raise ValueError("rows must be bfloat16, float16 or float32")
    n, k, dev = sort.row_of.numel(), sort.k, sort.row_of.device
    if rows.dim() != 2 or rows.shape[1] < 1 or rows.shape[0] != n:
        raise ValueError(f"rows must be [{n}, H], one for each entry of the sort")
    if rows.device != dev or (weights is not None and weights.device != dev):
        raise ValueError(f"rows and weights must be on the device of the sort's tables, {dev}")
    if weights is not None:
        if weights.dtype != torch.float32 or weights.shape != (n // k, k):
            raise ValueError(f"routing weights must be float32 [{n // k}, {k}]")
        weights = ops._carried_out(weights).contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)) or _forward_mode():
        return _Unpermute.apply(rows, weights, sort)
    return _unpermute(rows, sort, weights)
