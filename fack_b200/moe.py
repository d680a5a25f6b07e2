"""Tokens sorted by expert and back (``fack_moe_*``).

The data movement around the expert products of a routed layer: a stable sort
of the (token, slot) pairs by expert, the tokens' rows in that order -- as they
are, or as the FP8 GEMM's codes and scales -- and the weighted sum back to
tokens, with gradients.  A layer's use::

    plan = moe_sort(topk_ids, num_experts)               # ids [T, k] of torch.topk
    xq, xs = moe_gather_quant(x, plan)                   # sorted FP8 rows; expert e owns offsets[e] .. offsets[e+1]
    ... gemm_blockscale(xq[a:b], w[e], xs[a:b], ws[e], out=y[a:b]) per expert, or gemv_w4_experts(x, ...) ...
    out = moe_combine(y, topk_weights, plan)             # [T, D]

Sorted buffers always hold T*k rows, so nothing here depends on a value on the
host: every call can be captured in a CUDA graph and nothing synchronises.
Ids outside ``[0, num_experts)`` have no row: an expert-parallel rank passes
``ids - first_expert`` and the pairs of the other ranks' experts drop out.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import BLOCK, FP8, _stream_handle

MAX_EXPERTS = 1024
MAX_TOPK = 64

DTYPES = {torch.float32: _lib.FACK_DTYPE_F32, torch.bfloat16: _lib.FACK_DTYPE_BF16,
          torch.float16: _lib.FACK_DTYPE_F16}


class MoePlan(NamedTuple):
    """What :func:`moe_sort` computes; T tokens, k slots, E experts.

    ``row_of`` int32 [T, k]: the sorted row of each (token, slot) pair, -1
    where the pair has none.  ``src`` int32 [T*k]: the pair t*k + j of each
    sorted row, -1 behind the last.  ``offsets`` int32 [E + 1]: each expert's
    first row; ``offsets[E]`` rows have a pair.
    """
    row_of: torch.Tensor
    src: torch.Tensor
    offsets: torch.Tensor


class _on:
    """The device made current for a call, unless it is already."""
    __slots__ = ("index", "guard")

    def __init__(self, dev):
        self.index = dev.index
        self.guard = None

    def __enter__(self):
        if torch.cuda.current_device() != self.index:
            self.guard = torch.cuda.device(self.index)
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _check_plan(plan, dev: torch.device):
    """(T, k, E) of a plan on ``dev``."""
    row_of, src, offsets = plan
    for name, t, dim in (("row_of", row_of, 2), ("src", src, 1), ("offsets", offsets, 1)):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dim or t.device != dev \
                or not t.is_contiguous():
            raise ValueError(f"plan.{name} must be a contiguous {dim}-D int32 tensor on {dev}")
    T, topk = row_of.shape
    E = offsets.shape[0] - 1
    if src.shape[0] != T * topk or not 1 <= topk <= MAX_TOPK or not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"plan shapes do not belong together: row_of {tuple(row_of.shape)}, "
                         f"src {tuple(src.shape)}, offsets {tuple(offsets.shape)}")
    return T, topk, E


def _check_rows(t, name: str, rows: Optional[int] = None, width: Optional[int] = None, dtypes=DTYPES):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 2:
        raise ValueError(f"{name} must be a 2-D CUDA tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {', '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if (rows is not None and t.shape[0] != rows) or (width is not None and t.shape[1] != width) or t.shape[1] < 1:
        raise ValueError(f"{name} must be [{'rows' if rows is None else rows}, {'D' if width is None else width}], "
                         f"got {tuple(t.shape)}")
    if t.shape[1] > 1 and t.stride(1) != 1 and t.shape[0]:
        raise ValueError(f"{name} must be contiguous along its rows")


def _ld(t: torch.Tensor) -> int:
    """Row stride of a checked 2-D tensor (that of a lone row says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_weights(weights, T, topk, dev):
    if not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32 or tuple(weights.shape) != (T, topk) \
            or weights.device != dev:
        raise ValueError(f"weights must be a float32 [{T}, {topk}] tensor on {dev}")
    return weights.contiguous()


def moe_sort(topk_ids: torch.Tensor, num_experts: int) -> MoePlan:
    """Sort the (token, slot) pairs of ``topk_ids`` [T, k] (int32 or int64) by
    expert, pairs of one expert in the order t*k + j; see :class:`MoePlan`."""
    if not isinstance(topk_ids, torch.Tensor) or not topk_ids.is_cuda or topk_ids.dim() != 2 \
            or topk_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("topk_ids must be a 2-D int32 or int64 CUDA tensor")
    T, topk = topk_ids.shape
    E = int(num_experts)
    if not 1 <= topk <= MAX_TOPK or not 1 <= E <= MAX_EXPERTS or T * topk >= 1 << 31:
        raise ValueError(f"moe_sort takes 1 to {MAX_TOPK} slots, 1 to {MAX_EXPERTS} experts and fewer than 2^31 pairs")
    dev = topk_ids.device
    ids = topk_ids.contiguous()
    row_of = torch.empty((T, topk), dtype=torch.int32, device=dev)
    src = torch.empty((T * topk,), dtype=torch.int32, device=dev)
    if T == 0:
        return MoePlan(row_of, src, torch.zeros((E + 1,), dtype=torch.int32, device=dev))
    offsets = torch.empty((E + 1,), dtype=torch.int32, device=dev)
    lib = _lib.load()
    nb = ctypes.c_size_t()
    _lib.check(lib.fack_moe_sort_workspace_size(T, topk, E, ctypes.byref(nb)), "fack_moe_sort_workspace_size")
    # of this call alone: two captured sorts, or two streams, never share one
    ws = torch.empty((nb.value,), dtype=torch.uint8, device=dev) if nb.value else None
    with _on(dev):
        st = lib.fack_moe_sort(ids.data_ptr(), ids.element_size(), T, topk, E, row_of.data_ptr(), src.data_ptr(),
                               offsets.data_ptr(), None if ws is None else ws.data_ptr(), nb.value,
                               _stream_handle(dev))
    _lib.check(st, "fack_moe_sort")
    return MoePlan(row_of, src, offsets)


def _gather(x, plan):
    _check_rows(x, "x")
    dev = x.device
    T, topk, E = _check_plan(plan, dev)
    D = x.shape[1]
    if x.shape[0] != T:
        raise ValueError(f"x has {x.shape[0]} rows, the plan {T} tokens")
    y = torch.empty((T * topk, D), dtype=x.dtype, device=dev)
    if T:
        with _on(dev):
            st = _lib.load().fack_moe_gather(x.data_ptr(), DTYPES[x.dtype], _ld(x), T, topk, D,
                                             plan.row_of.data_ptr(), plan.offsets.data_ptr(), E, y.data_ptr(), D,
                                             _stream_handle(dev))
        _lib.check(st, "fack_moe_gather")
    return y


def _combine(y, weights, plan):
    _check_rows(y, "y")
    dev = y.device
    T, topk, _ = _check_plan(plan, dev)
    D = y.shape[1]
    if y.shape[0] != T * topk:
        raise ValueError(f"y has {y.shape[0]} rows, the plan {T * topk}")
    w = None if weights is None else _check_weights(weights, T, topk, dev)
    out = torch.empty((T, D), dtype=y.dtype, device=dev)
    if T:
        with _on(dev):
            st = _lib.load().fack_moe_combine(y.data_ptr(), DTYPES[y.dtype], _ld(y), None if w is None else w.data_ptr(),
                                              T, topk, D, plan.row_of.data_ptr(), out.data_ptr(), D,
                                              _stream_handle(dev))
        _lib.check(st, "fack_moe_combine")
    return out


def moe_gather_backward(dy: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """dx [T, D] of :func:`moe_gather` from dy [T*k, D]: each token's rows
    summed in fp32, slots in order, rounded once."""
    return _combine(dy, None, plan)


def moe_combine_backward(dout: torch.Tensor, y: Optional[torch.Tensor], weights: torch.Tensor, plan: MoePlan,
                         need_dy: bool = True, need_dweights: bool = True):
    """(dy [T*k, D], dweights fp32 [T, k]) of :func:`moe_combine` from dout
    [T, D]; None in the place of one that is not needed (``y`` may be None
    without ``need_dweights``).  Rows of dy without a pair are zero."""
    _check_rows(dout, "dout")
    dev = dout.device
    T, topk, E = _check_plan(plan, dev)
    D = dout.shape[1]
    if dout.shape[0] != T:
        raise ValueError(f"dout has {dout.shape[0]} rows, the plan {T} tokens")
    w = _check_weights(weights, T, topk, dev)
    if need_dweights:
        _check_rows(y, "y", T * topk, D)
        if y.dtype != dout.dtype or y.device != dev:
            raise ValueError("y and dout must have one type and device")
    dy = torch.empty((T * topk, D), dtype=dout.dtype, device=dev) if need_dy else None
    dw = torch.empty((T, topk), dtype=torch.float32, device=dev) if need_dweights else None
    if T and (need_dy or need_dweights):
        with _on(dev):
            st = _lib.load().fack_moe_combine_bwd(
                dout.data_ptr(), DTYPES[dout.dtype], _ld(dout), y.data_ptr() if need_dweights else None,
                _ld(y) if need_dweights else 0, w.data_ptr(), T, topk, D, plan.row_of.data_ptr(),
                plan.offsets.data_ptr(), E, dy.data_ptr() if need_dy else None, D,
                dw.data_ptr() if need_dweights else None, _stream_handle(dev))
        _lib.check(st, "fack_moe_combine_bwd")
    return dy, dw


def _grad_rows(g: torch.Tensor) -> torch.Tensor:
    """An incoming gradient as rows the kernels read: autograd also hands out
    transposed and, from sums, broadcast ones."""
    return g if g.shape[1] == 1 or g.stride(1) == 1 else g.contiguous()


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, row_of, src, offsets):
        plan = MoePlan(row_of, src, offsets)
        ctx.save_for_backward(*plan)
        return _gather(x, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return moe_gather_backward(_grad_rows(dy), MoePlan(*ctx.saved_tensors)), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, row_of, src, offsets):
        plan = MoePlan(row_of, src, offsets)
        need_dw = ctx.needs_input_grad[1]
        ctx.save_for_backward(y if need_dw else None, weights, *plan)
        return _combine(y, weights, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, weights, *plan = ctx.saved_tensors
        dy, dw = moe_combine_backward(_grad_rows(dout), y, weights, MoePlan(*plan), ctx.needs_input_grad[0],
                                      ctx.needs_input_grad[1])
        return dy, dw, None, None, None


def moe_gather(x: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """The tokens' rows in expert order: y [T*k, D] with y[r] = x[src[r] // k],
    zeros where a row has no pair.  ``x`` [T, D] fp32, bf16 or fp16, any row
    stride.  Differentiable in x (:func:`moe_gather_backward`)."""
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        return _Gather.apply(x, *plan)
    return _gather(x, plan)


def moe_combine(y: torch.Tensor, weights: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """The experts' rows back to tokens: out[t] = sum_j weights[t, j] *
    y[row_of[t, j]] over the pairs that have a row, in fp32, slots in order,
    rounded once to y's type.  ``y`` [T*k, D] fp32, bf16 or fp16, any row
    stride; ``weights`` fp32 [T, k].  Differentiable in both
    (:func:`moe_combine_backward`)."""
    if weights is None:
        raise ValueError("weights must be a float32 [T, k] tensor")
    if torch.is_grad_enabled() and (getattr(y, "requires_grad", False) or getattr(weights, "requires_grad", False)):
        return _Combine.apply(y, weights, *plan)
    return _combine(y, weights, plan)


def moe_gather_quant(x: torch.Tensor, plan: MoePlan):
    """:func:`moe_gather` and :func:`fack_b200.quantize_activations` in one
    pass: (xq e4m3 [T*k, K], x_scale fp32 [T*k, K/128]), the sorted rows' codes
    and logical scales as :func:`fack_b200.gemm_blockscale` takes them per
    expert.  ``x`` [T, K] fp32 or bf16, K % 128 == 0, rows 16-byte aligned.
    Rows without a pair have zero codes and scale 1; a 128-wide group that
    holds NaN has scale and codes NaN.  Not differentiable."""
    _check_rows(x, "x", dtypes=(torch.float32, torch.bfloat16))
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("moe_gather_quant has no gradient; detach x or call it under torch.no_grad()")
    dev = x.device
    T, topk, E = _check_plan(plan, dev)
    K = x.shape[1]
    if x.shape[0] != T:
        raise ValueError(f"x has {x.shape[0]} rows, the plan {T} tokens")
    if K % BLOCK:
        raise ValueError("K must be a multiple of 128")
    xq = torch.empty((T * topk, K), dtype=FP8, device=dev)
    xs = torch.empty((T * topk, K // BLOCK), dtype=torch.float32, device=dev)
    if T:
        with _on(dev):
            st = _lib.load().fack_moe_gather_quant(x.data_ptr(), DTYPES[x.dtype], _ld(x), T, topk, K,
                                                   plan.row_of.data_ptr(), plan.offsets.data_ptr(), E, xq.data_ptr(),
                                                   K, xs.data_ptr(), K // BLOCK, _stream_handle(dev))
        _lib.check(st, "fack_moe_gather_quant")
    return xq, xs
