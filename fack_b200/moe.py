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
from torch.autograd import forward_ad

from . import _lib
from .ops import BLOCK, FP8

MAX_EXPERTS = 1024
MAX_TOPK = 64
SORT_ONE_BLOCK = 512     # pairs that one block always sorts, without a workspace

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


def _call(name: str, dev: torch.device, *args) -> None:
    """One C entry on ``dev``'s current stream, with ``dev`` current meanwhile.

    A decode step makes these calls for microseconds of GPU work each, so the
    host's share is kept small: the stream's handle is read without making a
    stream object, and the device is switched only when it has to be."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == dev.index:
        st = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if st:
        _lib.check(st, name)


def _check_plan(plan, dev: torch.device):
    """(T, k, E) of a plan on ``dev``."""
    if not isinstance(plan, MoePlan):
        raise ValueError("plan must be the MoePlan of moe_sort")
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


def _refuse_tangent(t: torch.Tensor, name: str) -> None:
    """No forward-mode derivative: a dual tensor does not require grad, and its
    tangent would be lost without a word."""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a forward-mode tangent, which this operator does not take; "
                         "use its primal (torch.autograd.forward_ad.unpack_dual)")


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
    _refuse_tangent(t, name)


def _ld(t: torch.Tensor) -> int:
    """Row stride of a checked 2-D tensor (that of a lone row says nothing)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check_weights(weights, T, topk, dev):
    if not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32 or tuple(weights.shape) != (T, topk) \
            or weights.device != dev:
        raise ValueError(f"weights must be a float32 [{T}, {topk}] tensor on {dev}")
    _refuse_tangent(weights, "weights")
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
    row_of = ids.new_empty((T, topk), dtype=torch.int32)
    src = ids.new_empty((T * topk,), dtype=torch.int32)
    if T == 0:
        return MoePlan(row_of, src, ids.new_zeros((E + 1,), dtype=torch.int32))
    offsets = ids.new_empty((E + 1,), dtype=torch.int32)
    ws, nb = None, 0
    if T * topk > SORT_ONE_BLOCK:
        size = ctypes.c_size_t()
        _lib.check(_lib.load().fack_moe_sort_workspace_size(T, topk, E, ctypes.byref(size)),
                   "fack_moe_sort_workspace_size")
        nb = size.value
        # of this call alone: two captured sorts, or two streams, never share one
        ws = ids.new_empty((nb,), dtype=torch.uint8) if nb else None
    _call("fack_moe_sort", dev, ids.data_ptr(), ids.element_size(), T, topk, E, row_of.data_ptr(), src.data_ptr(),
          offsets.data_ptr(), None if ws is None else ws.data_ptr(), nb)
    return MoePlan(row_of, src, offsets)


def _gather(x, plan):
    _check_rows(x, "x")
    T, topk, E = _check_plan(plan, x.device)
    if x.shape[0] != T:
        raise ValueError(f"x has {x.shape[0]} rows, the plan {T} tokens")
    D = x.shape[1]
    y = x.new_empty((T * topk, D))
    if T:
        _call("fack_moe_gather", x.device, x.data_ptr(), DTYPES[x.dtype], _ld(x), T, topk, D, plan.row_of.data_ptr(),
              plan.offsets.data_ptr(), E, y.data_ptr(), D)
    return y


def _sum_rows(y, w, row_of):
    """The combine kernel on checked operands (w None: ones)."""
    T, topk = row_of.shape
    D = y.shape[1]
    out = y.new_empty((T, D))
    if T:
        _call("fack_moe_combine", y.device, y.data_ptr(), DTYPES[y.dtype], _ld(y), None if w is None else w.data_ptr(),
              T, topk, D, row_of.data_ptr(), out.data_ptr(), D)
    return out


def _check_sorted(y, plan):
    _check_rows(y, "y")
    T, topk, _ = _check_plan(plan, y.device)
    if y.shape[0] != T * topk:
        raise ValueError(f"y has {y.shape[0]} rows, the plan {T * topk}")
    return T, topk


def _combine(y, weights, plan):
    T, topk = _check_sorted(y, plan)
    return _sum_rows(y, _check_weights(weights, T, topk, y.device), plan.row_of)


def moe_gather_backward(dy: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """dx [T, D] of :func:`moe_gather` from dy [T*k, D]: each token's rows
    summed in fp32, slots in order, rounded once.  Not recorded by autograd."""
    _check_sorted(dy, plan)
    return _sum_rows(dy, None, plan.row_of)


def _combine_grads(dout, y, w, row_of, offsets, need_dy, need_dw):
    """The gradient kernel on checked operands (y is read for dw alone)."""
    T, topk = row_of.shape
    D = dout.shape[1]
    dy = dout.new_empty((T * topk, D)) if need_dy else None
    dw = dout.new_empty((T, topk), dtype=torch.float32) if need_dw else None
    if T and (need_dy or need_dw):
        _call("fack_moe_combine_bwd", dout.device, dout.data_ptr(), DTYPES[dout.dtype], _ld(dout),
              y.data_ptr() if need_dw else None, _ld(y) if need_dw else 0, w.data_ptr(), T, topk, D,
              row_of.data_ptr(), offsets.data_ptr(), offsets.shape[0] - 1, dy.data_ptr() if need_dy else None, D,
              dw.data_ptr() if need_dw else None)
    return dy, dw


def moe_combine_backward(dout: torch.Tensor, y: Optional[torch.Tensor], weights: torch.Tensor, plan: MoePlan,
                         need_dy: bool = True, need_dweights: bool = True):
    """(dy [T*k, D], dweights fp32 [T, k]) of :func:`moe_combine` from dout
    [T, D]; None in the place of one that is not needed (``y`` may be None
    without ``need_dweights``).  Rows of dy without a pair are zero.  Not recorded
    by autograd."""
    _check_rows(dout, "dout")
    dev = dout.device
    T, topk, _ = _check_plan(plan, dev)
    if dout.shape[0] != T:
        raise ValueError(f"dout has {dout.shape[0]} rows, the plan {T} tokens")
    w = _check_weights(weights, T, topk, dev)
    if need_dweights:
        _check_rows(y, "y", T * topk, dout.shape[1])
        if y.dtype != dout.dtype or y.device != dev:
            raise ValueError("y and dout must have one type and device")
    return _combine_grads(dout, y, w, plan.row_of, plan.offsets, need_dy, need_dweights)


def _grad_rows(g: torch.Tensor) -> torch.Tensor:
    """An incoming gradient as rows the kernels read: autograd also hands out
    transposed and, from sums, broadcast ones."""
    return g if g.shape[1] == 1 or g.stride(1) == 1 else g.contiguous()


def _refuse_captured_leaf(*inputs) -> None:
    """No gradient of a leaf inside a CUDA-graph capture: where an eager graph of
    the same leaf is alive, autograd would make the capture wait on that graph's
    stream, which ends the process.  The backward functions have no such state.
    Whether such a graph lives cannot be asked; where none does (the static inputs of
    torch.cuda.make_graphed_callables), a view of the leaf is taken."""
    for t in inputs:
        if t.requires_grad and t.is_leaf and t.is_cuda and torch.cuda.is_current_stream_capturing():
            raise ValueError("a captured gather or combine takes no leaf that requires grad; call "
                             "moe_gather_backward / moe_combine_backward in the capture instead, or detach the input")


# The plan goes through apply whole: as three tensors it costs a round trip 3-5 us more.
class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        y = _gather(x, plan)
        ctx.save_for_backward(plan.row_of)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return _sum_rows(_grad_rows(dy), None, ctx.saved_tensors[0]), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, plan):
        T, topk = _check_sorted(y, plan)
        w = _check_weights(weights, T, topk, y.device)
        ctx.save_for_backward(y if ctx.needs_input_grad[1] else None, w, plan.row_of, plan.offsets)
        return _sum_rows(y, w, plan.row_of)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, w, row_of, offsets = ctx.saved_tensors
        dy, dw = _combine_grads(_grad_rows(dout), y, w, row_of, offsets, *ctx.needs_input_grad[:2])
        return dy, dw, None


def moe_gather(x: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """The tokens' rows in expert order: y [T*k, D] with y[r] = x[src[r] // k],
    zeros where a row has no pair.  ``x`` [T, D] fp32, bf16 or fp16, any row
    stride.  Differentiable in x in reverse mode (:func:`moe_gather_backward`;
    a forward-mode tangent is refused); inside a CUDA-graph capture x may not be
    a leaf that requires grad."""
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled() and isinstance(plan, MoePlan):
        _refuse_captured_leaf(x)
        _refuse_tangent(x, "x")
        return _Gather.apply(x, plan)
    return _gather(x, plan)


def moe_combine(y: torch.Tensor, weights: torch.Tensor, plan: MoePlan) -> torch.Tensor:
    """The experts' rows back to tokens: out[t] = sum_j weights[t, j] *
    y[row_of[t, j]] over the pairs that have a row, in fp32, slots in order,
    rounded once to y's type.  ``y`` [T*k, D] fp32, bf16 or fp16, any row
    stride; ``weights`` fp32 [T, k].  Differentiable in both
    in reverse mode (:func:`moe_combine_backward`; a forward-mode tangent is
    refused); inside a CUDA-graph capture neither may be a leaf that requires grad."""
    if weights is None:
        raise ValueError("weights must be a float32 [T, k] tensor")
    if torch.is_grad_enabled() and isinstance(plan, MoePlan) and (getattr(y, "requires_grad", False)
                                                                  or getattr(weights, "requires_grad", False)):
        if isinstance(y, torch.Tensor) and isinstance(weights, torch.Tensor):
            _refuse_captured_leaf(y, weights)
            _refuse_tangent(y, "y")
            _refuse_tangent(weights, "weights")
        return _Combine.apply(y, weights, plan)
    return _combine(y, weights, plan)


def moe_gather_quant(x: torch.Tensor, plan: MoePlan):
    """:func:`moe_gather` and :func:`fack_b200.quantize_activations` in one
    pass: (xq e4m3 [T*k, K], x_scale fp32 [T*k, K/128]), the sorted rows' codes
    and logical scales as :func:`fack_b200.gemm_blockscale` takes them per
    expert.  ``x`` [T, K] fp32 or bf16, K % 128 == 0, rows 16-byte aligned.
    Rows without a pair have zero codes and scale 1.  NaN in a 128-wide group makes
    its scale and codes NaN; an infinity makes its scale infinite, the infinities
    NaN codes and the rest zero codes; an amax that is too small for a scale makes
    it 1 and the codes zero (quantize_activations: NaN left out of the amax, -240
    for NaN quotients, scale 0).  Not differentiable."""
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
    xq = x.new_empty((T * topk, K), dtype=FP8)
    xs = x.new_empty((T * topk, K // BLOCK), dtype=torch.float32)
    if T:
        _call("fack_moe_gather_quant", dev, x.data_ptr(), DTYPES[x.dtype], _ld(x), T, topk, K, plan.row_of.data_ptr(),
              plan.offsets.data_ptr(), E, xq.data_ptr(), K, xs.data_ptr(), K // BLOCK)
    return xq, xs
