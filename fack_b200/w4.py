"""Products of a few tokens with 4-bit weights (``fack_gemv_w4*``).

    y[m, n] = sum_k x[m, k] * (code[n, k] - zero[k // G, n]) * scale[k // G, n]

``w`` uint8 [N, K/2] holds two 4-bit codes a byte along K, the even k in the
low nibble; ``scales`` [K/G, N] (fp32 or x's type) and ``zeros`` uint8 [K/G, N]
(values 0..15; None = 8 everywhere) one value per output row and group of
G = 32, 64 or a multiple of 128 consecutive k.  The weights are read once and in
place -- no dequantised copy, no workspace -- which is what a decode step's
projections cost.  Products are exact, sums fp32, one rounding at the end.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from .moe import DTYPES, MoePlan, _call, _check_plan, _check_rows, _ld, _refuse_tangent

TYPES = (torch.bfloat16, torch.float16)


def _part(name: str, t, types: tuple, lead: tuple, dev) -> None:
    dims = len(lead) + 2
    if not isinstance(t, torch.Tensor) or t.device != dev or t.dtype not in types or t.dim() != dims \
            or (lead and t.shape[0] != lead[0]) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dims}-D tensor of {' or '.join(str(d) for d in types)} on {dev}"
                         + (f" with {lead[0]} experts" if lead else ""))


def _check_weight(x, w, scales, zeros, lead: tuple):
    """(N, K, G) of a 4-bit weight with leading dimensions ``lead`` for x [*, K]."""
    K, dev = x.shape[1], x.device
    _part("w", w, (torch.uint8,), lead, dev)
    _part("scales", scales, (torch.float32, x.dtype), lead, dev)
    if zeros is not None:
        _part("zeros", zeros, (torch.uint8,), lead, dev)
    N, half = w.shape[-2:]
    groups, width = scales.shape[-2:]
    if half * 2 != K or width != N or groups < 1 or K % groups or (zeros is not None and zeros.shape != scales.shape):
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, w {tuple(w.shape)}, scales {tuple(scales.shape)}, "
                         f"zeros {None if zeros is None else tuple(zeros.shape)}")
    G = K // groups
    if N < 16 or N % 16 or (G != 32 and G != 64 and G % 128):
        raise ValueError(f"4-bit products need N % 16 == 0 and groups of 32, 64 or a multiple of 128 along K "
                         f"(N = {N}, group = {G})")
    if (x.requires_grad or scales.requires_grad) and torch.is_grad_enabled():
        raise ValueError("4-bit products have no gradient; detach the operands or call under torch.no_grad()")
    _refuse_tangent(scales, "scales")
    return N, K, G


def _check_out(out, rows: int, N: int, x):
    if out is None:
        return x.new_empty((rows, N))
    if not isinstance(out, torch.Tensor) or out.dtype != x.dtype or tuple(out.shape) != (rows, N) or out.stride(1) != 1 \
            or out.device != x.device or (rows > 1 and out.stride(0) < N):
        raise ValueError(f"out must be a {x.dtype} [{rows}, {N}] tensor with unit column stride on {x.device}")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out is written outside autograd: it must not require grad")
    _refuse_tangent(out, "out")
    return out


def gemv_w4(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [M, N] = x [M, K] (bf16 or fp16, rows 16-byte aligned) times the 4-bit
    weight ``w`` [N, K/2] transposed.  Any M is right; the kernel is made for
    the M up to about 32 of a decode step (more tokens are taken 8 or 16 at a
    time).  Writes and returns ``out`` when given (it may not overlap an operand)."""
    _check_rows(x, "x", dtypes=TYPES)
    N, K, G = _check_weight(x, w, scales, zeros, ())
    M = x.shape[0]
    out = _check_out(out, M, N, x)
    if M:
        _call("fack_gemv_w4", x.device, x.data_ptr(), DTYPES[x.dtype], _ld(x), w.data_ptr(), scales.data_ptr(),
              DTYPES[scales.dtype], None if zeros is None else zeros.data_ptr(), G, out.data_ptr(), _ld(out), M, N, K)
    return out


def gemv_w4_experts(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, plan: MoePlan,
                    zeros: Optional[torch.Tensor] = None, sorted_rows: bool = False,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Each sorted row's product with its expert's 4-bit weight: y [T*k, N] for
    a :func:`fack_b200.moe_sort` plan, ``w`` [E, N, K/2], ``scales`` and ``zeros``
    [E, K/G, N].  ``x`` is the tokens [T, K], gathered on the way in, or with
    ``sorted_rows`` the rows [T*k, K] in sorted order (an earlier product's
    output).  Rows without a pair are written as zeros.  Only the experts that
    have rows are read; the row counts stay on the device.  Writes and returns
    ``out`` when given (it may not overlap an operand)."""
    _check_rows(x, "x", dtypes=TYPES)
    T, topk, E = _check_plan(plan, x.device)
    N, K, G = _check_weight(x, w, scales, zeros, (E,))
    if x.shape[0] != (T * topk if sorted_rows else T):
        raise ValueError(f"x has {x.shape[0]} rows, the plan {T} tokens of {topk} slots "
                         f"(sorted_rows={bool(sorted_rows)})")
    out = _check_out(out, T * topk, N, x)
    if T:
        _call("fack_gemv_w4_experts", x.device, x.data_ptr(), DTYPES[x.dtype], _ld(x), w.data_ptr(), scales.data_ptr(),
              DTYPES[scales.dtype], None if zeros is None else zeros.data_ptr(), G,
              None if sorted_rows else plan.src.data_ptr(), plan.offsets.data_ptr(), T, topk, E, out.data_ptr(),
              _ld(out), N, K)
    return out
