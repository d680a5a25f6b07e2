"""CPU oracle of the expert-sorted data movement and the 4-bit products, in 64 bits.

Test infrastructure only, as ``oracle/blockscale.py``: plain restatements of
the definitions, token by token.
"""
from __future__ import annotations

import torch

BLOCK = 128
QMAX = 240.0


def sort_ref(ids: torch.Tensor, num_experts: int):
    """(row_of [T, k], src [T*k], offsets [E + 1]) as int32, pair by pair."""
    flat = [int(i) for i in ids.reshape(-1).cpu()]
    by_expert = [[] for _ in range(num_experts)]
    for p, e in enumerate(flat):
        if 0 <= e < num_experts:
            by_expert[e].append(p)
    row_of, src, offsets = [-1] * len(flat), [], [0]
    for pairs in by_expert:
        for p in pairs:
            row_of[p] = len(src)
            src.append(p)
        offsets.append(len(src))
    src += [-1] * (len(flat) - len(src))
    as_int = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return as_int(row_of).reshape(ids.shape), as_int(src), as_int(offsets)


def gather_ref(x: torch.Tensor, src: torch.Tensor, topk: int) -> torch.Tensor:
    """Sorted rows of x, zero without a pair; x's own type (a copy)."""
    x, src = x.cpu(), src.cpu().long()
    y = torch.zeros((src.numel(), x.shape[1]), dtype=x.dtype)
    for r, p in enumerate(src.tolist()):
        if p >= 0:
            y[r] = x[p // topk]
    return y


def combine_ref(y: torch.Tensor, weights: torch.Tensor | None, row_of: torch.Tensor):
    """(out, sum of magnitudes) [T, D] in 64 bits; weights None = ones."""
    y, row_of = y.cpu().double(), row_of.cpu()
    T, topk = row_of.shape
    w = torch.ones((T, topk), dtype=torch.float64) if weights is None else weights.cpu().double()
    out, mag = torch.zeros((T, y.shape[1]), dtype=torch.float64), torch.zeros((T, y.shape[1]), dtype=torch.float64)
    for t in range(T):
        for j in range(topk):
            r = int(row_of[t, j])
            if r >= 0:
                out[t] += w[t, j] * y[r]
                mag[t] += (w[t, j] * y[r]).abs()
    return out, mag


def combine_bwd_ref(dout: torch.Tensor, y: torch.Tensor, weights: torch.Tensor, row_of: torch.Tensor):
    """(dy [T*k, D], dw [T, k], sum of magnitudes of dw) in 64 bits."""
    dout, y, w, row_of = dout.cpu().double(), y.cpu().double(), weights.cpu().double(), row_of.cpu()
    T, topk = row_of.shape
    dy, dw = torch.zeros((T * topk, dout.shape[1]), dtype=torch.float64), torch.zeros((T, topk), dtype=torch.float64)
    mag = torch.zeros_like(dw)
    for t in range(T):
        for j in range(topk):
            r = int(row_of[t, j])
            if r >= 0:
                dy[r] = w[t, j] * dout[t]
                dw[t, j] = (dout[t] * y[r]).sum()
                mag[t, j] = (dout[t] * y[r]).abs().sum()
    return dy, dw, mag


def gather_quant_ref(x: torch.Tensor, src: torch.Tensor, topk: int):
    """(codes e4m3 [T*k, K], scales fp32 [T*k, K/128]): each token quantised in
    fp32 as the FP8 GEMM's inputs are (scale = amax/240, 1 where that is 0),
    its rows put in sorted order; 0 and 1 without a pair."""
    x, src = x.cpu().float(), src.cpu().long()
    T, K = x.shape
    g = x.reshape(T, K // BLOCK, BLOCK)
    scale = g.abs().amax(dim=2) / QMAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = (g / scale.unsqueeze(2)).clamp(-QMAX, QMAX).reshape(T, K)
    xq, xs = torch.zeros((src.numel(), K)), torch.ones((src.numel(), K // BLOCK))
    for r, p in enumerate(src.tolist()):
        if p >= 0:
            xq[r], xs[r] = q[p // topk], scale[p // topk]
    return xq.to(torch.float8_e4m3fn), xs
