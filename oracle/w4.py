"""CPU oracle of the 4-bit products, in 64 bits (test infrastructure only)."""
from __future__ import annotations

import torch


def weights_ref(w: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None) -> torch.Tensor:
    """float64 [N, K]: (code - zero) * scale of packed w [N, K/2], scales and
    zeros [K/G, N] (None = 8)."""
    w, scales = w.cpu(), scales.cpu().double()
    N, K = w.shape[0], 2 * w.shape[1]
    codes = torch.zeros((N, K), dtype=torch.float64)
    codes[:, 0::2] = (w & 15).double()
    codes[:, 1::2] = (w >> 4).double()
    group = torch.arange(K) // (K // scales.shape[0])
    zero = torch.full_like(scales, 8.0) if zeros is None else zeros.cpu().double()
    return (codes - zero[group].t()) * scales[group].t()


def product_ref(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None):
    """(y, sum of magnitudes) float64 [M, N]."""
    v, x = weights_ref(w, scales, zeros), x.cpu().double()
    return x @ v.t(), x.abs() @ v.abs().t()


def experts_ref(x, w, scales, zeros, offsets, rows: int):
    """(y, sum of magnitudes) float64 [rows, N] of sorted rows x [rows, K]."""
    y = torch.zeros((rows, w.shape[1]), dtype=torch.float64)
    mag = torch.zeros_like(y)
    bounds = offsets.tolist()
    for e in range(w.shape[0]):
        a, b = bounds[e], bounds[e + 1]
        if b > a:
            y[a:b], mag[a:b] = product_ref(x[a:b], w[e], scales[e], None if zeros is None else zeros[e])
    return y, mag
