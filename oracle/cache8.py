"""The 8-bit rows of the rolling cache, and attention with its error bounds, in 64 bits.

A row x of D values is D e4m3 codes and one integer exponent e: the smallest
e >= -117 with max |x| <= 448 * 2^e over the finite values; a code is the e4m3 number
nearest to x * 2^-e, ties to even; infinities and NaN become NaN.
"""

from __future__ import annotations

import numpy as np
import torch

MIN_EXPONENT = -117


def e4m3_round(y: np.ndarray) -> np.ndarray:
    """The e4m3 number nearest to each |y| <= 448 (ties to even): multiples of
    2^(k - 3) for |y| in [2^k, 2^(k + 1)), of 2^-9 below 2^-6."""
    y = np.asarray(y, dtype=np.float64)
    _, e = np.frexp(np.abs(y))                       # |y| = m 2^e, m in [1/2, 1)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.round(y / step) * step                  # numpy rounds ties to even


def quantise(x: np.ndarray):
    """(codes as values, exponents) of the rows of x (last axis)."""
    x = np.asarray(x, dtype=np.float64)
    fine = np.isfinite(x)
    top = np.where(fine, np.abs(x), 0.0).max(-1)
    m, e = np.frexp(top)                              # 448 = 0.875 * 2^9
    e = np.where(top == 0, MIN_EXPONENT, np.maximum(np.where(m <= 0.875, e - 9, e - 8), MIN_EXPONENT))
    y = np.where(fine, x, 0.0) * np.ldexp(1.0, -e)[..., None]
    return np.where(fine, e4m3_round(y), np.nan), e


def stored_values(x: np.ndarray) -> np.ndarray:
    codes, e = quantise(x)
    return codes * np.ldexp(1.0, e)[..., None]


def held_positions(length: int, sink: int, ring: int) -> list:
    """Positions a rolling cache holds, ascending."""
    return [p for p in range(length) if p < sink or p >= length - ring]


def attention64(q, k, v, visible, scale):
    """O, LSE (0 where nothing is visible) and, for error bounds, P|V| and
    sum |q k| |scale| (its largest over a row's visible keys), all float64.

    q [B, H, n, D], k / v [B, H_kv, m, D]; visible broadcasts to [B, H, n, m]."""
    q, k, v = (t.double() for t in (q, k, v))
    group = q.shape[1] // k.shape[1]
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    visible = torch.as_tensor(visible, device=q.device)
    s = (q @ k.transpose(2, 3)) * scale
    visible = visible.expand(s.shape)
    s = s.masked_fill(~visible, float("-inf"))
    m = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full(s.shape[:-1] + (1,), float("-inf"))
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    empty = l == 0
    p = p / torch.where(empty, torch.ones_like(l), l)
    lse = torch.where(empty, torch.zeros_like(l), m + torch.log(torch.where(empty, torch.ones_like(l), l)))
    size = (q.abs() @ k.abs().transpose(2, 3)).masked_fill(~visible, 0.0)
    size = size.amax(-1) * abs(scale) if s.shape[-1] else torch.zeros_like(lse[..., 0])
    return p @ v, lse[..., 0], p @ v.abs(), size


def output_bound(o, pv, size, n_keys: int, dtype: torch.dtype, p_eps: float):
    """Largest |error| of an output: its own rounding (half a unit of ``dtype``), the
    rounding of the weights (``p_eps`` relative each, and once more where the row sum is
    taken over unrounded ones), and fp32 scores, exponents and sums: a score is off by at
    most (D + 8) 2^-24 of sum |q k| (D <= 128), which moves a weight by as much, and
    n_keys additions by 2^-24 each, over P|V| = ``pv``."""
    half = torch.finfo(dtype).eps / 2
    f32 = 2 * (136 * 2.0**-24) * size[..., None] + (n_keys + 16) * 2.0**-24
    return half * o.abs() + (p_eps + f32) * (1 + half) * pv * 1.01 + 1e-30 + torch.finfo(dtype).tiny * half * 2
