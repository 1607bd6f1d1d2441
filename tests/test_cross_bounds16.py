"""Cross attention in 16 bits against 64 bits, within bounds that a dropped slice, part or
term cannot pass.

Each element: half a unit of the output's rounding; the kernels round P, dS and (in Delta)
O by half a unit each, and P carries the rounding of a row sum taken over rounded weights
once more: at most 4 half units of the magnitude that is summed. An fp16 number below
2^-14 is off by up to 2^-25 instead, which counts once for every rounded P, dS and O with
what that is multiplied by, and for the output. Scores and sums are fp32.

All of a tensor: these roundings are independent, so the root mean square of the error is
that of the root of the summed squares of the single ones; twice it is allowed.
"""

from __future__ import annotations

import math

import pytest
import torch

from gki import _lib, cross_attention

DEV = "cuda"
NAMES = ("o", "dq", "dk", "dv")
DTYPES = [torch.bfloat16, torch.float16]


def _reference(q, k, v, do, lengths, dtype):
    """Per output: its value, the bound of each element, and the mean square that the
    roundings' independent errors have there, all in 64 bits."""
    B, H, n_q, D = q.shape
    H_kv = k.shape[1]
    g, scale = H // H_kv, 1 / math.sqrt(D)
    half = torch.finfo(dtype).eps / 2
    u = 2.0**-25 if dtype == torch.float16 else 0.0
    q, k, v, do = (t.double() for t in (q, k, v, do))
    out = [[torch.zeros_like(t) for t in (q, q, k, v)] for _ in range(3)]
    for b in range(B):
        n = lengths[b]
        for j in range(H_kv if n else 0):
            hs = slice(j * g, (j + 1) * g)
            Q, O_, K, V = q[b, hs].reshape(-1, D), do[b, hs].reshape(-1, D), k[b, j, :n], v[b, j, :n]
            P = torch.softmax(Q @ K.T * scale, -1)
            o = P @ V
            odo = o * O_
            ds = P * (O_ @ V.T - odo.sum(-1, keepdim=True)) * scale
            size = float((Q.abs() @ K.abs().T).max()) * scale
            # fp32: scores of D <= 128 terms off by 136 units of 2^-24 of their size, sums by 2^-24 a term
            f32 = 2 * 136 * 2.0**-24 * size + (max(n, g * n_q) + 300) * 2.0**-24
            rel = (4 * half + f32) * 1.02
            big = P * (O_.abs() @ V.abs().T + odo.abs().sum(-1, keepdim=True)) * scale
            # what 2^-25 in V scale, dO scale and O adds to dS, and the rounding of dS itself
            small = u * (1 + P * (O_.abs().sum(1, keepdim=True) * (1 + scale) + V.abs().sum(1)))
            x = (o, ds @ K, ds.T @ Q, P.T @ O_)
            bound = (rel * (P @ V.abs()) + u * (V.abs().sum(0) + n * (P @ V.abs())),
                     rel * (big @ K.abs()) + small @ K.abs(),
                     rel * (big.T @ Q.abs()) + small.T @ Q.abs(),
                     rel * (P.T @ O_.abs()) + u * O_.abs().sum(0))
            delta2 = half**2 * scale**2 * (odo**2).sum(1, keepdim=True)        # common to a row of dS
            eds = half**2 * 2 * ds**2 + (small + f32 * big) ** 2
            mean = (half**2 * (P**2 @ V**2 + 2 * o**2) + (f32 * (P @ V.abs())) ** 2 + u**2 * ((V**2).sum(0) + n * o**2),
                    eds @ K**2 + delta2 * (P @ K) ** 2 + 2 * half**2 * x[1] ** 2,
                    (eds + delta2 * P**2).T @ Q**2 + half**2 * x[2] ** 2,
                    (2 * half**2 * P**2 + (f32 * P) ** 2 + u**2).T @ O_**2 + half**2 * x[3] ** 2)
            for i, (a, e, m) in enumerate(zip(x, bound, mean)):
                e, m = half * a.abs() + e + u, m + u**2
                for kind, y in zip(out, (a, e, m)):
                    if i < 2:
                        kind[i][b, hs] = y.view(g, n_q, D)
                    else:
                        kind[i][b, j, :n] = y
    return out


def _wrong(got, reference):
    """The outputs that are off, with how far (1: at the bound)."""
    bad = {}
    for name, x, want, bound, mean in zip(NAMES, got, *reference):
        if x is None:
            continue
        err = (x.double() - want).abs()
        worst = float((err / bound).nan_to_num(0.0, 9.9e99, 9.9e99).max())        # 0 of 0 where there are no keys
        rms = float((err**2).mean().sqrt() / (2 * mean.mean().sqrt()))
        if not worst <= 1 or not rms <= 1 or not torch.isfinite(x).all():
            bad[name] = (worst, rms)
    return bad


def _inputs(B, H, H_kv, n_q, n_kv, D, dtype, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=gen).to(dtype).to(device)
            for s in ((B, H, n_q, D), (B, H_kv, n_kv, D), (B, H_kv, n_kv, D), (B, H, n_q, D))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,H_kv,n_q,n_kv,D", [(8, 1, 37, 3000, 128), (2, 2, 333, 5000, 64), (16, 2, 5, 1700, 128), (6, 2, 33, 1000, 128)])
def test_the_bounds_see_zeros_and_a_dropped_slice(dtype, H, H_kv, n_q, n_kv, D):
    tensors = _inputs(1, H, H_kv, n_q, n_kv, D, dtype, "cpu")
    ref = _reference(*tensors, [n_kv], dtype)
    right = [x.to(dtype) for x in ref[0]]
    assert not _wrong(right, ref)
    assert set(_wrong([torch.zeros_like(x) for x in right], ref)) == set(NAMES)
    fewer = _reference(*tensors, [n_kv - n_kv // 5], dtype)[0]         # the last fifth of the keys left out
    assert {"o", "dq", "dk", "dv"} == set(_wrong([x.to(dtype) for x in fewer], ref))
    q, k, v, do = tensors
    do = do.clone()
    do[:, :, -(-n_q // 5) * 4:] = 0                                    # of dK and dV the last rows' part
    part = _reference(q, k, v, do, [n_kv], dtype)[0]
    assert {"dk", "dv"} <= set(_wrong([None, None, part[2].to(dtype), part[3].to(dtype)], ref))


def _run(q, k, v, do, lengths):
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, n, enable_gqa=True)
    return (out.detach(), *torch.autograd.grad(out, leaves, do))


def _check(B, H, H_kv, n_q, n_kv, D, dtype, lengths=None, seed=0):
    tensors = _inputs(B, H, H_kv, n_q, n_kv, D, dtype, DEV, seed)
    ref = _reference(*tensors, lengths or [n_kv] * B, dtype)
    assert not _wrong(_run(*tensors, lengths), ref), (B, H, H_kv, n_q, n_kv, D)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,H_kv,n_q,n_kv,D,lengths", [
    (8, 1, 37, 3000, 128, (3000, 1777)), (2, 2, 333, 5000, 64, (5000,)), (16, 2, 5, 1700, 128, (1700, 3, 900)),
    (16, 16, 700, 500, 64, (500, 0, 333)), (6, 2, 33, 1000, 128, (999, 512)), (12, 1, 3, 400, 32, (400, 130)),
    (2, 2, 200, 31, 16, (31, 17)), (32, 4, 600, 1500, 128, (1500, 801)), (2, 2, 5000, 130, 128, None),
    (4, 1, 3000, 100, 32, None), (4, 4, 70, 2000, 16, (2000, 64)), (1, 1, 1, 8192, 64, (8192, 1)),
])
def test_shapes(dtype, H, H_kv, n_q, n_kv, D, lengths):
    _check(1 if lengths is None else len(lengths), H, H_kv, n_q, n_kv, D, dtype, lengths, seed=n_q + n_kv)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("splits", [0, 1, 2, 5, 33])
def test_any_number_of_slices(dtype, D, splits, monkeypatch):
    from gki import cross

    monkeypatch.setattr(cross, "_FWD_PLANS", {})
    monkeypatch.setattr(_lib.load(), "gki_cross_splits", lambda *a: splits)
    for H, H_kv, n_q, n_kv in ((4, 4, 1, 900), (16, 1, 2, 70), (20, 1, 4, 257), (2, 1, 70, 700)):
        _check(3, H, H_kv, n_q, n_kv, D, dtype, [n_kv, n_kv // 2, 0], seed=splits)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("parts,slices", [(1, 1), (2, 2), (3, 5), (7, 40)])
def test_any_number_of_parts(dtype, D, parts, slices, monkeypatch):
    from gki import cross

    def cut(*a):
        a[-1]._obj.value = slices
        return parts

    monkeypatch.setattr(cross, "_BWD_PLANS", {})
    monkeypatch.setattr(_lib.load(), "gki_cross_bwd_parts", cut)
    for H, H_kv, n_q, n_kv in ((2, 1, 3, 500), (3, 3, 130, 333), (2, 2, 20, 64)):
        _check(3, H, H_kv, n_q, n_kv, D, dtype, [n_kv, n_kv // 3, 0], seed=slices)
