"""Cross attention over padded batches: forward, gradients and single tokens.

GPU: outputs and gradients against 64 bits, each element within a bound derived from
the roundings on its way (``_bounds``); gradients also against differences. CPU:
refusals and the launch rules.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from gki import _lib, cross_attention
from oracle.cache8 import attention64

DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


# ---- CPU -------------------------------------------------------------------------


def test_python_refusals():
    q = torch.zeros(2, 4, 3, 64)
    with pytest.raises(ValueError, match="4-D"):
        cross_attention(q[0], q, q)
    with pytest.raises(ValueError, match="CUDA"):
        cross_attention(q, q, q)


def test_c_entries_refuse_before_launch():
    lib, null = _lib.load(), ctypes.c_void_p(0)

    def fwd(q=16, o=16, dtype=2, H=4, H_kv=2, n_q=3, n_kv=9, D=64, scale=0.1, ws=0, splits=0):
        return lib.gki_cross_fwd(q, 16, 16, o, 16, dtype, 1, H, H_kv, n_q, n_kv, D, None, scale, ws, splits, null)

    def bwd(dq=16, dtype=2, H_kv=2, n_kv=9, D=64, scale=0.1, parts=1, partials=0, slices=1, sums=0):
        return lib.gki_cross_bwd(16, 16, 16, 16, 16, 16, dq, 16, 16, 16, dtype, 1, 4, H_kv, 3, n_kv, D, None, scale,
                                 parts, partials, slices, sums, null)

    assert fwd(dtype=9) == 2 and fwd(D=48) == 2 and fwd(H_kv=3) == 1 and fwd(n_q=0) == 1 and fwd(n_kv=0) == 1
    assert fwd(q=0) == 1 and fwd(q=20) == 1 and fwd(scale=math.nan) == 1 and fwd(splits=-1) == 1
    assert fwd(splits=2) == 1 and b"workspace" in lib.gki_last_error()
    assert fwd(splits=2, dtype=0) == 1 and fwd(splits=1, D=16) == 2 and fwd(ws=20, splits=2) == 1
    assert fwd(n_kv=2**30) == 1
    assert bwd(dtype=9) == 2 and bwd(D=8) == 2 and bwd(H_kv=3) == 1 and bwd(dq=0) == 1 and bwd(dq=8) == 1
    assert bwd(slices=0) == 1 and bwd(slices=2) == 1 and bwd(sums=8) == 1 and bwd(slices=2**22, sums=16) == 1
    assert lib.gki_cross_bwd(16, 16, 16, 16, 16, 16, 16, 0, 16, 16, 2, 1, 4, 2, 3, 9, 64, None, 0.1, 1, 0, 1, 0, null) == 1
    assert bwd(parts=0) == 1 and bwd(parts=2) == 1 and bwd(partials=8) == 1 and bwd(scale=math.inf) == 1


def test_launch_rules():
    lib = _lib.load()
    assert lib.gki_cross_splits(2, 1, 4, 1, 2**29, 2000, 64) == 0         # group * n_q past 31 bits
    assert lib.gki_cross_splits(2, 1, 8, 8, 200, 8000, 128) > 1           # few tiles, long keys: streams
    assert lib.gki_cross_splits(2, 16, 16, 16, 200, 8000, 128) == 0
    assert lib.gki_cross_splits(2, 16, 16, 16, 1, 2000, 64) >= 1          # a step: streams
    assert lib.gki_cross_splits(0, 16, 16, 16, 300, 2000, 64) == 0        # fp32: q tiles
    assert lib.gki_cross_splits(0, 1, 8, 8, 1, 2000, 64) > 1              # or slices of their keys
    assert lib.gki_cross_splits(0, 1, 8, 8, 1, 300, 64) == 0
    assert lib.gki_cross_splits(2, 16, 16, 16, 1, 2000, 16) == 0
    assert lib.gki_cross_splits(2, 16, 16, 16, 500, 2000, 64) == 0
    for dtype in (0, 2):
        for n_q, n_kv, H, H_kv, D in ((1, 1, 1, 1, 16), (2048, 64, 32, 4, 128), (70000, 50, 8, 1, 64), (64, 8192, 4, 4, 32)):
            slices = ctypes.c_int32()
            parts = lib.gki_cross_bwd_parts(dtype, 1, H, H_kv, n_q, n_kv, D, ctypes.byref(slices))
            assert parts == lib.gki_cross_bwd_parts(dtype, 1, H, H_kv, n_q, n_kv, D, None)
            assert 1 <= slices.value <= max(1, n_kv // 256)
            assert 1 <= parts <= max(1, -(-n_q // 64) * H // H_kv)


# ---- GPU -------------------------------------------------------------------------


def _gradients64(q, k, v, do, lengths, scale):
    """O, dQ, dK, dV in 64 bits, entry by entry, and magnitudes for the bounds: |P||V| for
    O, |dS'||K| for dQ, |dS'|^T|Q| for dK, P^T|dO| for dV, where |dS'| is P (|dO||V| +
    |O||dO|) |scale|, what dS is a difference of."""
    B, H, n_q, D = q.shape
    H_kv = k.shape[1]
    g = H // H_kv
    q, k, v, do = (t.double() for t in (q, k, v, do))
    vals = [torch.zeros_like(t) for t in (q, q, k, v)]
    mags = [torch.zeros_like(t) for t in (q, q, k, v)]
    sizes = torch.zeros(B, H_kv, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lengths[b])
        if n == 0:
            continue
        for j in range(H_kv):
            hs = slice(j * g, (j + 1) * g)
            qq, dd, kk, vv = q[b, hs].reshape(-1, D), do[b, hs].reshape(-1, D), k[b, j, :n], v[b, j, :n]
            p = torch.softmax(qq @ kk.T * scale, -1)
            o = p @ vv
            ds = p * (dd @ vv.T - (o * dd).sum(-1, keepdim=True)) * scale
            big = p * (dd.abs() @ vv.abs().T + (o * dd).abs().sum(-1, keepdim=True)) * abs(scale)
            for t, x in ((vals[0], o), (vals[1], ds @ kk), (mags[0], p @ vv.abs()), (mags[1], big @ kk.abs())):
                t[b, hs] = x.view(g, n_q, D)
            for t, x in ((vals[2], ds.T @ qq), (vals[3], p.T @ dd), (mags[2], big.T @ qq.abs()), (mags[3], p.T @ dd.abs())):
                t[b, j, :n] = x
            sizes[b, j] = (qq.abs() @ kk.abs().T).max() * abs(scale)
    return vals, mags, float(sizes.max())


def _bounds(vals, mags, size, terms, dtype):
    """Largest |error| per element. Half a unit of the output's rounding; the 16-bit kernels
    round P, dS and (in Delta) O by half a unit each, and P carries the rounding of a row
    sum taken over rounded weights once more: at most 4 half units of the magnitude that
    is summed. fp32: scores of D <= 128 terms, off by at most 136 units of 2^-24 of their
    size, move P by as much; sums of `terms` terms by 2^-24 each."""
    half = torch.finfo(dtype).eps / 2
    rel = (4 * half if dtype != torch.float32 else 0) + 2 * 136 * 2.0**-24 * size + (terms + 300) * 2.0**-24
    tiny = torch.finfo(dtype).tiny * 2 if dtype == torch.float16 else 1e-30
    return [half * x.abs() + rel * 1.02 * m + tiny * terms for x, m in zip(vals, mags)]


def _run(q, k, v, do, lengths, scale=None, gqa=True):
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, lengths, scale, enable_gqa=gqa)
    grads = torch.autograd.grad(out, leaves, do)
    return (out.detach(), *grads)


def _compare(got, q, k, v, do, lengths, scale=None):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    n = [k.shape[2]] * q.shape[0] if lengths is None else [min(max(int(x), 0), k.shape[2]) for x in lengths]
    vals, mags, size = _gradients64(q, k, v, do, n, scale)
    terms = max(k.shape[2], q.shape[2] * q.shape[1] // k.shape[1])
    for name, x, want, bound in zip(("o", "dq", "dk", "dv"), got, vals, _bounds(vals, mags, size, terms, q.dtype)):
        assert torch.isfinite(x).all(), name
        err = (x.double() - want).abs()
        assert (err <= bound).all(), (name, (err / bound).max().item())
    for b, m in enumerate(n):
        assert not got[2][b, :, m:].any() and not got[3][b, :, m:].any()
        if m == 0:
            assert not got[0][b].any() and not got[1][b].any()


def _inputs(B, H, H_kv, n_q, n_kv, D, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(s, generator=gen, device=DEV) * scale).to(dtype)
            for s in ((B, H, n_q, D), (B, H_kv, n_kv, D), (B, H_kv, n_kv, D), (B, H, n_q, D))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_dim", [16, 32, 64, 128])
@pytest.mark.parametrize("H,H_kv,n_q,n_kv,lengths", [
    (1, 1, 1, 1, (1, 0)), (2, 2, 1, 64, (64, 63)), (3, 1, 5, 65, (65, 1, 0)), (2, 2, 64, 63, (62, 63)),
    (4, 2, 65, 129, (128, 64, 129)), (2, 1, 127, 300, (0, 300)), (8, 8, 128, 128, (128, 65)), (2, 2, 200, 31, (31, 17)),
    (6, 2, 33, 1000, (999, 512)), (4, 4, 300, 200, None), (12, 1, 3, 400, (400, 130)),
])
def test_forward_and_gradients(dtype, head_dim, H, H_kv, n_q, n_kv, lengths):
    B = 2 if lengths is None else len(lengths)
    q, k, v, do = _inputs(B, H, H_kv, n_q, n_kv, head_dim, dtype, seed=n_q * 1000 + n_kv)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    _compare(_run(q, k, v, do, n), q, k, v, do, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,H_kv,n_q,n_kv,D", [
    (3, 16, 16, 700, 500, 64),      # grids past the ones whose tiles share their keys
    (2, 32, 4, 600, 1500, 128), (1, 4, 1, 3000, 100, 32),    # long walks of few kv tiles: cut into parts
    (1, 2, 2, 5000, 130, 128), (9, 16, 8, 130, 640, 16),
    (2, 8, 1, 37, 3000, 128), (1, 2, 2, 333, 5000, 64), (8, 16, 2, 5, 1700, 128),    # few tiles: streams of several row tiles
])
def test_larger_grids(dtype, B, H, H_kv, n_q, n_kv, D):
    q, k, v, do = _inputs(B, H, H_kv, n_q, n_kv, D, dtype, seed=7)
    gen = torch.Generator().manual_seed(n_kv)
    n = torch.randint(0, n_kv + 1, (B,), generator=gen).to(torch.int32).to(DEV)
    n[0] = n_kv
    _compare(_run(q, k, v, do, n), q, k, v, do, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("splits", [0, 1, 2, 5, 33])
def test_single_tokens_at_any_number_of_slices(dtype, D, splits, monkeypatch):
    if D == 16 and dtype != torch.float32:
        splits = 0                                # no streams

    from gki import cross

    monkeypatch.setattr(cross, "_FWD_PLANS", {})
    lib = _lib.load()
    monkeypatch.setattr(lib, "gki_cross_splits", lambda *a: splits)
    for H, H_kv, n_q, n_kv in ((4, 4, 1, 900), (8, 2, 2, 130), (16, 1, 2, 70), (20, 1, 4, 257), (5, 1, 1, 1), (2, 1, 70, 300)):
        q, k, v, _ = _inputs(3, H, H_kv, n_q, n_kv, D, dtype, seed=splits)
        n = torch.tensor([n_kv, n_kv // 2, 0], device=DEV)          # int64
        out = cross_attention(q, k, v, n, enable_gqa=True)
        do = torch.zeros_like(q)
        vals, mags, size = _gradients64(q, k, v, do, n.tolist(), D**-0.5)
        bound = _bounds(vals[:1], mags[:1], size, n_kv, dtype)[0]
        assert ((out.double() - vals[0]).abs() <= bound).all(), (H, H_kv, n_q, n_kv)
        assert not out[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("parts,slices", [(1, 1), (2, 2), (3, 5), (7, 40)])
def test_gradients_at_any_number_of_parts(dtype, D, parts, slices, monkeypatch):
    from gki import cross

    monkeypatch.setattr(cross, "_BWD_PLANS", {})

    def cut(*a):
        a[-1]._obj.value = slices
        return parts

    monkeypatch.setattr(_lib.load(), "gki_cross_bwd_parts", cut)
    for H, H_kv, n_q, n_kv in ((2, 1, 3, 500), (3, 3, 130, 333), (2, 2, 20, 64)):
        q, k, v, do = _inputs(3, H, H_kv, n_q, n_kv, D, dtype, seed=slices)
        n = torch.tensor([n_kv, n_kv // 3, 0], dtype=torch.int32, device=DEV)
        _compare(_run(q, k, v, do, n), q, k, v, do, n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 0.125, 1.0, 2.0**-40])
def test_any_finite_scale(dtype, scale):
    for n_q in (2, 150):
        q, k, v, do = _inputs(2, 4, 2, n_q, 200, 64, dtype, seed=11)
        n = torch.tensor([200, 77], dtype=torch.int32, device=DEV)
        _compare(_run(q, k, v, do, n, scale), q, k, v, do, n, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("n_q", [1, 140])
def test_padding_may_hold_anything(dtype, D, n_q):
    q, k, v, do = _inputs(3, 4, 2, n_q, 190, D, dtype, seed=5)
    n = torch.tensor([190, 70, 0], dtype=torch.int32, device=DEV)
    want = _run(q, k, v, do, n)
    k2, v2 = k.clone(), v.clone()
    for t, bad in ((k2, math.nan), (v2, math.inf)):
        t[1, :, 70:] = bad
        t[2] = bad
    got = _run(q, k2, v2, do, n)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    _compare(want, q, k, v, do, n)


@pytest.mark.gpu
@pytest.mark.parametrize("n_q", [2, 70])
def test_keys_past_2_31_elements(n_q):
    n_kv, held = 9_000_000, 200                       # entry 2 starts 2.3e9 elements into K and V
    q, k0, v0, do = _inputs(3, 2, 1, n_q, held, 128, torch.bfloat16, seed=13)
    k, v = (torch.full((3, 1, n_kv, 128), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k[:, :, :held], v[:, :, :held] = k0, v0
    n = torch.tensor([1, 0, held], dtype=torch.int32, device=DEV)
    out, dq, dk, dv = _run(q, k, v, do, n)
    assert not dk[:, :, held:].any() and not dv[:, :, held:].any()
    _compare((out, dq, dk[:, :, :held], dv[:, :, :held]), q, k0, v0, do, n)


@pytest.mark.gpu
def test_strided_lengths_and_two_graphs():
    """Lengths from a strided tensor; two captured graphs of one shape replayed in turn."""
    q, k, v, _ = _inputs(2, 8, 2, 1, 3000, 128, torch.bfloat16, seed=17)
    pairs = torch.tensor([[3000, 5], [1234, 7]], dtype=torch.int32, device=DEV)
    want = [cross_attention(q, k, v, pairs[:, i].contiguous(), enable_gqa=True) for i in range(2)]
    assert all(torch.equal(cross_attention(q, k, v, pairs[:, i], enable_gqa=True), want[i]) for i in range(2))
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            outs.append(cross_attention(q, k, v, pairs[:, i], enable_gqa=True))
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
def test_lengths_outside_the_range_count_as_the_nearest():
    q, k, v, do = _inputs(4, 2, 2, 40, 100, 64, torch.bfloat16)
    inside = torch.tensor([100, 0, 100, 50], device=DEV)
    want = _run(q, k, v, do, inside)
    for n in (torch.tensor([200, -1, 2**31 - 1, 50], dtype=torch.int32, device=DEV),
              torch.tensor([2**40, -(2**40), 101, 50], device=DEV)):
        for a, b in zip(_run(q, k, v, do, n), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_empty_inputs():
    for n_q, n_kv in ((0, 5), (5, 0), (0, 0)):
        q, k, v, do = _inputs(2, 2, 2, n_q, n_kv, 64, torch.float16)
        got = _run(q, k, v, do, None)
        assert [t.shape for t in got] == [q.shape, q.shape, k.shape, v.shape]
        assert not any(t.any() for t in got)


@pytest.mark.gpu
def test_strides_broadcast_keys_and_odd_alignment():
    B, H, n_q, n_kv, D = 2, 4, 70, 90, 64
    gen = torch.Generator(device=DEV).manual_seed(3)
    kv = torch.randn((1, n_kv, 2, H, D), generator=gen, device=DEV).to(torch.bfloat16).requires_grad_(True)
    qs = torch.randn((B * n_q * H * D + 1,), generator=gen, device=DEV).to(torch.bfloat16)
    q = qs[1:].view(B, n_q, H, D).transpose(1, 2)
    k, v = (kv[:, :, i].transpose(1, 2).expand(B, H, n_kv, D) for i in range(2))
    out = cross_attention(q, k, v)
    do = torch.randn((B, H, n_q, D), generator=gen, device=DEV).to(torch.bfloat16)
    (grad,) = torch.autograd.grad(out, kv, do)
    kc, vc = k.detach().contiguous(), v.detach().contiguous()
    plain = _run(q.contiguous(), kc, vc, do, None)
    assert torch.equal(out, plain[0])
    want = torch.stack([plain[2].float().sum(0, keepdim=True), plain[3].float().sum(0, keepdim=True)], 1)
    torch.testing.assert_close(grad.float(), want.permute(0, 3, 1, 2, 4), rtol=2**-7, atol=1e-2)


@pytest.mark.gpu
def test_gradients_against_differences():
    q, k, v, do = _inputs(2, 2, 1, 5, 70, 16, torch.float32, seed=9, scale=0.5)
    n = torch.tensor([70, 33], dtype=torch.int32, device=DEV)
    got = _run(q, k, v, do, n)
    gen = torch.Generator(device=DEV).manual_seed(1)
    for i, t in enumerate((q, k, v)):
        step = torch.randn(t.shape, generator=gen, device=DEV)
        eps = 2.0**-7
        args = [[x, y] for x, y in ((q, q), (k, k), (v, v))]
        args[i] = [t + eps * step, t - eps * step]
        up, down = (cross_attention(*(a[j] for a in args), n, enable_gqa=True).double() for j in (0, 1))
        numeric = ((up - down) * do.double()).sum() / (2 * eps)
        exact = (got[i + 1].double() * step.double()).sum()
        # central differences: eps^2 of a third derivative of order one per term, and the
        # outputs' 2^-22 over 2 eps, summed over the outputs in quadrature
        assert abs(numeric - exact) <= 3e-3 * (1 + abs(exact)), i


@pytest.mark.gpu
def test_no_gradient_needed_once_differentiable_and_same_bits():
    q, k, v, do = _inputs(2, 2, 2, 50, 60, 64, torch.bfloat16)
    leaf = q.clone().requires_grad_(True)
    with torch.no_grad():
        a = cross_attention(leaf, k, v)
    b = cross_attention(leaf, k, v)
    assert not a.requires_grad and b.requires_grad and torch.equal(a, b)
    (g1,) = torch.autograd.grad(b, leaf, do, retain_graph=True)
    (g2,) = torch.autograd.grad(b, leaf, do)
    assert torch.equal(g1, g2)
    out = cross_attention(leaf, k, v)
    (g,) = torch.autograd.grad(out, leaf, do, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,n_q,n_kv", [(64, 50, 200), (128, 300, 130), (32, 5, 3000), (64, 5, 0)])
def test_gradients_of_some_inputs_only(dtype, D, n_q, n_kv):
    q, k, v, do = _inputs(2, 4, 2, n_q, n_kv, D, dtype, seed=19)
    full = _run(q, k, v, do, None)
    for wanted in ((0,), (1,), (2,), (0, 2)):
        leaves = [t.detach().clone().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        out = cross_attention(*leaves, enable_gqa=True)
        got = torch.autograd.grad(out, [leaves[i] for i in wanted], do)
        assert all(torch.equal(g, full[1 + i]) for g, i in zip(got, wanted)), wanted


@pytest.mark.gpu
def test_side_stream_and_graph():
    q, k, v, do = _inputs(2, 4, 2, 90, 300, 64, torch.bfloat16)
    n = torch.tensor([300, 111], dtype=torch.int32, device=DEV)
    want = _run(q, k, v, do, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, do, n)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(cross_attention(*leaves, n, enable_gqa=True), leaves, do)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cross_attention(*leaves, n, enable_gqa=True)
        grads = torch.autograd.grad(out, leaves, do)
    gen = torch.Generator(device=DEV).manual_seed(2)
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(q.shape, generator=gen, device=DEV).to(q.dtype))
            n.copy_(torch.tensor([300 - 17 * i, 5 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(*(t.detach() for t in leaves), do, n)
        for a, b in zip((out, *grads), eager):
            assert torch.equal(a, b), i


@pytest.mark.gpu
def test_gpu_refusals():
    q, k, v, _ = _inputs(2, 4, 2, 3, 9, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="mismatch"):
        cross_attention(q, k, v)                                 # grouped heads without enable_gqa
    with pytest.raises(ValueError, match="share shape"):
        cross_attention(q, k, v[:, :, :5], enable_gqa=True)
    with pytest.raises(ValueError, match="dtype"):
        cross_attention(q, k.half(), v.half(), enable_gqa=True)
    with pytest.raises(ValueError, match="head_dim"):
        cross_attention(*(t[..., :48] for t in (q, k, v)), enable_gqa=True)
    for bad in (torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(2, device=DEV), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="kv_lengths"):
            cross_attention(q, k, v, bad, enable_gqa=True)
    with pytest.raises(ValueError, match="finite"):
        cross_attention(q, k, v, softmax_scale=math.inf, enable_gqa=True)
