"""Rotary positions with several axes against complex products in 64 bits, forward and
gradient.

Bounds: an output is half a unit of its type off, and what fp32 adds: the cosine and sine
(half a unit of 2^-23 from the library's function, 2^-28 of a turn from the reduced angle
in fp32: together below 2^-22), two products and a sum of three half units of 2^-23: below
2^-21 of |a| + |b|. Below an fp16 normal: 2^-25.
"""

from __future__ import annotations

import ctypes
import math
from decimal import Decimal, localcontext

import pytest
import torch
from torch.autograd import forward_ad

from gki import MultiAxisRotary, StreamingMaskSpec, _lib, block_sparse_attention, cross_attention, make_streaming_mask

DEV = "cuda"
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
NULL = ctypes.c_void_p(0)


def test_c_entry_refuses_before_launch():
    lib = _lib.load()
    six, three = ctypes.c_int64 * 6, ctypes.c_int64 * 3

    def call(q=16, out=16, heads=2, strides=(0, 128, 64, 0, 128, 64), k=0, k_out=0, k_heads=0, dtype=2, batch=1, n=3, D=64,
             turns=16, pairs=32, at=16):
        return lib.gki_rotary(q, out, heads, six(*strides), k, k_out, k_heads, six(*strides), dtype, batch, n, D, turns, 16,
                              pairs, 0, 0, at, 0, three(0, 0, 1), NULL)

    assert call(dtype=5) == 2 and call(D=48) == 2 and call(D=256) == 2 and call(q=0) == 1 and call(out=0) == 1
    assert call(q=24) == 1 and call(heads=0) == 1 and call(k=16) == 1 and call(k_heads=2) == 1 and call(k=16, k_heads=2) == 1
    assert call(strides=(0, 132, 64, 0, 128, 64)) == 1 and call(strides=(0, 128, 64, 0, 128, 60)) == 1
    assert call(dtype=0, strides=(0, 130, 64, 0, 128, 64)) == 1
    assert call(turns=0) == 1 and call(at=0) == 1 and call(pairs=0) == 1 and call(pairs=12) == 1 and call(pairs=40) == 1
    assert call(n=2**24) == 1 and call(batch=2**13, n=2**13) == 1 and call(n=-1) == 1 and call(n=0) == 0 and call(batch=0) == 0


@pytest.mark.parametrize("arguments,message", [
    ((48, (24,)), "head_dim"), ((64, ()), "sections"), ((64, (33,)), "sections"), ((64, (40,)), "sections"), ((64, (0, 32)), "sections"),
    ((64, (-8, 16)), "sections"), ((64, (32,), 0.0), "base"), ((64, (32,), math.nan), "base"), ((64, (32,), math.inf), "base")])
def test_sections_are_checked(arguments, message):
    with pytest.raises(ValueError, match=message):
        MultiAxisRotary(*arguments)


def _reference(x, positions, sections, base, interleaved, per_axis, sign=1):
    """x [..., H, N, D] in 64 bits; positions [axes, ..., 1, N]."""
    P, z, j = sum(sections), x.double(), 0
    phase = []
    for axis, size in enumerate(sections):
        for i in range(size):
            phase.append(positions[axis].double() * base ** -(i / size if per_axis else j / P))
            j += 1
    phase = torch.stack(phase, -1)
    c, s = torch.cos(phase), sign * torch.sin(phase)
    a, b = (z[..., 0:2 * P:2], z[..., 1:2 * P:2]) if interleaved else (z[..., :P], z[..., P:2 * P])
    u, v = a * c - b * s, a * s + b * c
    out, size = z.clone(), torch.zeros_like(z)
    for t, (one, two) in ((out, (u, v)), (size, (a.abs() + b.abs(),) * 2)):
        if interleaved:
            t[..., 0:2 * P:2], t[..., 1:2 * P:2] = one, two
        else:
            t[..., :P], t[..., P:2 * P] = one, two
    return out, size


def _close(got, want, size, dtype, tag=""):
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0     # fp32: among the 2^-21
    bound = half * want.abs() + 2.0**-21 * (1 + half) * size + (2.0**-25 if dtype == torch.float16 else 1e-37)
    err = (got.double() - want).abs()
    assert got.dtype == dtype and got.is_contiguous() and torch.isfinite(got).all(), tag
    assert (err <= bound).all(), (tag, (err / bound).max().item())
    # independent roundings: half a unit of the result each
    assert err.square().mean() <= 4 * (half**2 * want.square().mean() / 3 + (2.0**-22) ** 2 * size.square().mean() + 1e-16), tag


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("per_axis", [False, True])
@pytest.mark.parametrize("D,sections", [(16, (8,)), (16, (3, 5)), (32, (8,)), (64, (16, 16)), (64, (11, 10, 11)), (128, (64,)),
                                        (128, (16, 24, 24)), (128, (1, 6, 1)), (128, (20, 20))])
def test_against_64_bits(dtype, interleaved, per_axis, D, sections):
    gen = torch.Generator(device=DEV).manual_seed(D + len(sections))
    rope = MultiAxisRotary(D, sections, base=10000.0, interleaved=interleaved, per_axis=per_axis)
    for B, H, H_kv, N, far, wide in ((1, 1, 1, 1, 10, False), (2, 3, 1, 77, 2**30, True), (3, 8, 2, 700, 5000, False)):
        q, k = (torch.randn(B, h, N, D, generator=gen, device=DEV).to(dtype) for h in (H, H_kv))
        at = torch.randint(-far, far, (len(sections), B, N), generator=gen, device=DEV, dtype=torch.int64 if wide else torch.int32)
        got = rope(q, k, at)
        for x, y in zip((q, k), got):
            _close(y, *_reference(x, at[:, :, None], sections, 10000.0, interleaved, per_axis), dtype, (B, N))
        # packed rows give the same bits
        rows = [x.transpose(1, 2).reshape(B * N, -1, D) for x in (q, k)]
        packed = rope(rows[0], rows[1], at.reshape(len(sections), B * N))
        for x, y in zip(packed, got):
            assert torch.equal(x.view(B, N, -1, D).transpose(1, 2), y)


_PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
_FAR = [2**30 - 1, 2**30 - 77, 1054937413, 1073140401, 2**29 + 3, 777777777, 123456, 2**20 + 1, 3]


def _exact_turns(rope, p):
    """Of each pair at position p, reduced to half a turn on either side, from 50 digits."""
    with localcontext() as c:
        c.prec = 50
        out = []
        for j in range(rope.pairs):
            t = p * Decimal(rope.base) ** (-Decimal(j) / rope.pairs) / (2 * _PI)
            out.append(t - t.to_integral_value())
        return out


@pytest.mark.parametrize("base,pairs", [(1e6, 64), (100.0, 64), (10000.0, 24), (2.0, 64), (1.0, 8)])
def test_far_angles_are_as_close_as_stated(base, pairs):
    """The kernels' arithmetic on the host. In units of 2^-53 of the largest angle, 2^30: the frequency and its place in
    the ladder 0.92, 2 pi 0.35, the division and the product 1 each; fp32 adds 2^-28 of a turn: below 2^-21 in all."""
    rope, worst = MultiAxisRotary(128, (pairs,), base=base), 0.0
    turns = rope._table(torch.device("cpu"))[0].tolist()
    for p in _FAR:
        for turn, exact in zip(turns, _exact_turns(rope, p)):
            r = p * turn
            r -= round(r)
            quarter = round(4 * r)
            x = torch.tensor(2 * (r - 0.25 * quarter), dtype=torch.float32).item()
            off = Decimal(quarter) / 4 + Decimal(x) / 2 - exact
            worst = max(worst, abs(float((off - off.to_integral_value()) * 2 * _PI)))
    assert worst < 2.0**-21, worst * 2**23


@pytest.mark.gpu
@pytest.mark.parametrize("base,pairs", [(1e6, 64), (100.0, 64), (10000.0, 24), (1.0, 8)])
def test_far_positions_against_exact_angles(base, pairs):
    """Rows of ones and zeros come out as cosines and sines: 2^-21 from the angle, 2^-22 from the functions and
    their rounding."""
    rope = MultiAxisRotary(128, (pairs,), base=base)
    q = torch.zeros(len(_FAR), 1, 128, device=DEV)
    q[..., :pairs] = 1
    got, _ = rope(q, None, torch.tensor(_FAR, device=DEV))
    for row, p in zip(got[:, 0].tolist(), _FAR):
        for j, t in enumerate(_exact_turns(rope, p)):
            phase = float(t * 2 * _PI)
            assert abs(row[j] - math.cos(phase)) < 2.0**-21 + 2.0**-22, (p, j)
            assert abs(row[pairs + j] - math.sin(phase)) < 2.0**-21 + 2.0**-22, (p, j)


@pytest.mark.gpu
def test_more_tokens_than_a_group_and_than_2_31_elements():
    rope = MultiAxisRotary(128, (64,))
    q = torch.empty(2, 130, 65537, 128, dtype=torch.bfloat16, device=DEV).normal_()
    at = torch.arange(65537, device=DEV)
    assert q.numel() > 2**31
    out, none = rope(q, None, at)
    assert none is None
    for b, h, part in ((0, 0, slice(0, 50)), (1, 129, slice(65400, 65537)), (1, 0, slice(2045, 2055))):
        _close(out[b, h, part].contiguous(), *_reference(q[b, h, part], at[None, part], (64,), 10000.0, False, False), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_positions_of_every_form(dtype):
    gen = torch.Generator(device=DEV).manual_seed(3)
    rope = MultiAxisRotary(64, (12, 20))
    q, k = (torch.randn(3, h, 40, 64, generator=gen, device=DEV).to(dtype) for h in (4, 2))
    line = torch.randint(0, 9000, (40,), generator=gen, device=DEV)
    full = line.expand(2, 3, 40).contiguous()
    want = rope(q, k, full)
    for at in (line, line.int(), line[None], line.expand(2, 40), line.expand(1, 3, 40), full.int(), line.expand(2, 3, 40),
               torch.stack([line, line, line], 1).T[:2], torch.stack([full, full], 3)[..., 0]):
        for a, b in zip(rope(q, k, at), want):
            assert torch.equal(a, b)
    rows_q, rows_k = q[0].transpose(0, 1), k[0].transpose(0, 1)
    for at in (line, line[None], line.expand(2, 40)):
        for a, b in zip(rope(rows_q, rows_k, at), want):
            assert torch.equal(a, b[0].transpose(0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    gen = torch.Generator(device=DEV).manual_seed(4)
    rope = MultiAxisRotary(64, (12, 20), interleaved=True)
    q, k = (torch.randn(2, h, 33, 64, generator=gen, device=DEV).to(dtype) for h in (4, 2))
    at = torch.randint(0, 9000, (2, 2, 33), generator=gen, device=DEV)
    want = rope(q, k, at)
    odd = torch.empty(q.numel() + 1, dtype=dtype, device=DEV)[1:].view(q.shape).copy_(q)
    fused = torch.cat([q, k], 1).transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(2, 4, 33, 128, dtype=dtype, device=DEV)
    wide[..., 5:69] = q
    forms = [(odd, k), (q.transpose(1, 2).contiguous().transpose(1, 2), k), (fused[:, :4], fused[:, 4:]), (wide[..., 5:69], k),
             (q.transpose(2, 3).contiguous().transpose(2, 3), k)]
    for x, y in forms:
        for a, b in zip(rope(x, y, at), want):
            assert torch.equal(a, b) and a.is_contiguous()
    one = q[:1, :1].expand(2, 4, -1, -1)
    assert torch.equal(rope(one, None, at)[0], rope(one.contiguous(), None, at)[0])


@pytest.mark.gpu
def test_empty_tensors():
    rope = MultiAxisRotary(64, (32,))
    for shape in ((0, 4, 5, 64), (2, 4, 0, 64), (2, 0, 5, 64)):
        q = torch.empty(shape, device=DEV, requires_grad=True)
        k = torch.randn(shape[0], 2, shape[2], 64, device=DEV)
        a, b = rope(q, k, torch.arange(shape[2], device=DEV))
        assert a.shape == q.shape and b.shape == k.shape
        a.sum().backward()
        assert q.grad.shape == q.shape


# ---- gradients ------------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_turn_back(dtype, interleaved):
    gen = torch.Generator(device=DEV).manual_seed(5)
    sections = (16, 24, 24)
    rope = MultiAxisRotary(128, sections, interleaved=interleaved)
    base = [torch.randn(2, 45, h, 128, generator=gen, device=DEV).to(dtype) for h in (6, 2)]
    leaves = [t.requires_grad_(True) for t in base]
    at = torch.randint(0, 3000, (3, 2, 45), generator=gen, device=DEV)
    dq, dk = (torch.randn(2, h, 45, 128, generator=gen, device=DEV).to(dtype) for h in (6, 2))
    q, k = rope(*(t.transpose(1, 2) for t in leaves), at)
    got = torch.autograd.grad((q, k), leaves, (dq, dk), retain_graph=True)
    for g, d in zip(got, (dq, dk)):
        _close(g.transpose(1, 2).contiguous(), *_reference(d, at[:, :, None], sections, 10000.0, interleaved, False, -1), dtype)
    # one output alone, a broadcast gradient, an input that needs none
    only_k, = torch.autograd.grad(k, leaves[1], dk, retain_graph=True)
    assert torch.equal(only_k, got[1])
    summed, = torch.autograd.grad(q.sum(), leaves[0])
    ones = torch.ones_like(dq)
    _close(summed.transpose(1, 2).contiguous(), *_reference(ones, at[:, :, None], sections, 10000.0, interleaved, False, -1), dtype)
    frozen, turned = rope(base[0].detach().transpose(1, 2), leaves[1].transpose(1, 2), at)
    assert torch.equal(torch.autograd.grad(turned, leaves[1], dk)[0], got[1])
    packed_leaf = base[0].detach().reshape(90, 6, 128).requires_grad_(True)
    packed, _ = rope(packed_leaf, None, at.reshape(3, 90))
    back, = torch.autograd.grad(packed, packed_leaf, dq.transpose(1, 2).reshape(90, 6, 128))
    assert torch.equal(back.view(2, 45, 6, 128), got[0])


def _turned_by_copies(monkeypatch):
    """Launches replaced by copies, counted: what autograd asks for shows on the CPU."""
    launched = []

    def launch(self, q, k, positions, strides, inverse):
        launched.append(sum(t is not None for t in (q, k)))
        return q.clone(), None if k is None else k.clone()

    monkeypatch.setattr(MultiAxisRotary, "_launch", launch)
    return launched


@pytest.mark.parametrize("trained", ["q", "k", "both", "none"])
def test_a_frozen_tensor_is_returned_frozen(trained, monkeypatch):
    launched = _turned_by_copies(monkeypatch)
    q, k = torch.randn(5, 4, 64), torch.randn(5, 2, 64)
    if trained in ("q", "both"):
        q.requires_grad_(True)
    if trained in ("k", "both"):
        k.requires_grad_(True)
    rope, at = MultiAxisRotary(64, (32,)), torch.arange(5)
    turned = rope._apply(q, k, at, None, False)
    assert [t.requires_grad for t in turned] == [q.requires_grad, k.requires_grad] and launched == [2]
    if trained == "none":
        return
    leaves = [t for t in (q, k) if t.requires_grad]
    sums = [t.square().sum() for t in turned if t.requires_grad]
    grads = torch.autograd.grad(sum(sums), leaves, create_graph=True)
    assert launched == [2, len(leaves)] and all(g.requires_grad for g in grads)
    for leaf, second in zip(leaves, torch.autograd.grad(sum(g.sum() for g in grads), leaves)):
        assert torch.equal(second, torch.full_like(leaf, 2.0))


def test_a_gradient_that_is_not_asked_for_is_not_turned(monkeypatch):
    launched = _turned_by_copies(monkeypatch)
    q, k = torch.randn(5, 4, 64, requires_grad=True), torch.randn(5, 2, 64, requires_grad=True)
    a, b = MultiAxisRotary(64, (32,))._apply(q, k, torch.arange(5), None, False)
    dq, = torch.autograd.grad(a.sum() + b.sum(), q)
    assert torch.equal(dq, torch.ones_like(q)) and launched[0] == 2


@pytest.mark.gpu
@pytest.mark.parametrize("trained", [0, 1])
def test_frozen_beside_trained_costs_no_gradient_behind(trained):
    """The other tensor needs no gradient after its turn either: attention behind it gives none."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    rope = MultiAxisRotary(64, (32,))
    q, k, v = (torch.randn(1, 2, 130, 64, generator=gen, device=DEV) for _ in range(3))
    leaf = (q, k)[trained].requires_grad_(True)
    at = torch.arange(130, device=DEV)
    turned = rope(q, k, at)
    assert [t.requires_grad for t in turned] == [trained == 0, trained == 1]
    apart = [t.detach().requires_grad_(i == trained) for i, t in enumerate(turned)]
    do = torch.randn(1, 2, 130, 64, generator=gen, device=DEV)
    got, = torch.autograd.grad(cross_attention(*turned, v), leaf, do)
    behind, = torch.autograd.grad(cross_attention(*apart, v), apart[trained], do)
    # -1 times each position turns back: the same angles, cosines and sines
    assert torch.equal(got, rope(behind, None, -at)[0])


@pytest.mark.gpu
def test_gradient_against_differences_and_of_second_order():
    gen = torch.Generator(device=DEV).manual_seed(6)
    rope = MultiAxisRotary(32, (5, 3), base=100.0)
    q = torch.randn(1, 2, 5, 32, generator=gen, device=DEV, requires_grad=True)
    k = torch.randn(1, 1, 5, 32, generator=gen, device=DEV, requires_grad=True)
    at = torch.randint(0, 50, (2, 5), generator=gen, device=DEV)
    weight = torch.randn(1, 2, 5, 32, generator=gen, device=DEV)

    def loss(q, k):
        a, b = rope(q, k, at)
        return (a * weight).sum() + (a * b).square().sum()

    grads = torch.autograd.grad(loss(q, k), (q, k), create_graph=True)
    for which, (x, g) in enumerate(zip((q, k), grads)):
        d = torch.randn(x.shape, generator=gen, device=DEV)
        e = 2.0**-6                                 # a polynomial of degree 4: the central difference is off by e^2 f''' / 6
        moved = [loss(*(t + s * e * d if i == which else t for i, t in enumerate((q, k)))).double() for s in (1, -1, 2, -2)]
        slope = (8 * (moved[0] - moved[1]) - (moved[2] - moved[3])) / (12 * e)     # exact for degree 4
        # the losses' fp32 sums, divided by the step
        bound = 18 / (12 * e) * 2.0**-22 * float(loss(q, k).abs() + 500)
        assert abs(float((g * d).sum()) - float(slope)) <= bound
    # the second order against the same loss written with torch's products
    second = torch.autograd.grad((grads[0] * weight).sum(), (q, k))

    def plain(x):
        P = 8
        angle = at.double()[torch.tensor([0] * 5 + [1] * 3, device=DEV)].T * 100.0 ** (-torch.arange(8, device=DEV).double() / P)
        c, s = angle.cos(), angle.sin()
        a, b = x[..., :8], x[..., 8:16]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., 16:]], -1)

    q64, k64 = (t.detach().double().requires_grad_(True) for t in (q, k))
    a, b = plain(q64), plain(k64)
    first = torch.autograd.grad((a * weight.double()).sum() + (a * b).square().sum(), (q64, k64), create_graph=True)
    want = torch.autograd.grad((first[0] * weight.double()).sum(), (q64, k64))
    for x, y, w in zip(grads, first, (q64, k64)):
        assert (x.double() - y).abs().max() <= 2.0**-18 * y.abs().max()
    for x, y in zip(second, want):
        assert (x.double() - y).abs().max() <= 2.0**-18 * y.abs().max()


@pytest.mark.gpu
def test_before_the_sparse_op():
    """Queries and keys turned, then attended, with gradients through both: scores depend on
    distances alone, so positions moved together change nothing but roundings."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    N, D = 200, 64
    rope = MultiAxisRotary(D, (32,))
    mask = make_streaming_mask(N, N, StreamingMaskSpec(4, 64), 64, 64, device=DEV)
    leaves = [torch.randn(1, 2, N, D, generator=gen, device=DEV, requires_grad=True) for _ in range(3)]
    do = torch.randn(1, 2, N, D, generator=gen, device=DEV)
    results = []
    for shift in (0, 12345):
        q, k = rope(leaves[0], leaves[1], torch.arange(N, device=DEV) + shift)
        o = block_sparse_attention(q, k, leaves[2], mask, is_causal=True, sink_size=4, window_size=64)
        results.append((o,) + torch.autograd.grad(o, leaves, do))
    for a, b in zip(*results):
        # fp32: turns off by 2^-21 move scores by 2^-21 of sum |q k| (below 64 here), weights and sums by as much
        assert (a - b).abs().max() <= 64 * 2.0**-21 * 8 * a.abs().max()


# ---- refusals, streams, graphs -----------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_python_refusals():
    rope = MultiAxisRotary(64, (12, 20))
    q, k = torch.randn(2, 4, 10, 64, device=DEV), torch.randn(2, 2, 10, 64, device=DEV)
    at = torch.zeros(2, 2, 10, dtype=torch.int32, device=DEV)
    for call, message in ((lambda: rope(q[0, 0], None, at), "4-D|B, H, N, D"), (lambda: rope(q, k[0], at), "both"),
                          (lambda: rope(q.cpu(), None, at), "CUDA"), (lambda: rope(q.double(), None, at), "dtype"),
                          (lambda: rope(q, k.half(), at), "dtype"), (lambda: rope(q[..., :32], None, at), "head_dim"),
                          (lambda: rope(q, k[:, :, :9], at), "same tokens"), (lambda: rope(q, k[:1], at), "same tokens"),
                          (lambda: rope(q, k, at.float()), "int32 or int64"), (lambda: rope(q, k, at.cpu()), "live on"),
                          (lambda: rope(q, k, at[:, :, :9]), "positions"), (lambda: rope(q, k, at[:, :1]), "positions"),
                          (lambda: rope(q, k, torch.zeros(3, 10, dtype=torch.int32, device=DEV)), "positions"),
                          (lambda: rope(q, k, at[None]), "positions"), (lambda: rope(q[0], k[0][:3], at[0]), "same tokens"),
                          (lambda: rope(q[0], None, at), "positions"), (lambda: rope(q, k, at[0, 0, 0]), "positions")):
        with pytest.raises(ValueError, match=message):
            call()
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            rope(q, forward_ad.make_dual(k, torch.ones_like(k)), at)


@pytest.mark.gpu
def test_graph_of_a_training_pass_and_side_streams():
    gen = torch.Generator(device=DEV).manual_seed(8)
    rope = MultiAxisRotary(64, (12, 20))
    q, k = (torch.randn(2, h, 50, 64, generator=gen, device=DEV, requires_grad=True) for h in (4, 2))
    dq, dk = (torch.randn(2, h, 50, 64, generator=gen, device=DEV) for h in (4, 2))
    at = torch.randint(0, 500, (2, 50), generator=gen, device=DEV)

    def step():
        a, b = rope(q, k, at)
        return (a, b) + torch.autograd.grad((a, b), (q, k), (dq, dk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, [t.detach().clone() for t in step()]):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = [t.detach() for t in step()]
    for i in range(4):
        with torch.no_grad():
            for t in (q, k, dq, dk):
                t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
            at.copy_(torch.randint(0, 500, (2, 50), generator=gen, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b), i
