"""A prefix that the sequences of a batch share, in front of their rolling caches (16-bit
and 8-bit): the decode against 64 bits over the joined keys, refusals, and a run of the
whole: prompt encoded, prefix set, sequences stepped, cross attention beside them.

Bounds: ``oracle.cache8.output_bound``. The weights are rounded once to 16 bits for P V
(half a unit each) and, where the rows run as 128-row tiles, summed as rounded: at most
one half unit more; 8-bit rows under fp16 queries take two pieces, but the prefix's do not.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from gki import StreamingKVCache, StreamingMaskSpec, _lib, cross_attention
from oracle import cache8
from oracle import streaming_oracle as so

DEV = "cuda"
F8 = torch.float8_e4m3fn


def test_c_entry_refuses_before_launch():
    lib, null = _lib.load(), ctypes.c_void_p(0)

    def call(q=16, ks=0, vs=0, pk=16, n_prefix=5, o=16, dtype=2, H=4, H_kv=2, n_q=1, D=64, ring=8, length=5, s=0.1,
             ws=16, n_ps=1, n_s=1):
        return lib.gki_rolling_prefix_decode(q, 16, 16, ks, vs, pk, 16, n_prefix, o, 16, dtype, 2, H, H_kv, n_q, D, 0, 8,
                                             ring, length, s, ws, n_ps, n_s, null)

    assert call(dtype=0) == 2 and call(dtype=7) == 2 and call(D=32) == 2 and call(n_q=5) == 2
    assert call(q=0) == 1 and call(pk=0) == 1 and call(ws=0) == 1 and call(ks=16) == 1 and call(pk=24) == 1
    assert call(ws=20) == 1 and call(o=8) == 1 and call(n_prefix=0) == 1 and call(n_prefix=2**30) == 1
    assert call(n_ps=0) == 1 and call(n_s=0) == 1 and call(H=3) == 1 and call(ring=2) == 1 and call(s=math.nan) == 1
    assert call(n_ps=2**24) == 1
    for rows in ((1, 1), (8, 8), (64, 8), (1024, 8)):
        own = ctypes.c_int32()
        assert lib.gki_prefix_splits(2, rows[0], rows[1], 1, 1, 128, 100, 100, ctypes.byref(own)) == 1 and own.value == 1
        assert 1 <= lib.gki_prefix_splits(2, rows[0], rows[1], 1, 1, 128, 100000, 5000, ctypes.byref(own)) <= 100000 // 256
        assert 1 <= own.value <= 5000 // 128
        assert lib.gki_prefix_splits(2, rows[0], rows[1], 1, 1, 128, 100, 100, None) == 1


def _check(cache, q, pk, pv, k, v, scale=None, tag=""):
    """One attend against 64 bits over [prefix, own]; k, v [B, H_kv, length, D]."""
    dtype, B, n_q, length, P = q.dtype, q.shape[0], q.shape[2], k.shape[2], pk.shape[2]
    o, lse = cache.attend(q, scale, return_lse=True)
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    own = torch.from_numpy(so.token_mask(n_q, length, cache.sink_size, cache.window_size)).to(DEV)
    vis = torch.cat([torch.ones(n_q, P, dtype=torch.bool, device=DEV), own], 1)
    rows = [k.double(), v.double()]
    if cache.k_scale is not None:
        rows = [torch.from_numpy(cache8.stored_values(t.cpu().numpy())).to(DEV) for t in rows]
    kk, vv = (torch.cat([p.double().expand(B, -1, -1, -1), t], 2) for p, t in zip((pk, pv), rows))
    want, want_lse, pabs, size = cache8.attention64(q, kk, vv, vis, scale)
    half = torch.finfo(dtype).eps / 2
    bound = cache8.output_bound(want, pabs, size, int(vis.sum(-1).max()), dtype, 2 * half)
    err = (o.double() - want).abs()
    assert torch.isfinite(o).all(), tag
    assert (err <= bound).all(), (tag, (err / bound).max().item())
    # a row sum over rounded weights moves the LSE by at most half a unit
    lse_bound = half * 1.01 + 136 * 2.0**-24 * size + (vis.shape[1] + 16) * 2.0**-24 + 2.0**-23 * want_lse.abs()
    assert ((lse.double() - want_lse).abs() <= lse_bound).all(), tag


def _make(B, H, H_kv, n_q, P, length, D, dtype, seed=0, sink=4, window=100, bits=16):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(b, h, n):
        return torch.randn((b, h, n, D), generator=gen, device=DEV).to(dtype)

    q, pk, pv, k, v = normal(B, H, n_q), normal(1, H_kv, P), normal(1, H_kv, P), normal(B, H_kv, length), normal(B, H_kv, length)
    cache = StreamingKVCache(B, H_kv, D, StreamingMaskSpec(sink, window), dtype, DEV,
                             storage_dtype=F8 if bits == 8 else None)
    cache.set_prefix(pk, pv)
    cache.append(k, v)
    return cache, q, pk, pv, k, v


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H,H_kv,n_q,P,length,sink,window", [
    (1, 1, 1, 1, 1, 1, 4, 100), (1, 2, 2, 1, 64, 5, 0, 3), (3, 4, 2, 1, 65, 200, 4, 64), (2, 8, 1, 2, 1000, 70, 1, 50),
    (4, 16, 2, 2, 130, 33, 0, 0), (5, 26, 2, 1, 333, 100, 4, 100), (9, 16, 1, 1, 500, 20, 4, 100), (40, 4, 1, 4, 129, 9, 2, 5),
    (33, 4, 4, 1, 63, 300, 4, 256), (129, 2, 2, 1, 64, 2, 4, 100), (64, 8, 2, 1, 2049, 1, 4, 8), (1, 40, 1, 4, 700, 500, 4, 300),
])
def test_decode_against_64_bits(dtype, bits, D, B, H, H_kv, n_q, P, length, sink, window):
    case = _make(B, H, H_kv, n_q, P, max(length, n_q), D, dtype, B * 100 + P, sink, window, bits)
    _check(*case)


@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 20])
@pytest.mark.parametrize("n_ps,n_s", [(1, 1), (3, 2), (40, 5)])
def test_any_number_of_slices(B, n_ps, n_s, monkeypatch):
    lib = _lib.load()

    def splits(*a):
        a[-1]._obj.value = n_s
        return n_ps

    monkeypatch.setattr(lib, "gki_prefix_splits", splits)
    for bits in (16, 8):
        _check(*_make(B, 8, 2, 1, 300, 150, 128, torch.bfloat16, 3, bits=bits))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.2, 0.7])
def test_any_finite_scale(scale):
    for B in (2, 40):
        for bits in (16, 8):
            _check(*_make(B, 4, 2, 2, 200, 90, 64, torch.float16, 5, bits=bits), scale=scale)


@pytest.mark.gpu
def test_large_logits_in_either_part():
    for B in (2, 40):
        for which in (0, 1):
            cache, q, pk, pv, k, v = _make(B, 8, 2, 1, 200, 90, 128, torch.bfloat16, 6)
            if which:
                pk = pk * 6
                cache.set_prefix(pk, pv)
            else:
                k = k * 6
                cache.reset()
                cache.append(k, v)
            _check(cache, q * 2, pk, pv, k, v)


@pytest.mark.gpu
def test_prefix_set_changed_and_removed():
    cache, q, pk, pv, k, v = _make(2, 4, 2, 1, 100, 50, 64, torch.bfloat16, 7)
    with_prefix = cache.attend(q)
    plain = StreamingKVCache(2, 2, 64, StreamingMaskSpec(4, 100), torch.bfloat16, DEV)
    plain.append(k, v)
    cache.set_prefix(None, None)
    assert torch.equal(cache.attend(q), plain.attend(q))
    cache.set_prefix(pk[:, :, :0], pv[:, :, :0])
    assert torch.equal(cache.attend(q), plain.attend(q))
    wide = torch.cat([pk, pk], 3)[..., :64]                      # not contiguous
    cache.set_prefix(wide, pv)
    assert torch.equal(cache.attend(q), with_prefix)
    cache.reset()
    cache.append(k[:, :, :3], v[:, :, :3])
    _check(cache, q, pk, pv, k[:, :, :3], v[:, :, :3])


@pytest.mark.gpu
def test_python_refusals():
    cache, q, pk, pv, k, v = _make(2, 4, 2, 1, 10, 5, 64, torch.bfloat16)
    for bad, message in (((pk, None), "both"), ((pk[0], pv[0]), r"\[1, 2, P, 64\]"), ((pk.half(), pv.half()), "bfloat16"),
                         ((pk, pv[:, :, :4]), "share shape"), ((pk.expand(2, -1, -1, -1), pv.expand(2, -1, -1, -1)), r"\[1, 2"),
                         ((pk.cpu(), pv.cpu()), "live on")):
        with pytest.raises(ValueError, match=message):
            cache.set_prefix(*bad)
    _check(cache, q, pk, pv, k, v)                               # the prefix before is still there
    fp32 = StreamingKVCache(1, 1, 64, StreamingMaskSpec(4, 8), torch.float32, DEV)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        fp32.set_prefix(torch.zeros(1, 1, 3, 64, device=DEV), torch.zeros(1, 1, 3, 64, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 24])
def test_graph_and_side_stream(B):
    cache, q, pk, pv, k, v = _make(B, 8, 2, 1, 300, 90, 128, torch.bfloat16, 8, bits=8)
    want = cache.attend(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(q)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = cache.attend(q)
    for i in range(3):
        q.copy_(torch.randn_like(q))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cache.attend(q)), i


@pytest.mark.gpu
def test_the_operators_together():
    """A decoder's layer: steps of a batch behind a shared prefix, its own tokens in 8
    bits, each step's output attending an encoder's padded states."""
    dtype, B, H, H_kv, D = torch.bfloat16, 6, 8, 2, 64
    gen = torch.Generator(device=DEV).manual_seed(9)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV).to(dtype)

    pk, pv = normal(1, H_kv, 200, D), normal(1, H_kv, 200, D)
    ek, ev = normal(B, H_kv, 90, D), normal(B, H_kv, 90, D)
    lengths = torch.tensor([90, 1, 50, 0, 33, 64], dtype=torch.int32, device=DEV)
    cache = StreamingKVCache(B, H_kv, D, StreamingMaskSpec(2, 20), dtype, DEV, storage_dtype=F8)
    cache.set_prefix(pk, pv)
    ks, vs = normal(B, H_kv, 40, D), normal(B, H_kv, 40, D)
    cache.append(ks[:, :, :5], vs[:, :, :5])
    for t in range(5, 40):
        q = normal(B, H, 1, D)
        o = cache.step(q, ks[:, :, t:t + 1], vs[:, :, t:t + 1])
        _check(cache, q, pk, pv, ks[:, :, :t + 1], vs[:, :, :t + 1], tag=f"step {t}")
        x = cross_attention(o, ek, ev, lengths, enable_gqa=True)
        seen = (torch.arange(90, device=DEV) < lengths[:, None])[:, None, None]
        want, _, pabs, size = cache8.attention64(o, ek, ev, seen, D**-0.5)
        bound = cache8.output_bound(want, pabs, size, 90, dtype, 2 * 2.0**-8)
        assert ((x.double() - want).abs() <= bound).all(), t
        assert not x[3].any()
    positions, kr, _ = cache.read()
    assert positions.tolist() == cache8.held_positions(40, 2, cache.ring_size)
    stored = cache8.stored_values(ks[:, :, positions.tolist()].double().cpu().numpy())
    np.testing.assert_array_equal(kr.double().cpu().numpy(), stored)
