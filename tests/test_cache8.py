"""The rolling cache held in 8 bits: codes and scales as they are written, what is
read back, and the decode over the stored values.

CPU: the oracle's rounding against torch's cast, and refusals. GPU: codes and scales
bit for bit, the read rows bit for bit, outputs within the bound that
``oracle.cache8.output_bound`` derives (bf16 queries: weights rounded to 2^-8, fp16 and
fp32: to two and three bfloat16 pieces, 2^-16 and 2^-24).
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from gki import StreamingKVCache, StreamingMaskSpec, _lib
from gki.kv_cache import ring_slot
from oracle import cache8
from oracle import streaming_oracle as so

DEV = "cuda"
F8 = torch.float8_e4m3fn
P_EPS = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-16, torch.float32: 2.0**-24}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


# ---- CPU -------------------------------------------------------------------------


def test_oracle_rounds_as_the_cast_does():
    y = torch.cat([torch.linspace(-448, 448, 100001), torch.randn(50000) * 2.0 ** torch.randint(-12, 8, (50000,)),
                   torch.arange(0, 449, 0.5), torch.arange(-40, 40) * 2.0**-11]).clamp(-448, 448)
    want = y.to(F8).double().numpy()
    np.testing.assert_array_equal(cache8.e4m3_round(y.double().numpy()), want)


def test_oracle_exponent_is_the_smallest():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((500, 16)) * np.ldexp(1.0, rng.integers(-60, 60, (500, 1)))
    x[0], x[1, 1:], x[1, 0], x[2, 0] = 0, 0, 448 * 2.0**-3, np.inf
    codes, e = cache8.quantise(x)
    top = np.where(np.isfinite(x), np.abs(x), 0).max(-1)
    assert (top <= 448 * np.ldexp(1.0, e)).all()
    assert ((top > 448 * np.ldexp(1.0, e - 1)) | (e == cache8.MIN_EXPONENT)).all()
    assert e[0] == cache8.MIN_EXPONENT and e[1] == -3 and np.isnan(codes[2, 0])


def test_c_entries_refuse_before_launch():
    lib, null = _lib.load(), ctypes.c_void_p(0)

    def append(ptrs=(16,) * 6, dtype=2, B=1, H=1, D=64, sink=4, ring=8, start=0, n=1):
        return lib.gki_rolling8_append(*ptrs, dtype, B, H, D, sink, ring, start, n, null)

    def decode(q=16, o=16, scale=16, ws=0, dtype=2, H=2, H_kv=1, n_q=1, D=64, ring=8, length=5, s=0.1, splits=1):
        return lib.gki_rolling8_decode(q, 16, 16, scale, 16, o, 16, dtype, 1, H, H_kv, n_q, D, 0, 8, ring, length, s,
                                       ws, splits, null)

    assert append(dtype=5) == 2 and append(D=32) == 2 and append(B=0) == 1 and append(ring=0) == 1
    assert append(start=-1) == 1 and append(start=2**30) == 1 and append(ptrs=(0,) * 6) == 1
    assert append(ptrs=(16, 24, 16, 16, 16, 16)) == 1 and b"aligned" in lib.gki_last_error()
    assert append(ptrs=(0,) * 6, n=0) == 0                       # nothing to write
    assert decode(D=32) == 2 and decode(n_q=5) == 2 and decode(H=3, H_kv=2) == 1 and decode(ring=3) == 1
    assert decode(s=math.inf) == 1 and decode(scale=0) == 1 and decode(splits=2) == 1 and decode(splits=0) == 1
    assert decode(o=24) == 1 and decode(ws=24, splits=2) == 1 and decode(length=0) == 1

    def step(k_new=16, k_scale=16, n_prefix=0, start=5, ws=0, splits=1, dtype=2):
        return lib.gki_rolling_step(16, k_new, 16, 16, 16, k_scale, k_scale, 0, 0, n_prefix, 16, 16, dtype, 1, 2, 1, 1, 64,
                                    0, 8, 8, start, 0.1, ws, 0, splits, null)

    assert step(k_new=0) == 1 and step(k_new=8) == 1 and step(k_scale=0) == 2 and step(start=-1) == 1
    assert step(start=2**30) == 1 and step(splits=2) == 1 and step(n_prefix=3) == 1 and step(dtype=8) == 2
    assert step(n_prefix=-1) == 1
    read = (16, 16, 16, 16, 16, 16, 16)
    assert lib.gki_rolling_read(*read, 2, 1, 1, 64, 4, 8, -1, null) == 1
    assert lib.gki_rolling_read(16, 16, 16, 0, 16, 16, 16, 2, 1, 1, 64, 4, 8, 3, null) == 1    # one scale
    assert lib.gki_rolling_read(*(0,) * 7, 2, 1, 1, 64, 4, 8, 0, null) == 0
    assert lib.gki_stream_workspace_floats(2, 4, 1, 64, 1) == 0
    assert lib.gki_stream_workspace_floats(2, 4, 3, 64, 5) == 2 * 4 * 3 * 5 * 66
    for tokens in (0, 1, 127, 128, 100000):
        assert 1 <= lib.gki_stream_splits(2, 1, 8, 8, 1, 128, tokens) <= max(1, tokens // 128)


def test_python_refusals():
    spec = StreamingMaskSpec(4, 16)
    with pytest.raises(ValueError, match="storage_dtype"):
        StreamingKVCache(1, 1, 64, spec, storage_dtype=torch.float8_e5m2)
    with pytest.raises(ValueError, match="storage_dtype"):
        StreamingKVCache(1, 1, 64, spec, dtype=torch.bfloat16, storage_dtype=torch.float16)


# ---- GPU -------------------------------------------------------------------------


def _rows(shape, dtype, seed, special=False):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.exp2(torch.randint(-3, 4, shape[:-1], generator=gen).float())[..., None]
    if special:
        flat = x.view(-1, shape[-1])
        n = flat.shape[0]
        flat[0 % n] = 0
        flat[1 % n, 0] = 448.0                                   # the border of an exponent
        flat[2 % n, 1:] = 0
        flat[2 % n, 0] = 449.0 if dtype == torch.float32 else 450.0
        flat[3 % n, 3], flat[3 % n, 5] = math.inf, math.nan
        flat[4 % n] = -math.inf
        flat[5 % n] *= 1e-6 if dtype == torch.float16 else 1e-38
        flat[6 % n, 7] = 60000.0 if dtype == torch.float16 else 3e38
        flat[7 % n] = torch.arange(shape[-1]).float() * 2.0**-9
        flat[8 % n, :9] = torch.tensor([448, 2.0**-9, 2.0**-10, 3 * 2.0**-10, -(2.0**-10), 2.0**-6, 17, 18, 19.0])
    return x.to(dtype)


def _same(got, want):
    got, want = got.detach().double().cpu().numpy(), np.asarray(want, dtype=np.float64)
    np.testing.assert_array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("sink,window,max_q,chunks", [(4, 16, 4, (9, 1, 40, 3)), (0, 1, 1, (1, 1, 5)),
                                                      (3, 0, 1, (7,)), (5, 33, 2, (2, 1, 1, 100, 1))])
def test_written_and_read_rows_are_exact(dtype, head_dim, sink, window, max_q, chunks):
    B, H = 2, 3
    cache = StreamingKVCache(B, H, head_dim, StreamingMaskSpec(sink, window), dtype, DEV, max_q, storage_dtype=F8)
    plain = StreamingKVCache(B, H, head_dim, StreamingMaskSpec(sink, window), dtype, DEV, max_q)
    assert [t.numel() for t in cache.read()] == [0, 0, 0]
    k = _rows((B, H, sum(chunks), head_dim), dtype, 1, special=True)
    v = _rows((B, H, sum(chunks), head_dim), dtype, 2, special=True)
    at = 0
    for n in chunks:
        for c in (cache, plain):
            c.append(k[:, :, at:at + n].to(DEV), v[:, :, at:at + n].to(DEV))
        at += n
        held = cache8.held_positions(at, sink, cache.ring_size)
        slots = [ring_slot(p, sink, cache.ring_size) for p in held]
        for name, x in (("k", k), ("v", v)):
            codes, e = cache8.quantise(x[:, :, held].double().numpy())
            _same(getattr(cache, name + "_cache")[:, :, slots], codes)
            _same(getattr(cache, name + "_scale")[:, :, slots], np.ldexp(1.0, e))
        positions, kr, vr = cache.read()
        assert positions.tolist() == held and kr.dtype == dtype
        for got, x in ((kr, k), (vr, v)):
            want = torch.from_numpy(cache8.stored_values(x[:, :, held].double().numpy())).to(dtype)
            _same(got, want.double().numpy())
        positions, kr, vr = plain.read()
        assert positions.tolist() == held
        _same(kr, k[:, :, held].double().numpy())
        _same(vr, v[:, :, held].double().numpy())


def _check_attend(cache, q, k, v, scale=None, tag=""):
    """One attend of the cache (holding k, v [B, H_kv, length, D]) against 64 bits."""
    dtype, n_q, length = q.dtype, q.shape[2], k.shape[2]
    o, lse = cache.attend(q, scale, return_lse=True)
    scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    vis = torch.from_numpy(so.token_mask(n_q, length, cache.sink_size, cache.window_size)).to(DEV)
    kv = [torch.from_numpy(cache8.stored_values(t.double().cpu().numpy())).to(DEV) for t in (k, v)]
    want, want_lse, pv, size = cache8.attention64(q, *kv, vis, scale)
    bound = cache8.output_bound(want, pv, size, int(vis.sum(-1).max()), dtype, P_EPS[dtype])
    err = (o.double() - want).abs()
    assert torch.isfinite(o).all(), tag
    assert (err <= bound).all(), (tag, (err / bound).max().item())
    # the LSE: the scores' error, and 2^-24 of itself and of each of the row sum's terms
    lse_bound = 136 * 2.0**-24 * size + (int(vis.sum(-1).max()) + 16) * 2.0**-24 + 2.0**-23 * want_lse.abs()
    assert ((lse.double() - want_lse).abs() <= lse_bound).all(), tag
    empty = ~vis.any(-1)
    assert not o[:, :, empty].any() and not lse[:, :, empty].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,n_q,sink,window,length", [
    (2, 2, 1, 4, 100, 1), (2, 2, 1, 4, 100, 63), (3, 3, 1, 4, 100, 64), (2, 2, 1, 0, 64, 300), (2, 1, 1, 1, 65, 500),
    (8, 2, 2, 4, 200, 777), (8, 1, 4, 4, 257, 1000), (12, 3, 3, 0, 1000, 1001), (32, 1, 4, 16, 300, 900),
    (5, 1, 4, 2, 3, 50), (2, 2, 4, 0, 1, 9), (2, 2, 4, 3, 0, 9), (2, 2, 2, 0, 0, 7), (2, 2, 4, 4, 100, 4),
    (17, 1, 1, 4, 2048, 3000), (4, 4, 1, 4, 5000, 5200),
])
def test_decode_against_64_bits(dtype, head_dim, heads, kv_heads, n_q, sink, window, length):
    B = 2
    gen = torch.Generator(device=DEV).manual_seed(heads * 1000 + length)
    k, v = (torch.randn((B, kv_heads, length, head_dim), generator=gen, device=DEV).to(dtype) for _ in range(2))
    k[..., 1] *= 6
    q = (torch.randn((B, heads, n_q, head_dim), generator=gen, device=DEV) * 0.7).to(dtype)
    cache = StreamingKVCache(B, kv_heads, head_dim, StreamingMaskSpec(sink, window), dtype, DEV, n_q, storage_dtype=F8)
    cut = max(0, length - 5)
    cache.append(k[:, :, :cut], v[:, :, :cut])
    cache.append(k[:, :, cut:], v[:, :, cut:])
    _check_attend(cache, q, k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 1e-6])
def test_any_finite_scale(dtype, scale):
    gen = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn((2, 2, 300, 64), generator=gen, device=DEV).to(dtype) for _ in range(2))
    q = torch.randn((2, 6, 2, 64), generator=gen, device=DEV).to(dtype)
    cache = StreamingKVCache(2, 2, 64, StreamingMaskSpec(4, 200), dtype, DEV, storage_dtype=F8)
    cache.append(k, v)
    _check_attend(cache, q, k, v, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 2, 3, 7, 40])
def test_any_number_of_slices(splits, monkeypatch):
    """More slices than tokens leave some empty."""
    lib = _lib.load()
    monkeypatch.setattr(lib, "gki_stream_splits", lambda *a: splits)
    gen = torch.Generator(device=DEV).manual_seed(4)
    for length in (1, 30, 700):
        k, v = (torch.randn((1, 2, length, 128), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
        q = torch.randn((1, 4, 1, 128), generator=gen, device=DEV).to(torch.bfloat16)
        cache = StreamingKVCache(1, 2, 128, StreamingMaskSpec(4, 600), torch.bfloat16, DEV, storage_dtype=F8)
        cache.append(k, v)
        _check_attend(cache, q, k, v)


@pytest.mark.gpu
def test_steps_over_a_turning_ring_and_large_logits():
    dtype, B, H, D = torch.bfloat16, 2, 2, 128
    gen = torch.Generator(device=DEV).manual_seed(5)
    ks, vs = (torch.randn((B, H, 200, D), generator=gen, device=DEV).to(dtype) * 3 for _ in range(2))
    cache = StreamingKVCache(B, H, D, StreamingMaskSpec(2, 50), dtype, DEV, max_query=2, storage_dtype=F8)
    for at in range(0, 160, 2):
        q = torch.randn((B, 4, 2, D), generator=gen, device=DEV).to(dtype) * 3
        k, v = ks[:, :, at:at + 2], vs[:, :, at:at + 2]
        got = cache.step(q, k, v)
        assert torch.equal(got, cache.attend(q))
        _check_attend(cache, q, ks[:, :, :at + 2], vs[:, :, :at + 2], tag=f"length {at + 2}")
    cache.reset()
    cache.append(ks[:, :, :3], vs[:, :, :3])
    _check_attend(cache, torch.randn((B, 2, 1, D), device=DEV).to(dtype), ks[:, :, :3], vs[:, :, :3])


def _twins(dtype, head_dim, sink, window, max_q, B, H_kv, storage, prefix=0, seed=8):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    caches = [StreamingKVCache(B, H_kv, head_dim, StreamingMaskSpec(sink, window), dtype, DEV, max_q, storage_dtype=storage)
              for _ in range(2)]
    if prefix:
        pk, pv = (torch.randn((1, H_kv, prefix, head_dim), generator=gen, device=DEV).to(dtype) for _ in range(2))
        for c in caches:
            c.set_prefix(pk, pv)
    return caches, gen


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,storage,prefix", [(torch.bfloat16, F8, 0), (torch.float16, F8, 0), (torch.float32, F8, 0),
                                                  (torch.bfloat16, F8, 70), (torch.float16, None, 70)])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("sink,window,max_q,n_q,heads", [(4, 20, 4, 1, 2), (2, 70, 3, 3, 4), (0, 1, 1, 1, 2), (5, 0, 2, 2, 2),
                                                         (3, 130, 4, 4, 32), (0, 0, 4, 3, 2), (1, 1, 2, 2, 40)])
def test_a_step_is_the_append_and_the_attend(dtype, storage, prefix, head_dim, sink, window, max_q, n_q, heads):
    """Same outputs and same cache, byte for byte, at every length across the sinks, the
    filling of the ring and its turn."""
    B, H_kv = 2, 2
    (one, two), gen = _twins(dtype, head_dim, sink, window, max_q, B, H_kv, storage, prefix)
    for t in range(0, 2 * (sink + window) + 9, n_q):
        k, v = (torch.randn((B, H_kv, n_q, head_dim), generator=gen, device=DEV).to(dtype) for _ in range(2))
        q = torch.randn((B, heads, n_q, head_dim), generator=gen, device=DEV).to(dtype)
        got = one.step(q, k, v)
        two.append(k, v)
        assert torch.equal(got, two.attend(q)), t
        assert one.length == two.length
    for name in ("k_cache", "v_cache") + (("k_scale", "v_scale") if storage else ()):
        a, b = (getattr(c, name).view(torch.uint8) for c in (one, two))
        assert torch.equal(a, b), name


@pytest.mark.gpu
def test_a_step_of_unlike_counts_and_a_refused_one():
    (one, two), gen = _twins(torch.bfloat16, 64, 4, 30, 4, 1, 2, F8)
    k, v = (torch.randn((1, 2, 9, 64), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((1, 2, 2, 64), generator=gen, device=DEV).to(torch.bfloat16)
    got = one.step(q, k, v)                                      # nine tokens, two queries
    two.append(k, v)
    assert torch.equal(got, two.attend(q))
    with pytest.raises(ValueError, match="share shape|must be"):
        one.step(q, k[:, :, :2], v[:, :1, :2])
    with pytest.raises(ValueError, match="multiple of 2"):
        one.step(q[:, :1], k[:, :, :2], v[:, :, :2])
    assert one.length == 9                                       # a refused step writes nothing
    assert torch.equal(one.attend(q), got)


@pytest.mark.gpu
def test_unseen_slots_do_not_matter():
    """What left the window, or was never written, may hold anything."""
    dtype = torch.float16
    gen = torch.Generator(device=DEV).manual_seed(6)
    k, v = (torch.randn((1, 2, 90, 64), generator=gen, device=DEV).to(dtype) for _ in range(2))
    q = torch.randn((1, 2, 1, 64), generator=gen, device=DEV).to(dtype)
    cache = StreamingKVCache(1, 2, 64, StreamingMaskSpec(4, 64), dtype, DEV, max_query=4, storage_dtype=F8)
    cache.append(k[:, :, :90], v[:, :, :90])
    want = cache.attend(q)
    seen = {ring_slot(p, 4, cache.ring_size) for p in range(90) if p < 4 or p >= 90 - 64}
    unseen = [s for s in range(cache.capacity) if s not in seen]
    assert unseen
    for t in (cache.k_cache, cache.v_cache):
        t.view(torch.uint8)[:, :, unseen] = 0x7F                # NaN
    assert torch.equal(cache.attend(q), want)


@pytest.mark.gpu
def test_slots_past_2_31_elements():
    B, H, D, window = 34, 8, 128, 65536               # 2.3e9 elements of K and of V
    gen = torch.Generator(device=DEV).manual_seed(8)
    k, v = (torch.randn((B, H, 70, D), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((B, H, 1, D), generator=gen, device=DEV).to(torch.bfloat16)
    cache = StreamingKVCache(B, H, D, StreamingMaskSpec(4, window), torch.bfloat16, DEV, storage_dtype=F8)
    assert cache.k_cache.numel() > 2**31
    cache.append(k, v)
    _check_attend(cache, q, k, v)
    _, kr, vr = cache.read()
    for x, got in ((k, kr), (v, vr)):
        _same(got, cache8.stored_values(x.double().cpu().numpy()))


@pytest.mark.gpu
def test_strided_tokens_side_stream_and_graph():
    dtype, B, H, D = torch.bfloat16, 2, 4, 64
    gen = torch.Generator(device=DEV).manual_seed(7)
    base = torch.randn((B, 50, 3, H, D), generator=gen, device=DEV).to(dtype)
    k, v = base[:, :, 0].transpose(1, 2), base[:, :, 1].transpose(1, 2)
    q = base[:, :1, 2].transpose(1, 2)
    cache = StreamingKVCache(B, H, D, StreamingMaskSpec(4, 30), dtype, DEV, storage_dtype=F8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(k, v)
        got = cache.attend(q)
    torch.cuda.current_stream().wait_stream(side)
    _check_attend(cache, q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(got, cache.attend(q))
    qs = q.contiguous().clone()
    graph = torch.cuda.CUDAGraph()
    cache.attend(qs)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = cache.attend(qs)
    for i in range(3):
        qs.copy_(torch.randn(qs.shape, generator=gen, device=DEV).to(dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cache.attend(qs)), i


@pytest.mark.gpu
def test_gpu_refusals():
    cache = StreamingKVCache(1, 2, 64, StreamingMaskSpec(4, 30), torch.bfloat16, DEV, storage_dtype=F8)
    k = torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="must be torch.bfloat16"):
        cache.append(k.half(), k.half())
    with pytest.raises(ValueError, match="share shape"):
        cache.append(k, k[:, :, :2])
    with pytest.raises(ValueError, match="positions"):
        cache.attend(k[:, :, :1])                                # nothing held yet
    cache.append(k, k)
    with pytest.raises(ValueError, match="multiple of 2"):
        cache.attend(torch.zeros((1, 3, 1, 64), dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="rows"):
        cache.attend(torch.zeros((1, 2, 5, 64), dtype=torch.bfloat16, device=DEV))
