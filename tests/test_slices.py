"""Slices of streams: the launch rules that choose their number, and steps whose own
tokens the launch that attends them writes, at several slices.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from gki import StreamingKVCache, StreamingMaskSpec, _lib

DEV = "cuda"
F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("B,H,H_kv,n_q,n_kv,D", [
    (1, 8, 8, 64, 8192, 128), (1, 8, 8, 64, 8192, 64), (1, 8, 8, 200, 8000, 128), (8, 32, 8, 16, 8192, 64),
    (2, 8, 1, 37, 3000, 128), (1, 4, 4, 17, 5000, 32), (4, 8, 2, 4, 6000, 128),
])
def test_both_16_bit_types_take_the_same_slices(B, H, H_kv, n_q, n_kv, D):
    """They run the same row tiles: 32 rows a workgroup for more than 16."""
    lib = _lib.load()
    bf16, fp16 = (lib.gki_cross_splits(dtype, B, H, H_kv, n_q, n_kv, D) for dtype in (2, 1))
    assert bf16 >= 1 and fp16 == bf16


@pytest.mark.parametrize("B,H,H_kv,n_q,n_tokens,D", [(2, 64, 2, 4, 3000, 128), (1, 32, 1, 2, 9000, 64), (4, 20, 1, 1, 5000, 128),
                                                     (3, 12, 12, 2, 700, 64), (16, 64, 2, 2, 8192, 128)])
def test_both_types_take_the_same_slices_behind_a_prefix(B, H, H_kv, n_q, n_tokens, D):
    lib, own = _lib.load(), ctypes.c_int32()

    def splits(dtype):
        return lib.gki_prefix_splits(dtype, B, H, H_kv, n_q, D, 4000, n_tokens, ctypes.byref(own)), own.value

    assert splits(1) == splits(2)


def _twins(dtype, storage, prefix, head_dim, sink, window, max_q, H_kv, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV).to(dtype)

    caches = [StreamingKVCache(2, H_kv, head_dim, StreamingMaskSpec(sink, window), dtype, DEV, max_q, storage_dtype=storage)
              for _ in range(2)]
    if prefix:
        pk, pv = normal(1, H_kv, prefix, head_dim), normal(1, H_kv, prefix, head_dim)
        for c in caches:
            c.set_prefix(pk, pv)
    return caches, normal


def _same_steps(caches, normal, heads, first, count, n_q):
    """After a prompt of `first` tokens, `count` steps of n_q: the same outputs and the same
    cache, byte for byte, from step as from append and attend."""
    one, two = caches
    B, H_kv, D = one.batch, one.heads, one.head_dim
    k, v = normal(B, H_kv, first, D), normal(B, H_kv, first, D)
    for c in caches:
        c.append(k, v)
    for t in range(count):
        q, k, v = normal(B, heads, n_q, D), normal(B, H_kv, n_q, D), normal(B, H_kv, n_q, D)
        got = one.step(q, k, v)
        two.append(k, v)
        assert torch.isfinite(got).all() and torch.equal(got, two.attend(q)), (t, one.length)
    assert one.length == two.length
    for name in ("k_cache", "v_cache") + (("k_scale", "v_scale") if one.k_scale is not None else ()):
        a, b = (getattr(c, name).view(torch.uint8) for c in caches)
        assert torch.equal(a, b), name


KINDS = [(torch.bfloat16, F8, 0), (torch.float16, F8, 0), (torch.float32, F8, 0), (torch.bfloat16, F8, 300),
         (torch.float16, None, 300), (torch.bfloat16, None, 300)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,storage,prefix", KINDS)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("splits", [2, 5, 40])
@pytest.mark.parametrize("n_q,heads", [(1, 2), (4, 6)])
def test_steps_at_any_number_of_slices(dtype, storage, prefix, head_dim, splits, n_q, heads, monkeypatch):
    """Slices that start and end between the step's own tokens, or where the ring turns."""
    lib = _lib.load()

    def both(*a):
        a[-1]._obj.value = splits
        return 3

    monkeypatch.setattr(lib, "gki_stream_splits", lambda *a: splits)
    monkeypatch.setattr(lib, "gki_prefix_splits", both)
    caches, normal = _twins(dtype, storage, prefix, head_dim, 3, 150, 4, 2, seed=splits)
    _same_steps(caches, normal, heads, 100, 240 // n_q, n_q)      # the sinks, a filling ring and its turn
    assert caches[0].length > 2 * caches[0].ring_size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,storage,prefix", KINDS)
@pytest.mark.parametrize("n_q", [1, 3])
def test_steps_of_a_long_window_while_its_ring_turns(dtype, storage, prefix, n_q):
    caches, normal = _twins(dtype, storage, prefix, 128, 4, 2048, 4, 2, seed=9)
    ring = caches[0].ring_size
    _same_steps(caches, normal, 4, 4 + ring - 20, 60 // n_q, n_q)
    plan = list(caches[0]._plans.values())
    assert all(p[0] > 1 for p in plan)                            # several slices, unforced


@pytest.mark.gpu
@pytest.mark.parametrize("storage,prefix", [(None, 0), (F8, 0), (None, 70), (F8, 70)])
def test_a_refused_step_writes_nothing(storage, prefix):
    (cache, _), normal = _twins(torch.bfloat16, storage, prefix, 64, 4, 30, 2, 2, seed=1)
    k, v = normal(2, 2, 3, 64), normal(2, 2, 3, 64)
    cache.append(k, v)
    held = [t.view(torch.uint8).clone() for t in (cache.k_cache, cache.v_cache)]
    q = normal(2, 4, 3, 64)
    for args, match in (((q, k, v), "rows"),                              # more queries than max_query
                        ((q[:, :, :0], k, v), "rows"), ((q[:, :3, :1], k, v), "multiple of 2"),
                        ((q[..., :32], k, v), "must be"), ((q.half()[:, :, :1], k[:, :, :1], v[:, :, :1]), "bfloat16"),
                        ((q[:, :, :1], k, v[:, :, :1]), "share shape"), ((q[:, :, :1].cpu(), k, v), "live on"),
                        ((q[:, :, :1], k, v, float("inf")), "finite"), ((q[:, :, :1], k[:, :, :1], v[:, :, :1], float("nan")), "finite")):
        with pytest.raises(ValueError, match=match):
            cache.step(*args)
        assert cache.length == 3
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(held, (cache.k_cache, cache.v_cache)))
    cache.reset()
    with pytest.raises(ValueError, match="positions"):
        cache.step(q[:, :, :2], k[:, :, :1], v[:, :, :1])
    assert cache.length == 0
