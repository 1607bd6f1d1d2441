"""Rolling StreamingLLM KV cache for the decode step.

The reference decodes from a full ``[B, H, N_KV, D]`` cache
(``sparse_triton_kernel.py:636-641``) although a StreamingLLM query only ever
sees the ``S`` sink tokens and the last ``W`` tokens (``README.md:41-67``): its
Θ((S+W)·D) claim holds for HBM reads but not for memory. ``StreamingKVCache``
keeps only what can still be seen, per (b, h):

* ``sink_size`` sink slots: position ``p < S`` lives in slot ``p``;
* a ring of ``R = W + max_query - 1`` slots: position ``p >= S`` lives in slot
  ``S + (p - S) mod R`` -- the ring holds the last ``R`` positions, which is what
  ``max_query`` decode rows at the end of the sequence can see.

``append`` writes new tokens (a whole prefill or one token per step) with
``gki_rolling_append``; ``attend`` runs the decode kernel over the compact cache
with ``gki_rolling_decode``. Its token stream, split rule and arithmetic are
those of the full-cache decode (``block_sparse_attention`` with the StreamingLLM
mask and ``is_causal=True``), so both give the same bits.

For c4's shape (B8 H32 D128 bf16, S4 W2048) the cache holds 2055 of 100000
positions: 2 x 135 MB instead of 2 x 6.55 GB.

``storage_dtype=torch.float8_e4m3fn`` holds each row in 8 bits: e4m3 codes and one
power of two (``k_scale`` / ``v_scale``), the smallest 2^e with the row's largest
magnitude at most 448 * 2^e. Rows are quantised as they are appended, attention runs
over the stored values (code * 2^e), and ``read`` gives back what either kind holds.

``set_prefix`` puts keys and values that all sequences of the batch share (a system
prompt, a document) in front of every sequence's own positions, held once: the decode
runs the queries of all sequences against each read of them.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib
from .masks import StreamingMaskSpec
from .ops import _DTYPE_CODE, _aligned, _current_stream, _decode_plan, _on_device

_DECODE_HEAD_DIMS = (64, 128)


def ring_slot(position: int, sink_size: int, ring_size: int) -> int:
    """Cache slot of an absolute position (host-side statement of the layout)."""
    if position < sink_size:
        return position
    return sink_size + (position - sink_size) % ring_size


def rolling_stream(length: int, n_q: int, sink_size: int, window_size: int,
                   ring_size: int) -> Tuple[int, int, int]:
    """``(n_sink, window_lo, n_tokens)`` of the visible-token stream of the last
    ``n_q`` of ``length`` positions, as computed by the library."""
    lib = _lib.load()
    a, b, c = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_int32()
    _lib.check(lib.gki_rolling_stream(int(length), int(n_q), int(sink_size), int(window_size),
                                      int(ring_size), ctypes.byref(a), ctypes.byref(b),
                                      ctypes.byref(c)), "gki_rolling_stream")
    return a.value, b.value, c.value


class StreamingKVCache:
    """Sink + ring KV cache on the GPU for StreamingLLM decoding.

    ``k_cache`` / ``v_cache``: ``[B, H, sink_size + ring_size, D]`` in ``dtype``,
    ``H`` = ``heads`` = the K/V heads. Queries may have any multiple of ``heads``
    (grouped-query attention: q head h reads kv head h // (Hq // heads)).
    ``length`` counts the positions appended so far (0 .. length-1).

    ``storage_dtype``: what the cache holds its rows in, ``dtype`` (the default) or
    ``torch.float8_e4m3fn``. In 8 bits ``k_cache`` / ``v_cache`` are the codes and
    ``k_scale`` / ``v_scale`` (``float8_e8m0fnu``, ``[B, H, sink_size + ring_size]``)
    the rows' powers of two; infinities and NaN are stored as NaN, and tokens, queries
    and outputs keep ``dtype``. No gradient flows through the cache. A NaN or infinity among
    the values reaches every query of the call that reads it, as in the sparse op.
    """

    def __init__(self, batch: int, heads: int, head_dim: int, spec: StreamingMaskSpec,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda",
                 max_query: int = 4, storage_dtype: Optional[torch.dtype] = None) -> None:
        if dtype not in _DTYPE_CODE:
            raise ValueError(f"dtype must be one of float32/float16/bfloat16, got {dtype}")
        if storage_dtype not in (None, dtype, torch.float8_e4m3fn):
            raise ValueError(f"storage_dtype must be {dtype} or torch.float8_e4m3fn, got {storage_dtype}")
        if head_dim not in _DECODE_HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {_DECODE_HEAD_DIMS}, got {head_dim}")
        max_q = _lib.tile_sizes()["decode_max_q"]
        if not 1 <= max_query <= max_q:
            raise ValueError(f"max_query must be in [1, {max_q}], got {max_query}")
        if batch <= 0 or heads <= 0:
            raise ValueError("batch and heads must be positive")
        self.spec = spec
        self.batch, self.heads, self.head_dim = int(batch), int(heads), int(head_dim)
        self.dtype = dtype
        self.max_query = int(max_query)
        self.sink_size = int(spec.sink_size)
        self.window_size = int(spec.window_size)
        self.ring_size = max(1, self.window_size + self.max_query - 1)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("StreamingKVCache lives on a CUDA (HIP) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        shape = (self.batch, self.heads, self.sink_size + self.ring_size, self.head_dim)
        self.storage_dtype = storage_dtype or dtype
        self.k_cache = torch.zeros(shape, dtype=self.storage_dtype, device=self.device)
        self.v_cache = torch.zeros(shape, dtype=self.storage_dtype, device=self.device)
        self.k_scale = self.v_scale = None
        if self.storage_dtype != dtype:
            self.k_scale, self.v_scale = (
                torch.zeros(shape[:3], dtype=torch.uint8, device=self.device).view(torch.float8_e8m0fnu)
                for _ in range(2))
        self.length = 0
        self._prefix: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
        self._plans: dict = {}           # (Hq, n_q, tokens, prefix) -> launch plan of _attend_streams

    @property
    def capacity(self) -> int:
        return self.sink_size + self.ring_size

    def reset(self) -> None:
        """Forget every sequence's positions (not the shared prefix)."""
        self.length = 0

    def set_prefix(self, k: Optional[torch.Tensor], v: Optional[torch.Tensor]) -> None:
        """Keys and values ``[1, H, P, D]`` in ``dtype`` (float16 or bfloat16) that every
        query of every sequence sees in full, whatever the window, beside its own
        positions; ``None, None`` (or ``P = 0``) removes them. Positions and ``length``
        count the sequences' own tokens only. Contiguous, 16-byte aligned tensors are
        kept, not copied: they must not change while the cache uses them."""
        if k is None and v is None:
            self._prefix = None
            return
        if k is None or v is None:
            raise ValueError("the prefix needs both keys and values")
        if self.dtype == torch.float32:
            raise ValueError("a shared prefix takes a float16 or bfloat16 cache")
        for name, t in (("k", k), ("v", v)):
            if t.dim() != 4 or t.shape[:2] != (1, self.heads) or t.shape[3] != self.head_dim:
                raise ValueError(f"prefix {name} must be [1, {self.heads}, P, {self.head_dim}], "
                                 f"got {tuple(t.shape)}")
            if t.dtype != self.dtype:
                raise ValueError(f"prefix {name} must be {self.dtype}, got {t.dtype}")
            if t.device != self.device:
                raise ValueError(f"prefix {name} must live on {self.device}")
        if k.shape != v.shape:
            raise ValueError("prefix k and v must share shape")
        self._prefix = (_aligned(k.detach()), _aligned(v.detach())) if k.shape[2] else None

    def _check_tokens(self, name: str, t: torch.Tensor, grouped: bool = False) -> int:
        """The tokens of ``t``, which must be ``[B, H, n, D]`` of the cache."""
        shape = t.shape                      # read once: a decode step's host time counts
        if len(shape) == 4:
            b, h, n, d = shape
            heads_ok = h == self.heads or (grouped and h > 0 and h % self.heads == 0)
        if len(shape) != 4 or b != self.batch or not heads_ok or d != self.head_dim:
            want = "a multiple of " + str(self.heads) if grouped else str(self.heads)
            raise ValueError(f"{name} must be [{self.batch}, {want}, n, {self.head_dim}], "
                             f"got {tuple(shape)}")
        if t.dtype != self.dtype:
            raise ValueError(f"{name} must be {self.dtype}, got {t.dtype}")
        if t.device != self.device:
            raise ValueError(f"{name} must live on {self.device}")
        return n

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """Append ``[B, H, n, D]`` keys / values at positions length .. length+n-1."""
        n = self._check_tokens("k", k)
        if n != self._check_tokens("v", v):
            raise ValueError("k and v must share shape")
        self._append(k, v, n)

    def _append(self, k: torch.Tensor, v: torch.Tensor, n: int) -> None:
        if n == 0:
            return
        k, v = _aligned(k), _aligned(v)
        lib = _lib.load()
        with _on_device(self.device):
            stream = _current_stream(self.device)
            if self.k_scale is None:
                _lib.check(lib.gki_rolling_append(
                    self.k_cache.data_ptr(), self.v_cache.data_ptr(), k.data_ptr(), v.data_ptr(),
                    _DTYPE_CODE[self.dtype], self.batch, self.heads, self.head_dim, self.sink_size,
                    self.ring_size, self.length, n, stream), "gki_rolling_append")
            else:
                _lib.check(lib.gki_rolling8_append(
                    self.k_cache.data_ptr(), self.v_cache.data_ptr(), self.k_scale.data_ptr(),
                    self.v_scale.data_ptr(), k.data_ptr(), v.data_ptr(), _DTYPE_CODE[self.dtype],
                    self.batch, self.heads, self.head_dim, self.sink_size, self.ring_size, self.length,
                    n, stream), "gki_rolling8_append")
        self.length += n

    def read(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """What the cache holds: ``(positions, k, v)``, the held positions ascending
        (``int64 [n]``: the sinks, then the last ``ring_size``) and their keys and
        values ``[B, H, n, D]`` in ``dtype`` -- from 8 bits the stored values, those
        past ``dtype``'s range as its infinities."""
        n = min(self.length, self.sink_size) + max(
            0, self.length - max(self.sink_size, self.length - self.ring_size))
        positions = torch.empty(n, dtype=torch.int64, device=self.device)
        shape = (self.batch, self.heads, n, self.head_dim)
        k, v = (torch.empty(shape, dtype=self.dtype, device=self.device) for _ in range(2))
        if n:
            lib = _lib.load()
            eight = self.k_scale is not None
            with _on_device(self.device):
                _lib.check(lib.gki_rolling_read(
                    self.k_cache.data_ptr(), self.v_cache.data_ptr(),
                    self.k_scale.data_ptr() if eight else 0, self.v_scale.data_ptr() if eight else 0,
                    k.data_ptr(), v.data_ptr(), positions.data_ptr(), _DTYPE_CODE[self.dtype],
                    self.batch, self.heads, self.head_dim, self.sink_size, self.ring_size, self.length,
                    _current_stream(self.device)), "gki_rolling_read")
        return positions, k, v

    def attend(self, q: torch.Tensor, softmax_scale: Optional[float] = None,
               return_lse: bool = False):
        """Decode attention of ``q`` (``[B, Hq, n_q, D]``, the last n_q positions
        of the cache; Hq a multiple of the cache's heads) over the shared prefix,
        if there is one, and the visible tokens: ``O`` (and the natural-log LSE ``[B, Hq, n_q]`` fp32 when
        ``return_lse``)."""
        return self._attend(q, self._check_queries(q, self.length), softmax_scale, return_lse)

    def _check_queries(self, q: torch.Tensor, length: int) -> int:
        """The rows of ``q``, which must be those of the last of ``length`` positions."""
        n_q = self._check_tokens("q", q, grouped=True)
        if not 1 <= n_q <= self.max_query:
            raise ValueError(f"q must hold 1..{self.max_query} rows, got {n_q}")
        if n_q > length:
            raise ValueError(f"q has {n_q} rows but the cache holds {length} positions")
        return n_q

    def _attend(self, q: torch.Tensor, n_q: int, softmax_scale: Optional[float], return_lse: bool):
        if softmax_scale is None:
            softmax_scale = 1.0 / math.sqrt(self.head_dim)
        q = _aligned(q)
        if self.k_scale is not None or self._prefix is not None:
            return self._attend_streams(q, n_q, float(softmax_scale), return_lse)
        _, _, n_tokens = rolling_stream(self.length, n_q, self.sink_size, self.window_size,
                                        self.ring_size)
        B, H, H_kv = self.batch, int(q.shape[1]), self.heads
        lib = _lib.load()
        dtype = _DTYPE_CODE[self.dtype]
        _, n_splits, ws_floats = _decode_plan(lib, dtype, B, H, H_kv, n_q, self.head_dim, n_tokens, True)
        o = torch.empty_like(q)
        # the LSE rows (padded to 256 bytes), then the split workspace: one allocation
        pad = (B * H * n_q + 63) & ~63
        scratch = torch.empty(pad + ws_floats, dtype=torch.float32, device=self.device)
        with _on_device(self.device):
            stream = _current_stream(self.device)
            _lib.check(lib.gki_rolling_decode(
                q.data_ptr(), self.k_cache.data_ptr(), self.v_cache.data_ptr(), o.data_ptr(),
                scratch.data_ptr(), dtype, B, H, H_kv, n_q, self.head_dim, self.sink_size,
                self.window_size, self.ring_size, self.length, float(softmax_scale),
                scratch.data_ptr() + 4 * pad if ws_floats else 0, n_splits, stream),
                "gki_rolling_decode")
        if not return_lse:
            return o
        return o, scratch[:B * H * n_q].view(B, H, n_q).clone()

    def _attend_streams(self, q: torch.Tensor, n_q: int, softmax_scale: float, return_lse: bool,
                        new: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
        """The decode over 8-bit rows, or behind a shared prefix. ``new``: the keys and
        values of the n_q tokens, which the same launch writes (``length`` is not moved)."""
        lib = _lib.load()
        B, H, H_kv, D = self.batch, int(q.shape[1]), self.heads, self.head_dim
        length = self.length + (n_q if new else 0)
        oldest = length - n_q - self.window_size + 1         # of the positions that some row's window holds
        n_tokens = length if oldest <= self.sink_size else self.sink_size + length - oldest
        prefix = self._prefix
        n_prefix = int(prefix[0].shape[2]) if prefix is not None else 0
        dtype = _DTYPE_CODE[self.dtype]
        key = (H, n_q, n_tokens, n_prefix)
        plan = self._plans.get(key)
        if plan is None:
            if len(self._plans) >= 4096:     # a filling window adds one key per step
                self._plans.clear()
            shared = 0
            if n_prefix:
                own = ctypes.c_int32()
                shared = int(lib.gki_prefix_splits(dtype, B, H, H_kv, n_q, D, n_prefix, n_tokens, ctypes.byref(own)))
                splits = own.value
            else:
                splits = int(lib.gki_stream_splits(dtype, B, H, H_kv, n_q, D, n_tokens))
            plan = self._plans[key] = (
                splits, shared, int(lib.gki_stream_workspace_floats(B, H, n_q, D, splits + shared)))
        n_splits, n_shared, ws_floats = plan
        o = torch.empty_like(q)
        # the LSE rows (padded to 256 bytes), then the slices' states: one allocation
        pad = (B * H * n_q + 63) & ~63
        scratch = torch.empty(pad + ws_floats, dtype=torch.float32, device=self.device)
        lse = scratch.data_ptr()
        rows = (self.k_cache.data_ptr(), self.v_cache.data_ptr())
        scales = (0, 0) if self.k_scale is None else (self.k_scale.data_ptr(), self.v_scale.data_ptr())
        shared = (prefix[0].data_ptr(), prefix[1].data_ptr(), n_prefix) if n_prefix else (0, 0, 0)
        place = (dtype, B, H, H_kv, n_q, D, self.sink_size, self.window_size, self.ring_size)
        ws = lse + 4 * pad if ws_floats else 0
        with _on_device(self.device):
            stream = _current_stream(self.device)
            if new:
                what = "gki_rolling_step"
                rc = lib.gki_rolling_step(q.data_ptr(), new[0].data_ptr(), new[1].data_ptr(), *rows, *scales, *shared,
                                          o.data_ptr(), lse, *place, self.length, softmax_scale, ws, n_shared,
                                          n_splits, stream)
            elif n_prefix:
                what = "gki_rolling_prefix_decode"
                rc = lib.gki_rolling_prefix_decode(q.data_ptr(), *rows, *scales, *shared, o.data_ptr(), lse, *place,
                                                   length, softmax_scale, ws, n_shared, n_splits, stream)
            else:
                what = "gki_rolling8_decode"
                rc = lib.gki_rolling8_decode(q.data_ptr(), *rows, *scales, o.data_ptr(), lse, *place, length,
                                             softmax_scale, ws, n_splits, stream)
        if rc:
            _lib.check(rc, what)
        if not return_lse:
            return o
        return o, scratch[:B * H * n_q].view(B, H, n_q).clone()

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
             softmax_scale: Optional[float] = None) -> torch.Tensor:
        """One decode step: append the new tokens' K / V, then attend with q. Arguments
        are checked before anything is written."""
        n_k = self._check_tokens("k", k)
        if n_k != self._check_tokens("v", v):
            raise ValueError("k and v must share shape")
        n = self._check_queries(q, self.length + n_k)
        if softmax_scale is not None and not math.isfinite(softmax_scale):
            raise ValueError(f"softmax_scale must be finite, got {softmax_scale}")
        if n == n_k and (self.k_scale is not None or self._prefix is not None):
            # the tokens are written by the launch that attends them
            scale = 1.0 / math.sqrt(self.head_dim) if softmax_scale is None else float(softmax_scale)
            o = self._attend_streams(_aligned(q), n, scale, False, (_aligned(k), _aligned(v)))
            self.length += n
            return o
        self._append(k, v, n_k)
        return self._attend(q, n, softmax_scale, False)
