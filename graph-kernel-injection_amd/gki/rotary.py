"""Rotary positions with several axes (text; height and width; time, height and width).

Queries and keys are turned by their positions before they attend: the sparse op, cross
attention and the caches take them as they come out of here. ``PagedKVCache`` turns keys
as it writes them (``append_rotated``).

A row's first ``2 P`` elements are ``P`` pairs; pair ``j`` belongs to one axis and turns by
``positions[axis] * frequency_j``: ``(a, b) -> (a cos - b sin, a sin + b cos)``. The gradient
turns back. Queries and keys take one launch (``gki_rotary``) in either direction.

There is no CPU or eager fallback: a missing library raises ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import _DTYPE_CODE, _HEAD_DIMS, _current_stream, _on_device, _refuse_tangents

_Strides3, _Strides6 = ctypes.c_int64 * 3, ctypes.c_int64 * 6


def _in_place(t: torch.Tensor) -> bool:
    """Whether rows lie in one piece on 16-byte boundaries."""
    per16 = 16 // t.element_size()
    return t.data_ptr() % 16 == 0 and t.stride(-1) == 1 and all(s % per16 == 0 for s in t.stride()[:-1])


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    """A new contiguous tensor of ``t``'s shape (1.2 us of host time; ``torch.empty`` of the shape takes 2.3)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _copied(t: torch.Tensor) -> torch.Tensor:
    return t.clone(memory_format=torch.contiguous_format)


def _strides(src: torch.Tensor, dst: torch.Tensor):
    """(batch, token, head) strides of both; packed rows are one batch entry."""
    out = []
    for t in (src, dst):
        s = t.stride()
        out += [s[0], s[2], s[1]] if t.dim() == 4 else [0, s[0], s[1]]
    return _Strides6(*out)


class _Rotate(torch.autograd.Function):
    """Both tensors turned, or turned back; linear, so its own gradient of any order."""

    @staticmethod
    def forward(ctx, rope, q, k, positions, strides, inverse):  # type: ignore[override]
        ctx.rope, ctx.strides, ctx.inverse = rope, strides, inverse
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        outs = rope._rotate(q, k, positions, strides, inverse)
        # a frozen tensor comes out frozen: what attends it computes no gradient for it
        frozen = [o for o, needed in zip(outs, ctx.needs_input_grad[1:3]) if o is not None and not needed]
        if frozen:
            ctx.mark_non_differentiable(*frozen)
        return outs

    @staticmethod
    def backward(ctx, dq, dk):  # type: ignore[override]
        dq = dq if ctx.needs_input_grad[1] else None
        dk = dk if ctx.needs_input_grad[2] else None
        if dq is not None or dk is not None:
            dq, dk = ctx.rope._apply(dq, dk, ctx.saved_tensors[0], ctx.strides, not ctx.inverse)
        return None, dq, dk, None, None, None


class MultiAxisRotary:
    """Rotary positions of ``sections``: how many pairs of elements belong to each axis, in
    order (text: one section of ``head_dim / 2``). They sum to a multiple of 8 pairs, at most
    ``head_dim / 2``; elements behind the pairs stay as they are.

    Pair ``j`` of all ``P`` turns with frequency ``base ** (-j / P)``; with ``per_axis`` each
    axis has a ladder of its own, ``base ** (-i / size)`` for the ``i``-th pair of a section of
    that size. Pairs are elements ``(j, j + P)`` or, ``interleaved``, ``(2 j, 2 j + 1)``. Angles
    are made and reduced in 64 bits: off by less than 2^-21 of a radian for positions below 2^30
    and frequencies up to 1 (a ``base`` of at least 1), in proportion more beyond either.
    """

    def __init__(self, head_dim: int, sections: Sequence[int], base: float = 10000.0, interleaved: bool = False,
                 per_axis: bool = False) -> None:
        if head_dim not in _HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
        self.sections = tuple(int(s) for s in sections)
        pairs = sum(self.sections)
        if not self.sections or min(self.sections) <= 0 or pairs % 8 or 2 * pairs > head_dim:
            raise ValueError(f"sections must be positive and sum to a multiple of 8, at most {head_dim // 2}, "
                             f"got {self.sections}")
        if not (math.isfinite(base) and base > 0):
            raise ValueError(f"base must be positive and finite, got {base}")
        self.head_dim, self.base = int(head_dim), float(base)
        self.interleaved, self.per_axis = bool(interleaved), bool(per_axis)
        self.pairs = pairs
        self._known: dict = {}               # shapes, strides, ... of checked calls -> the positions' strides
        self._launches: dict = {}            # of the tensors of a launch -> its sizes and strides
        self._tables: dict = {}              # device -> (turns per position, axis) of the pairs

    def _table(self, device: torch.device) -> Tuple[torch.Tensor, torch.Tensor]:
        table = self._tables.get(device)
        if table is None:
            turns, axis, j = [], [], 0
            for a, size in enumerate(self.sections):
                for i in range(size):
                    ladder = i / size if self.per_axis else j / self.pairs
                    turns.append(self.base ** -ladder / (2 * math.pi))
                    axis.append(a)
                    j += 1
            table = self._tables[device] = (torch.tensor(turns, dtype=torch.float64, device=device),
                                            torch.tensor(axis, dtype=torch.int32, device=device))
        return table

    def _position_strides(self, positions: torch.Tensor, q: torch.Tensor):
        """(axis, batch, token) strides; raises for positions that do not fit ``q``."""
        shape, axes, packed = tuple(positions.shape), len(self.sections), q.dim() == 3
        batch, n = (1, q.shape[0]) if packed else (q.shape[0], q.shape[2])
        dim = len(shape)
        if not 1 <= dim <= (2 if packed else 3) or shape[-1] != n or (dim == 3 and shape[1] != batch) or (
                dim > 1 and shape[0] not in (1, axes)):
            want = f"[{axes}, {n}]" if packed else f"[{axes}, {batch}, {n}], [{axes}, {n}]"
            raise ValueError(f"positions must be {want} (or 1 for the axes) or [{n}], got {shape}")
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.device != q.device:
            raise ValueError(f"positions must live on {q.device}")
        s = positions.stride()
        return s[0] if dim > 1 and shape[0] > 1 else 0, s[1] if dim == 3 else 0, s[-1]

    def __call__(self, q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor
                 ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """``q`` and ``k`` (or ``None``) turned: ``[B, H, N, D]``, or packed rows
        ``[rows, H, D]``, each with its own heads; fp32/fp16/bf16. ``positions``: int32 or
        int64, ``[axes, B, N]`` or ``[axes, N]`` (packed: ``[axes, rows]``); an axis dimension
        of 1, or ``[N]`` (``[rows]``), gives every axis the same. Rows may lie anywhere (a
        projection's ``[B, N, H, D]`` transposed is read in place); the results are
        contiguous. Differentiable in reverse mode, any number of times; of a tensor that
        needs no gradient, the result needs none."""
        key = (q.shape, q.stride(), q.dtype, q.device, None if k is None else (k.shape, k.stride(), k.dtype, k.device),
               positions.shape, positions.stride(), positions.dtype, positions.device)
        strides = self._known.get(key)           # checked before: a step's host time counts
        if strides is None:
            if len(self._known) >= 4096:
                self._known.clear()
            strides = self._known[key] = self._check(q, k, positions)
        _refuse_tangents(*((q,) if k is None else (q, k)))
        return self._apply(q, k, positions, strides, False)

    def _check(self, q, k, positions):
        """The positions' strides; raises for tensors that do not fit."""
        if q.dim() not in (3, 4) or (k is not None and k.dim() != q.dim()):
            raise ValueError("q and k must both be [B, H, N, D] or both [rows, H, D]")
        for name, t in (("q", q), ("k", k)):
            if t is None:
                continue
            if not t.is_cuda:
                raise ValueError("All inputs must live on a CUDA device")
            if t.dtype not in _DTYPE_CODE or t.dtype != q.dtype:
                raise ValueError(f"q and k must share one dtype among float32/float16/bfloat16, got {t.dtype} for {name}")
            if t.shape[-1] != self.head_dim:
                raise ValueError(f"{name} must have head_dim {self.head_dim}, got {t.shape[-1]}")
            if t.device != q.device:
                raise ValueError("q and k must live on one device")
        if k is not None and (k.shape[0] != q.shape[0] or (q.dim() == 4 and k.shape[2] != q.shape[2])):
            raise ValueError("q and k must hold the same tokens")
        return _Strides3(*self._position_strides(positions, q))

    def _apply(self, q, k, positions, strides, inverse):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k)):
            return _Rotate.apply(self, q, k, positions, strides, inverse)
        return self._rotate(q, k, positions, strides, inverse)

    def _rotate(self, q, k, positions, strides, inverse):
        """The launch; either tensor may be missing."""
        if q is None or k is None or not (q.numel() and k.numel()):
            outs = [None if t is None else self._launch(t, None, positions, strides, inverse)[0] for t in (q, k)]
            return tuple(outs)
        return self._launch(q, k, positions, strides, inverse)

    def _launch(self, q, k, positions, strides, inverse):
        """``q``, and ``k`` if there is one (neither then empty)."""
        out, out_k = _dense_like(q), None
        if not q.numel():
            return out, None
        # the plan: (copy, heads, strides) of each, (batch, tokens, head_dim)
        key = (q.shape, q.stride(), q.dtype, q.data_ptr() % 16,
               None if k is None else (k.shape, k.stride(), k.data_ptr() % 16))
        plan = self._launches.get(key)
        if plan is None:
            if len(self._launches) >= 4096:
                self._launches.clear()
            plan = self._launches[key] = self._plan(q, k)
        copy, heads, at, copy_k, heads_k, at_k, sizes = plan
        if copy:
            q = _copied(q)
        src_k = dst_k = 0
        if k is not None:
            out_k = _dense_like(k)
            if copy_k:
                k = _copied(k)
            src_k, dst_k = k.data_ptr(), out_k.data_ptr()
        device = q.device
        turns, axis = self._table(device)
        with _on_device(device):
            rc = _lib.load().gki_rotary(
                q.data_ptr(), out.data_ptr(), heads, at, src_k, dst_k, heads_k, at_k, _DTYPE_CODE[q.dtype], *sizes,
                turns.data_ptr(), axis.data_ptr(), self.pairs, self.interleaved, inverse, positions.data_ptr(),
                positions.dtype == torch.int64, strides, _current_stream(device))
        if rc:
            _lib.check(rc, "gki_rotary")
        return out, out_k

    def _plan(self, q, k):
        plan = []
        for t in (q, k):
            if t is None:
                plan += [False, 0, None]
                continue
            copy, dense = not _in_place(t), torch.empty(t.shape, dtype=t.dtype, device="meta")
            plan += [copy, t.shape[1], _strides(dense if copy else t, dense)]
        shape = q.shape
        return (*plan, (1, shape[0], self.head_dim) if len(shape) == 3 else (shape[0], shape[2], self.head_dim))
