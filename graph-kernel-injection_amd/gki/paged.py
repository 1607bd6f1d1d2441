"""Requests of different lengths over paged keys and values, with sinks and a window.

``StreamingKVCache`` holds a batch whose sequences have one length. Here requests come and
go, each with a length of its own:

* ``PageTable`` says where tokens live. Position ``p`` of a request lies in its page ``p //
  page_size``; pages come from a queue of free ones. Everything is on the GPU: ``extend``
  gives a step's tokens their slots (and pages that no later token can see under the
  StreamingLLM rule back), ``accept`` keeps some of them, ``release`` ends requests. No call
  synchronises; a step that does not fit changes nothing and is told by ``check``.
* ``PagedKVCache`` holds a layer's keys and values, ``[num_pages, H, page_size, D]``, for the
  table that all layers share. ``append`` writes a step's tokens, ``append_rotated`` turns
  queries and keys by their positions on the way, ``attend`` runs the queries, ``accept``
  moves the rows of an accepted draft.

A step's tokens are packed, one request's after the other's: ``[rows, H, D]``. Requests
bring any number each, a chunk of a prompt beside single tokens::

    table = PageTable(max_requests, num_pages, StreamingMaskSpec(4, 2048))
    cache = PagedKVCache(table, kv_heads, 128)
    batch = table.extend(counts, rows)              # counts: int32 [max_requests]
    cache.append(k, v, batch)
    o = cache.attend(q, batch)

Drafted tokens form trees: ``extend(..., parents=...)`` places node ``i`` at ``base +
depth_i``, where it sees its request's earlier keys by the rule and of the step's own only
its ancestors and itself. After verification ``cache.accept`` (each layer) and
``table.accept`` keep a path.

There is no CPU or eager fallback: a missing library raises ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib
from .masks import StreamingMaskSpec
from .ops import _DTYPE_CODE, _current_stream, _on_device, _refuse_tangents
from .rotary import MultiAxisRotary, _dense_like

_HEAD_DIMS = (64, 128)
_MAX_DRAFT = 256
_REFUSALS = ((1, "no free pages were left"), (2, "the counts sum to more than the rows given"),
             (4, "a count was negative, above max_count, or took a request past max_length"))


def _int_vector(name: str, t: torch.Tensor, shape: Tuple[int, ...], device: torch.device) -> torch.Tensor:
    if t.dtype == torch.int32 and t.shape == shape and t.device == device and t.is_contiguous():
        return t                     # a step's host time counts
    if tuple(t.shape) != shape or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be an int32 or int64 tensor {list(shape)}, got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must live on {device}")
    if t.dtype == torch.int64:
        t = t.clamp(-1, 1 << 30).to(torch.int32)     # past either end every value means the same
    return t.contiguous()


class TokenBatch:
    """Where a step's tokens go (``PageTable.extend``): ``rows`` packed rows, those of request
    ``r`` being ``row_starts[r] .. row_starts[r + 1] - 1``; ``base[r]`` positions came before
    them. ``slots`` (page * page_size + place in it) and ``positions`` of each row, -1 and 0
    behind the last request. Drafts: ``ancestors``, 64 nodes to a word, which of a request's
    nodes a row sees. A batch serves its requests until their next ``extend`` or ``release``,
    which may give pages back that its rows see."""

    __slots__ = ("table", "rows", "max_count", "words", "ancestors", "_ints")

    def __init__(self, table, rows, max_count, words, ancestors, ints) -> None:
        self.table, self.rows, self.max_count, self.words = table, rows, max_count, words
        # requests (PageTable's for attend), slots (int64), row_starts, base and positions, in one
        # allocation of int32
        self.ancestors, self._ints = ancestors, ints

    @property
    def slots(self) -> torch.Tensor:
        at = 4 * (self.table.max_requests + 1)
        return self._ints[at:at + 2 * self.rows].view(torch.int64)

    def _after_slots(self, start: int, end: Optional[int]) -> torch.Tensor:
        at = 4 * (self.table.max_requests + 1) + 2 * self.rows
        return self._ints[at + start:None if end is None else at + end]

    @property
    def row_starts(self) -> torch.Tensor:
        return self._after_slots(0, self.table.max_requests + 1)

    @property
    def base(self) -> torch.Tensor:
        n = self.table.max_requests
        return self._after_slots(n + 1, 2 * n + 1)

    @property
    def positions(self) -> torch.Tensor:
        return self._after_slots(2 * self.table.max_requests + 1, None)

    def _pointers(self) -> Tuple[int, int, int, int, int]:
        """Of requests, slots, row_starts, base and positions."""
        at, n = self._ints.data_ptr(), self.table.max_requests
        slots = at + 16 * (n + 1)
        starts = slots + 8 * self.rows
        return at, slots, starts, starts + 4 * (n + 1), starts + 4 * (2 * n + 1)


class PageTable:
    """Pages of up to ``max_requests`` requests of up to ``max_length`` positions each
    (rounded up to whole pages).

    ``page_size``: a power of two from 16 to 1024. ``spec``: what a query sees, the first
    ``sink_size`` and the last ``window_size`` positions; pages behind the window, sinks
    apart, return to the queue when their request is extended, so ``max_length`` bounds
    positions, not memory. ``max_length``: up to 2^30; it defaults to all pages for one request.

    ``lengths`` (int32 ``[max_requests]``) and ``block_table`` (int32 ``[max_requests,
    pages]``, -1: none) are the table's own: read them, do not write.
    """

    def __init__(self, max_requests: int, num_pages: int, spec: StreamingMaskSpec, page_size: int = 64,
                 max_length: Optional[int] = None, device: torch.device | str = "cuda") -> None:
        if not 1 <= max_requests <= 1 << 20:
            raise ValueError(f"max_requests must be in [1, 2^20], got {max_requests}")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError(f"page_size must be a power of two in [16, 1024], got {page_size}")
        if not 1 <= num_pages or num_pages * page_size >= 1 << 31:
            raise ValueError(f"num_pages must be positive, num_pages * page_size below 2^31, got {num_pages}")
        if spec.sink_size >= 1 << 30:
            raise ValueError("sink_size must be below 2^30")
        max_length = min(num_pages * page_size, 1 << 30) if max_length is None else int(max_length)
        if not 1 <= max_length <= 1 << 30:
            raise ValueError(f"max_length must be in [1, 2^30], got {max_length}")
        self.max_requests, self.num_pages, self.page_size = int(max_requests), int(num_pages), int(page_size)
        self.spec = spec
        self.sink_size, self.window_size = int(spec.sink_size), min(int(spec.window_size), 1 << 30)
        self.max_pages = -(-max_length // self.page_size)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError("PageTable lives on a CUDA (HIP) device")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        n = self.max_requests
        self._sizes = (n, self.max_pages, self.page_size, self.num_pages, self.sink_size, self.window_size)
        # lengths, pages taken, first page behind the sinks that is kept; the queue's head and count, the status
        self._state = torch.zeros(3 * n + 3, dtype=torch.int32, device=self.device)
        self._state[2 * n:3 * n] = -(-self.sink_size // self.page_size)
        self._state[3 * n + 1] = self.num_pages
        self.lengths = self._state[:n]
        self._status = self._state[3 * n + 2:]
        self.block_table = torch.full((n, self.max_pages), -1, dtype=torch.int32, device=self.device)
        self._ring = torch.arange(self.num_pages, dtype=torch.int32, device=self.device)

    def _arguments(self) -> tuple:
        at, n = self._state.data_ptr(), self.max_requests
        return (at, at + 4 * n, at + 8 * n, self.block_table.data_ptr(), self._ring.data_ptr(), at + 12 * n,
                at + 12 * n + 8, *self._sizes)

    def extend(self, counts: torch.Tensor, rows: int, max_count: Optional[int] = None,
               parents: Optional[torch.Tensor] = None) -> TokenBatch:
        """Places ``counts[r]`` new tokens of each request ``r`` (int32 or int64
        ``[max_requests]`` on the device) behind its ``lengths[r]``, which grow by them.

        ``rows``: the packed rows that the step's tensors have, at least the sum of the
        counts. ``max_count``: the largest count there can be (default: ``rows``); small ones
        let ``attend`` run short rows as such. ``parents`` (``[rows]``): the tokens are drafts,
        trees of up to 256 nodes a request, each with the number of its parent among the
        request's tokens, which is smaller than its own (any other value: no parent).

        A step for which pages run out, whose counts do not fit ``rows``, or with a count that
        is negative, above ``max_count`` or leads past ``max_length``, changes nothing: its
        batch has no tokens (``check`` tells)."""
        counts = _int_vector("counts", counts, (self.max_requests,), self.device)
        rows = int(rows)
        if not 0 <= rows < 1 << 30:
            raise ValueError(f"rows must be in [0, 2^30), got {rows}")
        max_count = rows if max_count is None else int(max_count)
        if max_count < 0:
            raise ValueError(f"max_count must not be negative, got {max_count}")
        max_count = min(max_count, rows)
        words, ancestors = 0, None
        if parents is not None:
            parents = _int_vector("parents", parents, (rows,), self.device)
            if max_count > _MAX_DRAFT:
                raise ValueError(f"trees hold up to {_MAX_DRAFT} nodes: max_count is {max_count}")
            words = max(1, -(-max_count // 64))
            ancestors = torch.empty((rows, words), dtype=torch.int64, device=self.device)
        ints = torch.empty(6 * self.max_requests + 5 + 3 * rows, dtype=torch.int32, device=self.device)
        batch = TokenBatch(self, rows, max_count, words, ancestors, ints)
        requests, slots, row_starts, base, positions = batch._pointers()
        lib = _lib.load()
        with _on_device(self.device):
            rc = lib.gki_page_extend(
                counts.data_ptr(), 0 if parents is None else parents.data_ptr(), rows, max_count, words,
                *self._arguments(), row_starts, base, positions, slots,
                0 if ancestors is None else ancestors.data_ptr(), requests, _current_stream(self.device))
        if rc:
            _lib.check(rc, "gki_page_extend")
        return batch

    def accept(self, batch: TokenBatch, accepted: torch.Tensor) -> None:
        """Of the tokens that ``batch`` placed, request ``r`` keeps the first ``accepted[r]``
        (clamped to ``0 .. count``); their pages stay the request's. Requests without tokens
        in the batch keep their length, and none grows: what a call gave up is gone."""
        if batch.table is not self:
            raise ValueError("the batch belongs to another table")
        accepted = _int_vector("accepted", accepted, (self.max_requests,), self.device)
        _, _, row_starts, base, _ = batch._pointers()
        with _on_device(self.device):
            rc = _lib.load().gki_page_accept(self._state.data_ptr(), base, row_starts, accepted.data_ptr(),
                                             self.max_requests, _current_stream(self.device))
        if rc:
            _lib.check(rc, "gki_page_accept")

    def release(self, done: torch.Tensor) -> None:
        """Requests marked in ``done`` (bool ``[max_requests]`` on the device) give their
        pages back and hold nothing."""
        if tuple(done.shape) != (self.max_requests,) or done.dtype != torch.bool:
            raise ValueError(f"done must be a bool tensor [{self.max_requests}], got {done.dtype} {tuple(done.shape)}")
        if done.device != self.device:
            raise ValueError(f"done must live on {self.device}")
        done = done.contiguous()
        with _on_device(self.device):
            _lib.check(_lib.load().gki_page_release(done.data_ptr(), *self._arguments(), _current_stream(self.device)),
                       "gki_page_release")

    def check(self) -> int:
        """Synchronises: raises ``RuntimeError`` if a step was refused since the last check,
        else returns the number of free pages."""
        n = self.max_requests
        free, status = self._state[3 * n + 1:].tolist()
        if status:
            self._status.zero_()
            raise RuntimeError("PageTable.extend refused a step: " + "; ".join(m for bit, m in _REFUSALS if status & bit))
        return free


class PagedKVCache:
    """A layer's keys and values in the pages of ``table``: ``k_pages`` / ``v_pages``,
    ``[num_pages, heads, page_size, head_dim]`` in ``dtype`` (float16 or bfloat16), head_dim 64
    or 128. Queries may have any multiple of ``heads`` (grouped-query attention).

    No gradient flows through the cache, and tensors with a forward-mode tangent are refused
    (``NotImplementedError``). A NaN or infinity among a request's own values
    reaches the rows of the call that read it, as in the sparse op; what other requests
    left in a page is never seen. Calls on other streams than the table's last ``extend``
    have to be ordered behind it by the caller.
    """

    def __init__(self, table: PageTable, heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16) -> None:
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a paged cache takes float16 or bfloat16, got {dtype}")
        if head_dim not in _HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
        if not 1 <= heads <= 65535:
            raise ValueError(f"heads must be in [1, 65535], got {heads}")
        self.table, self.heads, self.head_dim, self.dtype = table, int(heads), int(head_dim), dtype
        self.device = table.device
        shape = (table.num_pages, self.heads, table.page_size, self.head_dim)
        self.k_pages, self.v_pages = (torch.zeros(shape, dtype=dtype, device=self.device) for _ in range(2))
        self._dtype = _DTYPE_CODE[dtype]
        self._strides: dict = {}         # (shape, strides, ...) of rows -> their row stride, 0: to be copied
        self._plans: dict = {}           # (max_count, Hq) -> workgroups, floats of their workspace

    def _batch(self, batch: TokenBatch) -> None:
        if batch.table is not self.table:
            raise ValueError("the batch belongs to another table")

    def _rows(self, name: str, t: torch.Tensor, rows: int, grouped: bool = False) -> Tuple[torch.Tensor, int]:
        """``t`` as the kernels read it, and its row stride."""
        key = (t.shape, t.stride(), t.dtype, t.device, rows, grouped)
        stride = self._strides.get(key)          # checked before: a step's host time counts
        if stride is None:
            if len(self._strides) >= 4096:
                self._strides.clear()
            stride = self._strides[key] = self._row_stride(name, t, rows, grouped)
        if stride and t.data_ptr() % 16 == 0:
            return t, stride
        t = t.contiguous()
        return (t if t.data_ptr() % 16 == 0 else t.clone()), t.shape[1] * self.head_dim

    def _row_stride(self, name: str, t: torch.Tensor, rows: int, grouped: bool) -> int:
        """The row stride of ``t``, 0 if it has to be copied; raises where it does not fit."""
        shape = t.shape
        ok = len(shape) == 3 and shape[0] == rows and shape[2] == self.head_dim
        if not ok or not (shape[1] == self.heads or (grouped and shape[1] > 0 and shape[1] % self.heads == 0)):
            want = "a multiple of " + str(self.heads) if grouped else str(self.heads)
            raise ValueError(f"{name} must be [{rows}, {want}, {self.head_dim}], got {tuple(shape)}")
        if t.dtype != self.dtype:
            raise ValueError(f"{name} must be {self.dtype}, got {t.dtype}")
        if t.device != self.device:
            raise ValueError(f"{name} must live on {self.device}")
        row, head, one = t.stride()
        width = shape[1] * self.head_dim
        # rows of a fused projection are read in place
        return row if one == 1 and (head == self.head_dim or shape[1] == 1) and row >= width and row % 8 == 0 else 0

    def append(self, k: torch.Tensor, v: torch.Tensor, batch: TokenBatch) -> None:
        """Writes the step's keys and values (``[rows, heads, D]``) to their slots; rows
        behind the last request are left out."""
        self._batch(batch)
        _refuse_tangents(k, v)
        (k, k_stride), (v, v_stride) = self._rows("k", k, batch.rows), self._rows("v", v, batch.rows)
        t = self.table
        with _on_device(self.device):
            rc = _lib.load().gki_paged_append(
                k.data_ptr(), v.data_ptr(), k_stride, v_stride, self.k_pages.data_ptr(), self.v_pages.data_ptr(),
                batch._pointers()[1], self._dtype, batch.rows, self.heads, self.head_dim, t.num_pages, t.page_size,
                _current_stream(self.device))
        if rc:
            _lib.check(rc, "gki_paged_append")

    def append_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: TokenBatch,
                       rotary: MultiAxisRotary, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``append`` with the keys turned by ``rotary`` as they are written; returns the
        queries (``[rows, Hq, D]``) turned, contiguous. ``positions``: as ``rotary`` takes
        them for packed rows; default: the batch's, for every axis."""
        self._batch(batch)
        _refuse_tangents(q, k, v)
        q, q_stride = self._rows("q", q, batch.rows, grouped=True)
        (k, k_stride), (v, v_stride) = self._rows("k", k, batch.rows), self._rows("v", v, batch.rows)
        if rotary.head_dim != self.head_dim:
            raise ValueError(f"rotary must have head_dim {self.head_dim}, got {rotary.head_dim}")
        if positions is None:
            at, wide, axis_stride, row_stride = batch._pointers()[4], 0, 0, 1
        else:
            axis_stride, _, row_stride = rotary._position_strides(positions, q)
            at, wide = positions.data_ptr(), int(positions.dtype == torch.int64)
        out = _dense_like(q)
        turns, axis = rotary._table(self.device)
        t = self.table
        with _on_device(self.device):
            rc = _lib.load().gki_paged_append_rotated(
                q.data_ptr(), out.data_ptr(), q_stride, q.shape[1], k.data_ptr(), v.data_ptr(), k_stride, v_stride,
                self.k_pages.data_ptr(), self.v_pages.data_ptr(), batch._pointers()[1], self._dtype, batch.rows,
                self.heads, self.head_dim, t.num_pages, t.page_size, turns.data_ptr(), axis.data_ptr(), rotary.pairs,
                int(rotary.interleaved), at, wide, axis_stride, row_stride, _current_stream(self.device))
        if rc:
            _lib.check(rc, "gki_paged_append_rotated")
        return out

    def attend(self, q: torch.Tensor, batch: TokenBatch, softmax_scale: Optional[float] = None,
               return_lse: bool = False):
        """``O`` of the step's queries ``[rows, Hq, D]`` over their requests' keys, the step's
        own among them, which ``append`` has written before (and the natural-log LSE
        ``[rows, Hq]`` fp32 when ``return_lse``). A row that sees no key, and rows behind the
        last request, give zeros."""
        self._batch(batch)
        _refuse_tangents(q)
        q, q_stride = self._rows("q", q, batch.rows, grouped=True)
        scale = 1.0 / math.sqrt(self.head_dim) if softmax_scale is None else float(softmax_scale)
        if not math.isfinite(scale):
            raise ValueError(f"softmax_scale must be finite, got {scale}")
        t, H = self.table, q.shape[1]
        lib = _lib.load()
        key = (batch.max_count, H)
        plan = self._plans.get(key)
        if plan is None:
            if len(self._plans) >= 4096:
                self._plans.clear()
            n = ctypes.c_int64()
            groups = lib.gki_paged_groups(batch.max_count, H, self.heads, self.head_dim, t.max_pages, t.page_size,
                                          t.sink_size, t.window_size, ctypes.byref(n))
            plan = self._plans[key] = groups, n.value
        groups, floats = plan
        work = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
        o = _dense_like(q)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if return_lse else None
        requests, _, _, _, positions = batch._pointers()
        with _on_device(self.device):
            rc = lib.gki_paged_attend(
                q.data_ptr(), q_stride, self.k_pages.data_ptr(), self.v_pages.data_ptr(), o.data_ptr(),
                0 if lse is None else lse.data_ptr(), requests, positions, t.block_table.data_ptr(),
                0 if batch.ancestors is None else batch.ancestors.data_ptr(), batch.words, self._dtype, batch.rows,
                batch.max_count, t.max_requests, H, self.heads, self.head_dim, t.max_pages, t.num_pages, t.page_size,
                t.sink_size, t.window_size, scale, work.data_ptr() if floats else 0, groups,
                _current_stream(self.device))
        if rc:
            _lib.check(rc, "gki_paged_attend")
        return o if lse is None else (o, lse)

    def accept(self, batch: TokenBatch, paths: torch.Tensor, accepted: torch.Tensor) -> None:
        """Moves the rows of each request's accepted path, nodes ``paths[r, 0 .. accepted[r] -
        1]`` of the batch's drafts from the root down (int32 or int64 ``[max_requests, n]``),
        to the slots of positions ``base[r], base[r] + 1, ...``; ``table.accept`` with the same
        ``accepted`` (at most ``n``) then sets the lengths. A node that is not ``i .. count - 1`` at place ``i`` moves nothing."""
        self._batch(batch)
        t = self.table
        if paths.dim() != 2:
            raise ValueError(f"paths must be [{t.max_requests}, n], got {tuple(paths.shape)}")
        paths = _int_vector("paths", paths, (t.max_requests, paths.shape[1]), self.device)
        accepted = _int_vector("accepted", accepted, (t.max_requests,), self.device)
        with _on_device(self.device):
            rc = _lib.load().gki_paged_accept(
                self.k_pages.data_ptr(), self.v_pages.data_ptr(), *batch._pointers()[1:3],
                paths.data_ptr(), accepted.data_ptr(), self._dtype, t.max_requests, paths.shape[1], self.heads,
                self.head_dim, t.num_pages, t.page_size, _current_stream(self.device))
        if rc:
            _lib.check(rc, "gki_paged_accept")
