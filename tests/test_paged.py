"""Page tables, attention over pages and drafted trees: tables against ``oracle.pages.Book``
entry by entry, outputs against 64 bits.

Bounds: ``oracle.pages.attend`` (each rounding counted by half a unit); the root mean square of
an output's error may be twice that of independent roundings.
"""

from __future__ import annotations

import ctypes
import math
import random

import pytest
import torch

from gki import MultiAxisRotary, PagedKVCache, PageTable, StreamingMaskSpec, _lib, cross_attention
from oracle import pages as op

DEV = "cuda"
NULL = ctypes.c_void_p(0)


# ---- refusals, on the CPU ---------------------------------------------------------------------------------------


def test_c_entries_refuse_before_launch():
    lib = _lib.load()

    def extend(counts=16, parents=0, rows=5, max_count=5, words=1, R=2, max_pages=8, page=64, pages=9, sink=4, window=8,
               starts=16, slots=16, ancestors=16, requests=16):
        return lib.gki_page_extend(counts, parents, rows, max_count, words, *[16] * 7, R, max_pages, page, pages, sink,
                                   window, starts, 16, 16, slots, ancestors, requests, NULL)

    assert extend(page=48) == 1 and extend(page=8) == 1 and extend(page=2048) == 1 and extend(R=0) == 1
    assert extend(pages=0) == 1 and extend(pages=2**25) == 1 and extend(max_pages=2**25) == 1 and extend(sink=-1) == 1
    assert extend(sink=2**30) == 1 and extend(window=-1) == 1 and extend(rows=-1) == 1 and extend(counts=0) == 1
    assert extend(starts=0) == 1 and extend(slots=0) == 1 and extend(R=2**21) == 1
    assert extend(parents=16, rows=300, max_count=257, words=5) == 1 and extend(parents=16, max_count=65, rows=65) == 1
    assert extend(parents=16, ancestors=0) == 1 and extend(requests=0) == 1 and extend(requests=8) == 1
    assert lib.gki_page_release(0, *[16] * 7, 2, 8, 64, 9, 4, 8, NULL) == 1
    assert lib.gki_page_accept(16, 16, 16, 16, 0, NULL) == 1 and lib.gki_page_accept(16, 0, 16, 16, 2, NULL) == 1

    def append(k=16, stride=128, kp=16, dtype=2, rows=3, H=2, D=64, pages=9, page=64):
        return lib.gki_paged_append(k, 16, stride, 128, kp, 16, 16, dtype, rows, H, D, pages, page, NULL)

    assert append(dtype=0) == 2 and append(D=32) == 2 and append(H=0) == 1 and append(k=0) == 1 and append(k=24) == 1
    assert append(stride=120) == 1 and append(stride=132) == 1 and append(kp=8) == 1 and append(page=20) == 1
    assert append(rows=-1) == 1 and append(rows=0) == 0

    def rotated(q=16, out=16, H=4, pairs=32, turns=16, at=16, dtype=2, rows=3, stride=256):
        return lib.gki_paged_append_rotated(q, out, stride, H, 16, 16, 128, 128, 16, 16, 16, dtype, rows, 2, 64, 9, 64,
                                            turns, 16, pairs, 0, at, 0, 0, 1, NULL)

    assert rotated(pairs=12) == 1 and rotated(pairs=40) == 1 and rotated(turns=0) == 1 and rotated(at=0) == 1
    assert rotated(q=0) == 1 and rotated(out=8) == 1 and rotated(dtype=0) == 2 and rotated(stride=64) == 1
    assert rotated(H=0) == 1 and rotated(rows=2**24) == 1 and rotated(rows=0) == 0

    def attend(q=16, stride=256, o=16, words=0, ancestors=0, dtype=2, rows=3, most=3, R=2, H=4, H_kv=2, D=64, scale=0.1,
               ws=0, n=1, sink=4, window=8):
        return lib.gki_paged_attend(q, stride, 16, 16, o, 0, 16, 16, 16, ancestors, words, dtype, rows, most, R, H, H_kv,
                                    D, 8, 9, 64, sink, window, scale, ws, n, NULL)

    assert attend(dtype=0) == 2 and attend(D=16) == 2 and attend(H=3) == 1 and attend(R=0) == 1 and attend(q=0) == 1
    assert attend(o=8) == 1 and attend(stride=128) == 1 and attend(scale=math.inf) == 1 and attend(scale=math.nan) == 1
    assert attend(ancestors=16, words=0) == 1 and attend(ancestors=16, words=1, most=65, rows=65) == 1
    assert attend(n=0) == 1 and attend(n=4097) == 1 and attend(ws=8) == 1
    floats = ctypes.c_int64()
    groups = lib.gki_paged_groups(30, 8, 2, 128, 100, 64, 4, 2048, ctypes.byref(floats))
    assert groups >= 256 and floats.value == groups * (2 * 120 * 130 + 5)
    assert lib.gki_paged_groups(200, 8, 2, 64, 100, 64, 4, 2048, ctypes.byref(floats)) * (2 * 128 * 66 + 5) == floats.value
    for few in ((30, 8, 2, 128, 100, 64, 4, 100), (30, 8, 2, 128, 3, 64, 4, 2048), (0, 8, 2, 128, 100, 64, 4, 2048)):
        assert lib.gki_paged_groups(*few, ctypes.byref(floats)) == groups and floats.value == 0
    assert lib.gki_paged_groups(30, 8, 2, 128, 100, 64, 4, 2048, None) == groups
    assert attend(sink=2**30) == 1 and attend(window=-1) == 1 and attend(rows=0) == 0
    assert lib.gki_paged_accept(16, 16, 16, 16, 0, 16, 2, 2, 5, 2, 64, 9, 64, NULL) == 1
    assert lib.gki_paged_accept(16, 16, 16, 16, 16, 16, 0, 2, 5, 2, 64, 9, 64, NULL) == 2
    assert lib.gki_paged_accept(16, 16, 16, 16, 16, 16, 2, 2, 0, 2, 64, 9, 64, NULL) == 0


@pytest.mark.parametrize("pages,page", [(2**24, 64), (2**24 + 1, 64), (2**21 - 1, 1024), (2**27 - 1, 16)])
def test_pools_past_the_longest_request_need_no_max_length(pages, page):
    """Pools of 2^30 positions and more: all other arguments are right, so the device is what is refused."""
    spec = StreamingMaskSpec(4, 100)
    with pytest.raises(ValueError, match="CUDA"):
        PageTable(1, pages, spec, page_size=page, device="cpu")
    with pytest.raises(ValueError, match="max_length"):
        PageTable(1, pages, spec, page_size=page, max_length=2**30 + 1, device="cpu")


def test_oracle_sees_a_mistake():
    """The bounds are passed by neither zeros nor a shifted window."""
    gen = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 64, generator=gen) for n, h in ((5, 4), (70, 2), (70, 2)))
    right = op.seen(65, 5, 4, 20)
    o, _, bound, mean, _ = op.attend(q, k, v, right, 0.125, torch.bfloat16)
    wrong = op.attend(q, k, v, op.seen(65, 5, 4, 19), 0.125, torch.bfloat16)[0]
    assert ((o - wrong).abs() > bound).any() and (o.abs() > bound).any()
    assert (o - wrong).square().mean() > 16 * mean.mean()


# ---- helpers ----------------------------------------------------------------------------------------------------


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


class Run:
    """A table with one cache, and what they hold by plain lists."""

    def __init__(self, R, pages, sink, window, page=64, heads=2, D=64, dtype=torch.bfloat16, max_length=None, seed=0):
        self.table = PageTable(R, pages, StreamingMaskSpec(sink, window), page_size=page, max_length=max_length, device=DEV)
        self.book = op.Book(R, pages, page, sink, window, self.table.max_pages)
        self.cache = PagedKVCache(self.table, heads, D, dtype=dtype)
        # what no request has written must never be seen
        for pool in (self.cache.k_pages, self.cache.v_pages):
            pool.fill_(math.nan)
        self.R, self.sink, self.window, self.heads, self.D, self.dtype = R, sink, window, heads, D, dtype
        self.k = [torch.empty(0, heads, D, dtype=dtype, device=DEV) for _ in range(R)]
        self.v = [t.clone() for t in self.k]
        self.gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(self, n, heads):
        return torch.randn((n, heads, self.D), generator=self.gen, device=DEV).to(self.dtype)

    def extend(self, counts, rows=None, max_count=None, parents=None):
        rows = sum(counts) if rows is None else rows
        up = None if parents is None else _ints([p for t in parents for p in t] + [0] * (rows - sum(counts)))
        batch = self.table.extend(_ints(counts), rows, max_count=max_count, parents=up)
        self.base = self.book.extend(counts)
        self.counts, self.parents = counts, parents
        return batch

    def append(self, batch, k=None, v=None):
        k = self.normal(batch.rows, self.heads) if k is None else k
        v = self.normal(batch.rows, self.heads) if v is None else v
        self.cache.append(k, v, batch)
        self.hold(k, v)

    def hold(self, k, v):
        at = 0
        for r, n in enumerate(self.counts):
            self.k[r] = torch.cat([self.k[r][:self.base[r]], k[at:at + n]])
            self.v[r] = torch.cat([self.v[r][:self.base[r]], v[at:at + n]])
            at += n

    def grow(self, lengths, step=700):
        """Requests up to ``lengths``, a step at a time."""
        while any(a > b for a, b in zip(lengths, self.book.length)):
            self.append(self.extend([min(step, a - b) for a, b in zip(lengths, self.book.length)]))

    def check_tables(self, batch):
        torch.cuda.synchronize()
        t, b = self.table, self.book
        assert t.lengths.tolist() == b.length
        want = [[row.get(i, -1) for i in range(t.max_pages)] for row in b.table]
        assert t.block_table.tolist() == want
        assert t.check() == len(b.queue)
        starts = [0]
        for n in self.counts:
            starts.append(starts[-1] + n)
        assert batch.row_starts.tolist() == starts and batch.base.tolist() == self.base
        slots, positions, words = [], [], []
        for r, n in enumerate(self.counts):
            tree = op.chains(self.parents[r]) if self.parents else None
            slots += [b.slot(r, self.base[r] + i) for i in range(n)]
            positions += [self.base[r] + (len(tree[i]) - 1 if tree else i) for i in range(n)]
            if tree:
                vis = op.seen(self.base[r], n, self.sink, self.window, self.parents[r])[:, self.base[r]:]
                words += [[int(x) for x in row] + [0] * (64 * batch.words - n) for row in vis.tolist()]
        behind = batch.rows - len(slots)
        assert batch.slots.tolist() == slots + [-1] * behind
        assert batch.positions.tolist() == positions + [0] * behind
        if self.parents:
            bits = (batch.ancestors[:, :, None] >> torch.arange(64, device=DEV)) & 1
            assert bits.flatten(1).tolist() == words + [[0] * 64 * batch.words] * behind

    def check_attend(self, batch, q, got, lse=None, scale=None, tag=""):
        scale = 1 / math.sqrt(self.D) if scale is None else scale
        at, square, allowed, n_out = 0, 0.0, 0.0, 0
        for r, n in enumerate(self.counts):
            if n:
                parents = self.parents[r] if self.parents else None
                vis = op.seen(self.base[r], n, self.sink, self.window, parents).to(DEV)
                want, want_lse, bound, mean, lse_bound = op.attend(q[at:at + n], self.k[r], self.v[r], vis, scale, self.dtype)
                err = (got[at:at + n].double() - want).abs()
                assert torch.isfinite(got[at:at + n]).all(), (tag, r)
                assert (err <= bound).all(), (tag, r, n, self.base[r], (err / bound).max().item())
                square, allowed, n_out = square + float(err.square().sum()), allowed + float(mean.sum()), n_out + err.numel()
                if lse is not None:
                    off = (lse[at:at + n].double() - want_lse).abs()
                    assert (off <= lse_bound).all(), (tag, r, (off / lse_bound).max().item())
            at += n
        assert square <= 4 * allowed + 1e-30 * n_out, (tag, math.sqrt(square / max(allowed, 1e-300)))
        assert not got[at:].any() and (lse is None or not lse[at:].any()), tag


def _share(monkeypatch, groups):
    """Work shared among ``groups`` workgroups."""
    real = _lib.load().gki_paged_groups

    def fixed(*a):
        n, floats = real(*a), a[-1]._obj
        floats.value = floats.value // n * groups
        return groups

    monkeypatch.setattr(_lib.load(), "gki_paged_groups", fixed)


def _tree(rng, n):
    return [rng.choice([-1, i - 1, i - 1, rng.randint(0, i)]) if i else -1 for i in range(n)]


# ---- tables -----------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("R,page,sink,window,most", [
    (1, 64, 4, 100, 1), (3, 16, 0, 20, 50), (7, 32, 70, 33, 200), (70, 16, 4, 64, 40), (5, 128, 1, 0, 300),
    (1100, 16, 4, 40, 9), (2500, 64, 17, 1000, 3), (4, 1024, 4, 5, 2500)])
def test_tables_step_by_step(R, page, sink, window, most):
    """Random counts (none among them), releases and refused tokens, each step against plain lists."""
    rng = random.Random(R * page)
    longest = 12 * most + 200
    run = Run(R, R * (-(-(sink + window + 2 * most) // page) + 4), sink, window, page, max_length=longest)
    for step in range(14):
        counts = [0 if rng.random() < 0.3 else rng.randint(1, most) for _ in range(R)]
        counts = [min(c, longest - n) for c, n in zip(counts, run.book.length)]
        rows = sum(counts) + rng.choice([0, 0, 5])
        batch = run.extend(counts, rows, max_count=rng.choice([None, most]))
        run.check_tables(batch)
        if step % 3 == 1:
            keep = [rng.randint(0, c) for c in counts]
            run.table.accept(batch, _ints(keep))
            run.book.length = [b + k for b, k in zip(run.base, keep)]
        if step % 4 == 2:
            done = [rng.random() < 0.4 for _ in range(R)]
            run.table.release(_ints(done, torch.bool))
            run.book.release(done)
            assert run.table.check() == len(run.book.queue)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4096, 4097, 8192, 8193, 40000])
def test_tables_of_many_rows(rows):
    """Rows placed by the book-keeping workgroup and by a grid of their own."""
    run = Run(3, 3000, 4, 100000, 64)
    run.check_tables(run.extend([rows - 700, 0, 650], rows))


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 7, 64, 65, 200, 256])
def test_trees_of_tables(most):
    rng = random.Random(most)
    run = Run(6, 400, 4, 30, 16)
    run.grow([0, 5, 100, 64, 63, 1])
    for _ in range(3):
        counts = [most, 0, rng.randint(1, most), most, 1, rng.randint(1, most)]
        trees = [_tree(rng, n) for n in counts]
        batch = run.extend(counts, sum(counts) + 3, max_count=most, parents=trees)
        run.check_tables(batch)
        run.table.accept(batch, _ints([0] * 6))
        run.book.length = list(run.base)
    chain = [list(range(-1, most - 1))] + [[] for _ in range(5)]
    batch = run.extend([most, 0, 0, 0, 0, 0], max_count=most, parents=chain)
    run.check_tables(batch)


@pytest.mark.gpu
def test_refused_steps_change_nothing():
    run = Run(3, 10, 4, 1000, 16, max_length=100)
    run.grow([20, 0, 40])
    before = run.table._state.clone(), run.table.block_table.clone(), run.table._ring.clone()
    for counts, rows, most, parents, bit, message in (
            ([60, 60, 60], 180, None, None, 1, "no free pages"), ([5, 5, 5], 14, 5, None, 2, "more than the rows"),
            ([5, -1, 0], 5, 5, None, 4, "negative"), ([6, 0, 0], 6, 5, None, 4, "max_count"),
            ([0, 113, 0], 113, None, None, 4, "max_length"), ([60, 60, 60], 170, None, None, 3, "rows"),
            ([9, 9, 9], 20, 9, [0] * 20, 2, "rows")):
        assert run.book.refusal(counts, rows, rows if most is None else most) == bit
        batch = run.table.extend(_ints(counts), rows, max_count=most, parents=None if parents is None else _ints(parents))
        k, v, q = run.normal(rows, 2), run.normal(rows, 2), run.normal(rows, 4)
        held = run.cache.k_pages.clone(), run.cache.v_pages.clone()
        run.cache.append(k, v, batch)
        o, lse = run.cache.attend(q, batch, return_lse=True)
        run.cache.accept(batch, _ints([[0, 1]] * 3), _ints([2, 2, 2]))
        run.table.accept(batch, _ints([2, 2, 2]))
        assert not o.any() and not lse.any()
        assert batch.slots.eq(-1).all() and not batch.positions.any() and not batch.row_starts.any()
        assert batch.base.tolist() == run.book.length
        for a, b in zip(held, (run.cache.k_pages, run.cache.v_pages)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
        with pytest.raises(RuntimeError, match=message):
            run.table.check()
        assert run.table.check() == len(run.book.queue)
        assert all(torch.equal(a, b) for a, b in zip(before, (run.table._state, run.table.block_table, run.table._ring)))
    run.check_tables(run.extend([1, 2, 3]))


@pytest.mark.gpu
def test_counts_past_32_bits_are_refused():
    table = PageTable(2, 10, StreamingMaskSpec(4, 100), device=DEV)
    for big in (2**32 + 1, -2**32 - 1, 2**62):
        table.extend(_ints([big, 1], torch.int64), 5)
        with pytest.raises(RuntimeError, match="refused"):
            table.check()
    assert table.extend(_ints([1, 2], torch.int64), 5).row_starts.tolist() == [0, 1, 3]


# ---- attention --------------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv,sink,window,past,counts", [
    (1, 1, 4, 100, [0], [1]),
    (2, 2, 0, 3, [5, 0, 64], [1, 1, 1]),
    (8, 2, 4, 100, [300, 0, 63, 64, 65, 1], [1, 1, 1, 1, 1, 1]),
    (8, 1, 4, 130, [1000, 7, 500], [4, 0, 2]),
    (10, 2, 70, 50, [200, 3, 90], [3, 2, 7]),
    (4, 4, 4, 256, [0, 700, 100], [150, 40, 1]),
    (12, 2, 1, 1, [40, 129], [60, 3]),
    (6, 3, 4, 0, [40, 0], [5, 70]),
    (4, 2, 20, 5000, [900, 0, 0, 30], [130, 257, 0, 1]),
    (64, 1, 4, 90, [100, 2], [3, 1]),
    (2, 2, 4, 200, [100, 90, 300, 0, 500], [16, 17, 33, 32, 128])])
def test_attend_against_64_bits(dtype, D, page, heads, kv, sink, window, past, counts):
    run = Run(len(past), 4 * sum(past + counts) // page + 20, sink, window, page, kv, D, dtype, seed=sum(past) + heads)
    run.grow(past)
    batch = run.extend(counts, max_count=max(counts))
    run.append(batch)
    q = run.normal(batch.rows, heads)
    o, lse = run.cache.attend(q, batch, return_lse=True)
    run.check_tables(batch)
    run.check_attend(batch, q, o, lse)
    assert torch.equal(o, run.cache.attend(q, batch))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,page", [(64, 16), (64, 64), (128, 32), (128, 128)])
@pytest.mark.parametrize("heads,kv,sink,window,past,counts", [
    (1, 1, 4, 100, [0], [1]), (8, 8, 4, 512, [300], [7]), (8, 2, 4, 100, [300, 0, 63, 64, 65, 1], [26, 13, 20, 1, 0, 7]),
    (16, 2, 4, 2, [200, 9], [40, 12]), (4, 1, 66, 30, [500, 10, 70], [64, 60, 33]), (4, 2, 4, 130, [190, 64, 0], [256, 65, 130]),
    (5, 1, 0, 0, [30], [12])])
def test_trees_against_64_bits(dtype, D, page, heads, kv, sink, window, past, counts):
    rng = random.Random(sum(past))
    run = Run(len(past), 4 * sum(past + counts) // page + 20, sink, window, page, kv, D, dtype, seed=sum(past))
    run.grow(past)
    trees = [_tree(rng, n) for n in counts]
    batch = run.extend(counts, max_count=max(counts), parents=trees)
    run.append(batch)
    q = run.normal(batch.rows, heads)
    o, lse = run.cache.attend(q, batch, return_lse=True)
    run.check_tables(batch)
    run.check_attend(batch, q, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [1, 2, 7, 64, 500, 4096])
@pytest.mark.parametrize("counts,tree", [([1, 1, 1, 1], False), ([6, 1, 0, 20], False), ([40, 1, 300, 7], False), ([12, 30, 8, 1], True)])
def test_any_number_of_workgroups(groups, counts, tree, monkeypatch):
    _share(monkeypatch, groups)
    rng = random.Random(17)
    run = Run(4, 600, 4, 1500, 32, 2, 128, torch.bfloat16, seed=17)
    run.grow([5000, 900, 0, 1600])
    trees = [_tree(rng, n) for n in counts] if tree else None
    batch = run.extend(counts, max_count=max(counts), parents=trees)
    run.append(batch)
    q = run.normal(batch.rows, 8)
    o, lse = run.cache.attend(q, batch, return_lse=True)
    run.check_attend(batch, q, o, lse)
    assert torch.equal(o, run.cache.attend(q, batch))


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [1, 3, None])
@pytest.mark.parametrize("counts", [[1, 1], [2, 50]])
def test_more_pages_than_are_held_at_once(groups, counts, monkeypatch):
    """Walks of more than 1024 pages of 16 keys."""
    if groups:
        _share(monkeypatch, groups)
    run = Run(2, 4200, 4, 30000, 16, 1, 64, torch.float16, seed=18)
    run.grow([35000, 17000], 9000)
    batch = run.extend(counts)
    run.append(batch)
    q = run.normal(batch.rows, 2)
    o, lse = run.cache.attend(q, batch, return_lse=True)
    run.check_attend(batch, q, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [63, 64, 65, 200])
def test_many_requests(R):
    """More requests than a wave counts at once, some without tokens."""
    rng = random.Random(R)
    run = Run(R, 40 * R, 4, 700, 32, 2, 64, torch.bfloat16, seed=R)
    run.grow([rng.choice([0, 3, 100, 1100]) for _ in range(R)])
    for counts in ([rng.choice([0, 1, 1, 2]) for _ in range(R)], [rng.choice([0, 1, 20, 70]) for _ in range(R)], [0] * (R - 1) + [3]):
        batch = run.extend(counts, sum(counts) + 2, max_count=max(counts))
        run.append(batch)
        q = run.normal(batch.rows, 8)
        o, lse = run.cache.attend(q, batch, return_lse=True)
        run.check_attend(batch, q, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("most,kv,D", [(1, 2, 64), (20, 1, 128)])
def test_thousands_that_attend_at_once(most, kv, D):
    """More requests with tokens than 64 for each lane of a wave, some in between without."""
    rng = random.Random(most)
    R = 5000
    run = Run(R, 12 * R, 4, 60, 16, kv, D, torch.bfloat16, seed=most)
    run.grow([rng.choice([0, 3, 15, 64, 130]) for _ in range(R)])
    counts = [0 if r % 9 == 4 else rng.randint(1, most) for r in range(R)]
    assert sum(c > 0 for c in counts) > 4096
    batch = run.extend(counts, sum(counts) + 5, max_count=most)
    run.append(batch)
    q = run.normal(batch.rows, 4 * kv)
    o, lse = run.cache.attend(q, batch, return_lse=True)
    run.check_attend(batch, q, o, lse)
    assert torch.equal(o, run.cache.attend(q, batch))


@pytest.mark.gpu
def test_time_grows_with_the_requests_not_with_their_square():
    """65536 requests' single tokens, 8 heads: 524288 short walks. Counting all requests again for each walk
    takes 228 ms, the walks themselves less than 10."""
    R, heads = 65536, 8
    table = PageTable(R, 2 * R, StreamingMaskSpec(4, 100), page_size=16, max_length=32, device=DEV)
    cache = PagedKVCache(table, heads, 64)
    gen = torch.Generator(device=DEV).manual_seed(2)
    for n in (4, 1):
        batch = table.extend(torch.full((R,), n, dtype=torch.int32, device=DEV), n * R, max_count=n)
        k, v = (torch.randn((n * R, heads, 64), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
        cache.append(k, v, batch)
    q = torch.zeros((R, heads, 64), dtype=torch.bfloat16, device=DEV)
    took = []
    for _ in range(4):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        o = cache.attend(q, batch)
        end.record()
        end.synchronize()
        took.append(start.elapsed_time(end))
    # equal scores: the mean of a request's five values
    want = cache.v_pages[batch.slots // 16][:, :, :5].double().mean(2)
    # half a unit of the result and of each of five equal weights' sum, fp32 below
    assert (o.double() - want).abs().max() <= 2.0**-8 * want.abs().max() + 2.0**-20
    assert min(took) < 60, took


@pytest.mark.gpu
@pytest.mark.parametrize("page", [256, 512, 1024])
@pytest.mark.parametrize("dtype,D,heads,kv,counts,tree", [
    (torch.bfloat16, 128, 8, 2, [1, 3, 1, 0, 1], False), (torch.float16, 64, 4, 4, [1, 300, 40, 257, 5], False),
    (torch.float16, 128, 8, 1, [26, 60, 1, 0, 17], True)])
def test_attend_over_large_pages(page, dtype, D, heads, kv, counts, tree):
    """Pages that several key tiles lie in, among them of requests that end in the first and the last."""
    rng = random.Random(page)
    run = Run(5, 40, 70, 900, page, kv, D, dtype, max_length=8000, seed=page)
    run.grow([page - 1, 2 * page + 65, 3001, 0, 5])
    trees = [_tree(rng, n) for n in counts] if tree else None
    batch = run.extend(counts, max_count=max(counts), parents=trees)
    run.append(batch)
    q = run.normal(batch.rows, heads)
    o, lse = run.cache.attend(q, batch, return_lse=True)
    run.check_tables(batch)
    run.check_attend(batch, q, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("counts,tree", [([1] * 16, False), ([1] * 7 + [40, 300] + [2] * 7, False), ([1, 20, 7, 40] * 4, True)])
def test_steps_of_several_key_tiles(counts, tree):
    """A table whose longest requests could have more steps than 31 bits count: a step is two key tiles or more."""
    rng = random.Random(len(counts))
    run = Run(16, 130, 4, 2**30, 1024, 8, 64, torch.bfloat16, max_length=2**30, seed=22)
    # as gki_paged_attend reckons: row tiles of the rows given, times the steps of the longest walk
    tiles = (sum(counts) // 128 + 16) * 8
    assert tiles * (2**30 // 64 + 4) >= 2**31
    run.grow([rng.choice([0, 1, 63, 64, 500, 1025, 5000]) for _ in range(15)] + [9000], 3000)
    trees = [_tree(rng, n) for n in counts] if tree else None
    batch = run.extend(counts, max_count=max(counts), parents=trees)
    run.append(batch)
    q = run.normal(batch.rows, 8)
    o, lse = run.cache.attend(q, batch, return_lse=True)
    assert run.table.check() == len(run.book.queue)
    run.check_attend(batch, q, o, lse)
    assert torch.equal(o, run.cache.attend(q, batch))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_walks_of_more_than_65536_key_tiles(rows):
    """Equal scores over 4.3 million keys: every key tile adds 64 to one element's sum, all of them whole numbers."""
    past, page, D = 4300001, 1024, 64
    table = PageTable(1, past // page + 2, StreamingMaskSpec(4, 2**30), page_size=page, device=DEV)
    cache = PagedKVCache(table, 1, D, dtype=torch.float16)
    gen = torch.Generator(device=DEV).manual_seed(23)
    for n in (past, rows):
        batch = table.extend(_ints([n]), n)
        at = batch.positions[:, None] // 64 % D
        v = (at == torch.arange(D, device=DEV)).to(torch.float16)[:, None]
        cache.append(torch.zeros_like(v), v, batch)
    assert table.check() >= 0
    q = torch.randn((rows, 2, D), generator=gen, device=DEV).to(torch.float16)
    o, lse = cache.attend(q, batch, return_lse=True)
    n = past + 1 + torch.arange(rows, device=DEV).double()
    at = torch.arange(past + rows, device=DEV) // 64 % D
    held = torch.stack([torch.bincount(at[:past + 1 + i], minlength=D) for i in range(rows)]).double()
    want = (held / n[:, None])[:, None]
    # half a unit of fp16 (a tile of 64 more or less is two of them) and of the fp32 quotient
    assert ((o.double() - want).abs() <= (2.0**-11 + 2.0**-22) * want).all()
    # ln n is 15.3: fp32's logarithm and product, two units of 2^-23 of it each (a tile of 64 is 1.5e-5)
    assert ((lse.double() - n.log()[:, None]).abs() <= 4 * 2.0**-23 * 16).all()


@pytest.mark.gpu
def test_a_chain_is_plain_tokens():
    a, b = (Run(2, 60, 4, 50, 32, seed=3) for _ in range(2))
    for run in (a, b):
        run.grow([100, 3])
    q = a.normal(30, 8)
    plain = a.extend([20, 10])
    drafts = b.extend([20, 10], parents=[list(range(-1, 19)), list(range(-1, 9))])
    k, v = a.normal(30, 2), a.normal(30, 2)
    a.append(plain, k, v)
    b.append(drafts, k, v)
    assert torch.equal(a.cache.attend(q, plain), b.cache.attend(q, drafts))


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1, 1], [9, 100, 1]])
@pytest.mark.parametrize("scale", [0.0, -0.2, 0.7, 3e-5])
def test_any_finite_scale(scale, counts):
    run = Run(3, 60, 4, 80, 32, 2, 128, torch.float16, seed=4)
    run.grow([90, 0, 200])
    batch = run.extend(counts)
    run.append(batch)
    q = run.normal(batch.rows, 6)
    o, lse = run.cache.attend(q, batch, scale, return_lse=True)
    run.check_attend(batch, q, o, lse, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1], [3, 90]])
def test_large_logits(counts):
    run = Run(2, 60, 4, 300, 32, 2, 128, torch.bfloat16, seed=5)
    run.grow([500, 70])
    batch = run.extend(counts)
    run.append(batch, run.normal(batch.rows, 2) * 8)
    q = run.normal(batch.rows, 8) * 4
    run.check_attend(batch, q, run.cache.attend(q, batch))


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[2, 3, 1], [70, 30, 200]])
def test_rows_of_a_projection_and_strides(counts):
    """Views of one projection are read in place; strange strides and alignments are copied."""
    run = Run(3, 100, 4, 100, 16, 2, 64, torch.bfloat16, seed=6)
    run.grow([30, 100, 0])
    n, batch = sum(counts), None
    qkv = run.normal(n, 12).flatten(1)
    q, k, v = (t.unflatten(1, (-1, 64)) for t in qkv.split([512, 128, 128], 1))
    batch = run.extend(counts)
    run.append(batch, k, v)
    assert not q.is_contiguous()
    o = run.cache.attend(q, batch)
    run.check_attend(batch, q, o)
    odd = torch.empty(n * 8 * 64 + 1, dtype=q.dtype, device=DEV)[1:].view(n, 8, 64).copy_(q)
    heads_last = q.transpose(1, 2).contiguous().transpose(1, 2)
    for other in (odd, heads_last, q.contiguous()):
        assert torch.equal(run.cache.attend(other, batch), o)
    run.cache.append(k.flip(2).flip(2), v.transpose(0, 1).contiguous().transpose(0, 1), batch)
    assert torch.equal(run.cache.attend(q, batch), o)
    same = run.normal(1, 2).expand(n, -1, -1)               # one row for all
    run.append(batch, same, same)
    run.check_attend(batch, q, run.cache.attend(q, batch))


@pytest.mark.gpu
@pytest.mark.parametrize("counts,parents", [([1, 4], None), ([90, 40], None), ([5, 9], [[-1, 0, 0, 1, 1], [-1] * 9])])
def test_rows_behind_the_last_request(counts, parents):
    run = Run(2, 60, 4, 100, 16, seed=7)
    run.grow([30, 100])
    rows = sum(counts) + 70
    batch = run.extend(counts, rows, parents=parents)
    k, v, q = run.normal(rows, 2), run.normal(rows, 2), run.normal(rows, 4)
    for t in (k, v, q):
        t[sum(counts):] = math.nan
    run.append(batch, k, v)
    o, lse = run.cache.attend(q, batch, return_lse=True)
    run.check_tables(batch)
    run.check_attend(batch, q, o, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 1], [1, 300]])
def test_pages_of_others_are_never_seen(counts):
    """NaN and infinities in pages given back, in rows past a request's last and in refused drafts."""
    run = Run(2, 40, 4, 40, 16, seed=8)
    run.grow([100, 90])
    batch = run.extend([60, 50])
    bad = run.normal(110, 2).fill_(math.nan)
    run.cache.append(bad, bad, batch)
    run.table.accept(batch, _ints([0, 0]))
    run.book.length = list(run.base)
    run.table.release(_ints([False, True], torch.bool))
    run.book.release([False, True])
    run.cache.k_pages.view(-1, 2, 16, 64)[[p for p in run.book.queue]] = math.inf
    batch = run.extend(counts)
    run.append(batch)
    q = run.normal(batch.rows, 4)
    run.check_attend(batch, q, run.cache.attend(q, batch))


@pytest.mark.gpu
def test_long_requests_keep_their_pages():
    """A request of 40 windows holds a window of pages, and attends right all along."""
    run = Run(2, 14, 4, 64, 16, seed=9, max_length=4000)
    for step in range(60):
        batch = run.extend([43, 1 if step % 2 else 0])
        run.append(batch)
        q = run.normal(batch.rows, 4)
        run.check_attend(batch, q, run.cache.attend(q, batch), tag=step)
    run.check_tables(batch)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
def test_a_pool_past_2_31_elements(page):
    pages, heads, D = 2**31 // (page * 8 * 128) + 600 // page * 8, 8, 128
    table = PageTable(1, pages, StreamingMaskSpec(4, 300), page_size=page, max_length=700, device=DEV)
    cache = PagedKVCache(table, heads, D, dtype=torch.bfloat16)
    assert cache.k_pages.numel() > 2**31
    table._ring.copy_(table._ring.flip(0).clone())          # the last pages first
    gen = torch.Generator(device=DEV).manual_seed(1)
    k, v, q = (torch.randn((600, n, D), generator=gen, device=DEV).to(torch.bfloat16) for n in (8, 8, 16))
    batch = table.extend(_ints([600]), 600)
    assert batch.slots.min() * heads * D > 2**31 - 2**21 and batch.slots.max() * heads * D > 2**31
    cache.append(k, v, batch)
    o = cache.attend(q, batch)
    vis = op.seen(0, 600, 4, 300).to(DEV)
    want, _, bound, _, _ = op.attend(q, k, v, vis, D**-0.5, torch.bfloat16)
    assert ((o.double() - want).abs() <= bound).all()


# ---- drafts accepted, positions turned ------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
def test_an_accepted_path_moves_up(D, page):
    rng = random.Random(D)
    run = Run(5, 90, 4, 50, page, 3, D, torch.float16, seed=11)
    run.grow([30, 0, 100, 5, 64])
    for turn in range(4):
        counts = [26, 5, 0, 40, 1]
        trees = [_tree(rng, n) for n in counts]
        batch = run.extend(counts, max_count=40, parents=trees)
        run.append(batch)
        paths = [rng.choice(op.chains(t)) if t else [] for t in trees]
        if turn == 3:
            paths = [p[:1] for p in paths]
        before = run.cache.k_pages.clone()
        most = max(map(len, paths))
        accepted, padded = [len(p) for p in paths], [p + [0] * (most - len(p)) for p in paths]
        run.cache.accept(batch, _ints(padded, torch.int64 if turn % 2 else torch.int32), _ints(accepted))
        run.table.accept(batch, _ints(accepted))
        for r, p in enumerate(paths):
            for i, node in enumerate(p):
                a, b = run.book.slot(r, run.base[r] + node), run.book.slot(r, run.base[r] + i)
                assert torch.equal(run.cache.k_pages[b // page, :, b % page], before[a // page, :, a % page])
            for held in (run.k, run.v):
                held[r] = torch.cat([held[r][:run.base[r]], held[r][[run.base[r] + i for i in p]]])
            run.book.length[r] = run.base[r] + len(p)
    batch = run.extend([1, 1, 1, 1, 1])
    run.append(batch)
    run.check_tables(batch)
    q = run.normal(5, 6)
    run.check_attend(batch, q, run.cache.attend(q, batch))


@pytest.mark.gpu
def test_batches_of_different_requests_side_by_side():
    """Two steps of one table, each with requests of its own, attended and accepted in any order."""
    run = Run(3, 60, 4, 50, 16, seed=19)
    run.grow([60, 5, 90])
    one = run.extend([7, 0, 0])
    k, v, q = run.normal(7, 2), run.normal(7, 2), run.normal(7, 4)
    first = run.base, run.counts, k, v, q
    two = run.extend([0, 2, 30])
    run.append(two)
    q2 = run.normal(32, 4)
    run.cache.append(k, v, one)
    run.check_attend(two, q2, run.cache.attend(q2, two))
    run.table.accept(one, _ints([3, 9, 9]))
    assert run.table.lengths.tolist() == [63, 7, 120]
    run.table.accept(two, _ints([9, 1, 30]))
    assert run.table.lengths.tolist() == [63, 6, 120]
    run.base, run.counts, k, v, q = first
    run.hold(k, v)
    run.check_attend(one, q, run.cache.attend(q, one))


@pytest.mark.gpu
def test_accepting_never_lengthens():
    """A second accept, or one after its request was released, gives no position without a page."""
    run = Run(3, 60, 20, 50, 16, seed=21)
    run.grow([60, 5, 90])
    batch = run.extend([7, 2, 30])
    run.append(batch)
    run.table.accept(batch, _ints([3, 1, 20]))
    run.table.accept(batch, _ints([7, 0, 25]))
    assert run.table.lengths.tolist() == [63, 5, 110]
    run.table.release(torch.tensor([True, False, True], device=DEV))
    run.table.accept(batch, _ints([7, 2, 30]))
    assert run.table.lengths.tolist() == [0, 5, 0]
    run.book.release([True, False, True])
    run.book.length[1] = 5
    for r in (0, 2):
        run.k[r], run.v[r] = run.k[r][:0], run.v[r][:0]
    batch = run.extend([70, 3, 1])
    run.append(batch)
    run.check_tables(batch)
    q = run.normal(74, 4)
    run.check_attend(batch, q, run.cache.attend(q, batch))


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1, 2], [70, 3]])
def test_what_is_not_finite_stays_with_its_request(counts):
    """NaN in one request's keys, values or queries reaches no other request; a NaN query its own row alone."""
    run = Run(2, 60, 4, 100, 16, seed=20)
    run.grow([30, 100])
    batch = run.extend(counts)
    k, v, q = run.normal(batch.rows, 2), run.normal(batch.rows, 2), run.normal(batch.rows, 4)
    run.append(batch, k, v)
    want, want_lse = run.cache.attend(q, batch, return_lse=True)
    bad_q = q.clone()
    bad_q[counts[0], 1] = math.nan
    o, lse = run.cache.attend(bad_q, batch, return_lse=True)
    assert o[counts[0], 1].isnan().all() and lse[counts[0], 1].isnan()
    o[counts[0], 1], lse[counts[0], 1] = want[counts[0], 1], want_lse[counts[0], 1]
    assert torch.equal(o, want) and torch.equal(lse, want_lse)
    for bad in (math.nan, math.inf, -math.inf):
        bad_k, bad_v = k.clone(), v.clone()          # the first request's rows as before
        bad_k[counts[0]:] = bad_v[counts[0]:] = bad
        run.cache.append(bad_k, bad_v, batch)
        o = run.cache.attend(q, batch)
        assert torch.equal(o[:counts[0]], want[:counts[0]])
        assert not o[counts[0]:].isfinite().all()


@pytest.mark.gpu
def test_paths_that_are_none_move_nothing():
    run = Run(2, 30, 4, 50, 16, seed=12)
    batch = run.extend([6, 3], parents=[[-1, 0, 0, 1, 1, 2], [-1, 0, 1]])
    run.append(batch)
    before = run.cache.k_pages.clone(), run.cache.v_pages.clone()
    for paths, accepted in (([[0, 0, 1], [0, 1, 2]], [3, 3]), ([[-5, 6, 99], [7, 3, 2]], [3, 3]), ([[5, 5, 5], [2, 2, 2]], [0, -4]),
                            ([[0, 1, 2], [0, 1, 2]], [99, 99])):
        run.cache.accept(batch, _ints(paths), _ints(accepted))
        for a, b in zip(before, (run.cache.k_pages, run.cache.v_pages)):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), paths
    run.table.accept(batch, _ints([99, -7]))
    assert run.table.lengths.tolist() == [6, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,sections", [(64, (32,)), (128, (16, 24, 24)), (128, (5, 11)), (64, (8,))])
def test_append_rotated_is_rotary_and_append(dtype, interleaved, D, sections):
    """The same bits as ``MultiAxisRotary`` and ``append`` apart, and the rows behind left alone."""
    rope = MultiAxisRotary(D, sections, interleaved=interleaved)
    a, b = (Run(3, 60, 4, 100, 16, 2, D, dtype, seed=13) for _ in range(2))
    for run in (a, b):
        run.grow([100, 0, 37])
    for positions in (None, torch.randint(-5, 100000, (len(sections), 70), device=DEV),
                      torch.randint(0, 900, (70,), device=DEV, dtype=torch.int32)):
        one, two = a.extend([1, 60, 5], 70), b.extend([1, 60, 5], 70)
        qkv = a.normal(70, 10).flatten(1)
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([6 * D, 2 * D, 2 * D], 1))
        turned = a.cache.append_rotated(q, k, v, one, rope, positions)
        want_q, want_k = rope(q, k, two.positions if positions is None else positions)
        b.cache.append(want_k, v, two)
        assert torch.equal(turned, want_q)
        for x, y in ((a.cache.k_pages, b.cache.k_pages), (a.cache.v_pages, b.cache.v_pages)):
            assert torch.equal(x.view(torch.int16), y.view(torch.int16))


# ---- refusals, streams, graphs -----------------------------------------------------------------------------------------


@pytest.mark.gpu
def test_python_refusals():
    spec = StreamingMaskSpec(4, 100)
    for bad, message in ((dict(max_requests=0), "max_requests"), (dict(num_pages=0), "num_pages"), (dict(page_size=48), "page_size"),
                         (dict(max_length=0), "max_length"), (dict(num_pages=2**25), "2\\^31"), (dict(device="cpu"), "CUDA"),
                         (dict(max_length=2**30 + 1), "max_length")):
        with pytest.raises(ValueError, match=message):
            PageTable(**dict(dict(max_requests=2, num_pages=9, spec=spec, device=DEV), **bad))
    run = Run(2, 20, 4, 100)
    for bad, message in ((dict(dtype=torch.float32), "float16 or bfloat16"), (dict(head_dim=32), "head_dim"), (dict(heads=0), "heads")):
        with pytest.raises(ValueError, match=message):
            PagedKVCache(**dict(dict(table=run.table, heads=2, head_dim=64), **bad))
    t = run.table
    for call, message in ((lambda: t.extend(_ints([1, 1, 1]), 3), r"\[2\]"), (lambda: t.extend(torch.ones(2, device=DEV), 2), "int32"),
                          (lambda: t.extend(torch.ones(2, dtype=torch.int32), 2), "live on"), (lambda: t.extend(_ints([1, 1]), -1), "rows"),
                          (lambda: t.extend(_ints([1, 1]), 2, max_count=-1), "max_count"),
                          (lambda: t.extend(_ints([1, 1]), 2, parents=_ints([0])), r"\[2\]"),
                          (lambda: t.extend(_ints([300, 1]), 301, parents=_ints([0] * 301)), "256"),
                          (lambda: t.release(_ints([1, 0])), "bool")):
        with pytest.raises(ValueError, match=message):
            call()
    assert t.check() == 20 and t.lengths.tolist() == [0, 0]
    batch = run.extend([2, 1])
    other = PageTable(2, 20, spec, device=DEV).extend(_ints([2, 1]), 3)
    q, k, v = run.normal(3, 4), run.normal(3, 2), run.normal(3, 2)
    c, rope = run.cache, MultiAxisRotary(64, (32,))
    for call, message in ((lambda: c.append(k, v, other), "another table"), (lambda: c.append(k[:2], v, batch), r"\[3, 2, 64\]"),
                          (lambda: c.append(k, v.half(), batch), "bfloat16"), (lambda: c.append(k, q, batch), r"\[3, 2, 64\]"),
                          (lambda: c.attend(q[:, :3], batch), "multiple of 2"), (lambda: c.attend(q.cpu(), batch), "live on"),
                          (lambda: c.attend(q, batch, math.nan), "finite"), (lambda: c.attend(q, other), "another table"),
                          (lambda: c.append_rotated(q, k, v, batch, MultiAxisRotary(128, (64,))), "head_dim"),
                          (lambda: c.append_rotated(q, k, v, batch, rope, batch.positions[:2]), "positions"),
                          (lambda: c.append_rotated(q, k, v, other, rope), "another table"),
                          (lambda: c.accept(batch, _ints([0, 1]), _ints([1, 1])), "paths"),
                          (lambda: c.accept(batch, _ints([[0], [1]]), _ints([1])), "accepted"),
                          (lambda: t.accept(other, _ints([1, 1])), "another table")):
        with pytest.raises(ValueError, match=message):
            call()


@pytest.mark.gpu
def test_no_rows():
    run = Run(2, 20, 4, 100)
    run.grow([5, 0])
    batch = run.extend([0, 0])
    run.cache.append(run.normal(0, 2), run.normal(0, 2), batch)
    assert run.cache.attend(run.normal(0, 4), batch).shape == (0, 4, 64)
    run.check_tables(batch)
    batch = run.extend([0, 0], parents=[[], []])
    assert run.cache.attend(run.normal(0, 4), batch).shape == (0, 4, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("counts,tree", [([1, 1, 1], False), ([1, 200, 40], False), ([5, 9, 1], True)])
def test_graph_of_a_step_and_side_streams(counts, tree):
    """A captured step (tables, rows, attention, path) replayed between eager ones follows
    the lengths, like the same steps run eagerly; two graphs run in turn."""
    rng = random.Random(14)
    trees = [_tree(rng, n) for n in counts] if tree else None
    chain = [op.chains(t)[-1] for t in trees] if tree else [list(range(n)) for n in counts]
    most = max(map(len, chain))
    a, b = (Run(3, 200, 4, 60, 16, seed=15) for _ in range(2))
    for run in (a, b):
        run.grow([50, 0, 129])
    n, accepted = sum(counts), _ints([len(c) for c in chain])
    count, paths = _ints(counts), _ints([c + [0] * (most - len(c)) for c in chain])
    up = _ints([p for t in trees for p in t]) if tree else None
    q, k, v = a.normal(n, 4), a.normal(n, 2), a.normal(n, 2)

    def step(run):
        batch = run.table.extend(count, n, max_count=max(counts), parents=up)
        run.cache.append(k, v, batch)
        o = run.cache.attend(q, batch)
        run.cache.accept(batch, paths, accepted)
        run.table.accept(batch, accepted)
        return o

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one = step(a)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(one, step(b))
    graphs = []
    for _ in range(2):
        graphs.append((torch.cuda.CUDAGraph(), None))
        with torch.cuda.graph(graphs[-1][0]):
            graphs[-1] = (graphs[-1][0], step(a))
    for i in range(6):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=a.gen, device=DEV))
        graph, out = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        want = step(b)
        assert torch.equal(out, want), i
        assert torch.equal(a.table.lengths, b.table.lengths) and torch.equal(a.table.block_table, b.table.block_table)
        if i == 3:
            for run in (a, b):
                run.table.release(_ints([True, False, False], torch.bool))
    assert a.table.check() == b.table.check()


@pytest.mark.gpu
def test_the_operators_together():
    """A decoder layer's requests served: prompts in chunks, single tokens, drafts that are
    verified, new requests in the place of finished ones; keys turned by text positions, an
    encoder's states attended after."""
    rng, D = random.Random(16), 64
    run = Run(4, 80, 4, 90, 16, 2, D, torch.bfloat16, seed=16)
    rope = MultiAxisRotary(D, (16, 16))
    ek, ev = (torch.randn(1, 2, 50, D, generator=run.gen, device=DEV).to(run.dtype) for _ in range(2))

    def serve(counts, parents=None, tag=""):
        batch = run.extend(counts, max_count=max(counts), parents=parents)
        q, k, v = (run.normal(batch.rows, n) for n in (8, 2, 2))
        turned_q, turned_k = rope(q, k, batch.positions)
        got = run.cache.append_rotated(q, k, v, batch, rope)
        assert torch.equal(got, turned_q), tag
        run.hold(turned_k, v)
        o = run.cache.attend(got, batch)
        run.check_tables(batch)
        run.check_attend(batch, got, o, tag=tag)
        x = cross_attention(o.transpose(0, 1)[None], ek, ev, enable_gqa=True)
        assert torch.isfinite(x).all() and x.shape == (1, 8, batch.rows, D)
        return batch

    serve([100, 1, 30, 0], tag="prompts")
    serve([70, 1, 1, 200], tag="chunks beside tokens")
    for i in range(5):
        serve([1, 1, 1, 1], tag=f"tokens {i}")
        counts = [12, 7, 1, 20]
        trees = [_tree(rng, n) for n in counts]
        batch = serve(counts, trees, tag=f"drafts {i}")
        paths = [rng.choice(op.chains(t)) for t in trees]
        most = max(map(len, paths))
        accepted = _ints([len(p) for p in paths])
        run.cache.accept(batch, _ints([p + [0] * (most - len(p)) for p in paths]), accepted)
        run.table.accept(batch, accepted)
        for r, p in enumerate(paths):
            for held in (run.k, run.v):
                held[r] = torch.cat([held[r][:run.base[r]], held[r][[run.base[r] + j for j in p]]])
            run.book.length[r] = run.base[r] + len(p)
        if i == 2:
            done = [False, True, False, True]
            run.table.release(_ints(done, torch.bool))
            run.book.release(done)
            for r in (1, 3):
                run.k[r], run.v[r] = run.k[r][:0], run.v[r][:0]
            serve([1, 40, 1, 9], tag="new requests")
