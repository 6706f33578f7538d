"""Pages of a paged cache: copied, forked, given back, moved together.  Everything here is a copy or a
whole number: results are equal to a plain restatement."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC

pytestmark = pytest.mark.gpu

# rows [kv_heads, head_dim], page size: 16-byte rows, rows of other sizes, pages over several workgroups
SHAPES = [((4, 128), 256), ((2, 64), 16), ((3, 37), 5), ((1, 1), 1), ((2, 3), 7)]


def make_caches(gpu, n, pages, row, page, dt, seed=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(n):
        x = torch.randint(-100, 100, (pages * page, *row), generator=g).to(dt).to(gpu)
        raw = torch.empty(x.numel() + offset, dtype=dt, device=gpu)
        out.append(raw[offset:].view(x.shape).copy_(x))
    return out


def host(caches, pages):
    return [c.view(pages, -1).cpu().clone() for c in caches]


def same(caches, want, pages):
    for c, w in zip(caches, want):
        assert torch.equal(c.view(pages, -1).cpu(), w)


@pytest.mark.parametrize("dt", LC.DTYPES + [torch.int8], ids=LC.DT_IDS + ["i8"])
@pytest.mark.parametrize("row,page", SHAPES)
@pytest.mark.parametrize("n", [1, 7, 300])
def test_copy_pages(gpu, dt, row, page, n):
    pages = 2 * n + 3
    if pages * page * row[0] * row[1] > 1 << 24:
        row = (row[0], row[1] // 8)
    for offset in (0, 1):
        caches = make_caches(gpu, 3, pages, row, page, dt, n, offset)
        want = host(caches, pages)
        r = np.random.default_rng(n)
        p = r.permutation(pages)
        src, dst = p[:n], p[n:2 * n]
        src[n // 2:] = src[:n - n // 2]  # one page to several places
        for w in want:
            w[dst] = w[src]
        print(f"[case] copy {n} pages of {page} x {row} {dt} offset {offset}", flush=True)
        ops.copy_pages(caches, src, dst, page)
        same(caches, want, pages)
    ops.copy_pages(caches, [], [], page)
    ops.copy_pages([], [0], [1], page)
    same(caches, want, pages)


def test_copy_pages_of_many_caches(gpu):
    """More caches than one launch's arguments hold."""
    caches = make_caches(gpu, 150, 6, (2, 8), 4, torch.float16)
    want = host(caches, 6)
    for w in want:
        w[[5, 0]] = w[[2, 3]]
    ops.copy_pages(caches, [2, 3], [5, 0], 4)
    same(caches, want, 6)


class Pool:
    """The plain restatement: tables, counts, lengths and pages on the host."""

    def __init__(self, seed, rows, cols, pages, page, live):
        r = np.random.default_rng(seed)
        self.page, self.pages = page, pages
        self.table = np.full((rows, cols), -1, np.int32)
        self.ref = np.zeros(pages, np.int32)
        self.key_len = np.zeros(rows, np.int32)
        free = list(r.permutation(pages))
        for s, n in live.items():
            used = [free.pop() for _ in range(-(-n // page))]
            self.table[s, :len(used)] = used
            self.ref[used] += 1
            self.key_len[s] = n

    def gpu(self, device):
        return [torch.from_numpy(x.copy()).to(device) for x in (self.table, self.key_len, self.ref)]

    def fork(self, parent, child, caches):
        free = list(np.flatnonzero(self.ref == 0))
        new = []
        for p, c in zip(parent, child):
            n = int(self.key_len[p])
            full, rest = divmod(n, self.page)
            self.table[c] = -1
            self.table[c, :full] = self.table[p, :full]
            self.ref[self.table[p, :full]] += 1
            self.key_len[c] = n
            page = -1
            if rest and free:
                page = int(free.pop(0))
                self.table[c, full] = page
                self.ref[page] = 1
                for x in caches:
                    x = x.view(self.pages, self.page, -1)
                    x[page, :rest] = x[int(self.table[p, full]), :rest]
            elif rest:
                page, self.key_len[c] = -2, full * self.page
            new.append(page)
        return new

    def free(self, seqs, window=None, sinks=0):
        for s in seqs:
            for b in range(self.table.shape[1]):
                keys = np.arange(b * self.page, (b + 1) * self.page)
                if window is not None and ((keys < sinks) | (keys >= int(self.key_len[s]) + 1 - window)).any():
                    continue
                if self.table[s, b] >= 0:
                    self.ref[self.table[s, b]] -= 1
                self.table[s, b] = -1
            if window is None:
                self.key_len[s] = 0

    def check(self, t):
        for name, got, want in zip(("tables", "key_len", "ref_count"), t, (self.table, self.key_len, self.ref)):
            assert np.array_equal(got.cpu().numpy(), want), name


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("row,page", SHAPES)
def test_fork_and_free(gpu, dt, row, page):
    lens = {0: 3 * page + page // 2, 5: 2 * page, 2: 1, 7: 0}
    pool = Pool(3, 40, 6, 40, page, lens)
    caches = make_caches(gpu, 4, 40, row, page, dt)
    want, t = host(caches, 40), pool.gpu(gpu)
    parent, child = [0, 0, 5, 2, 7, 0], [10, 11, 12, 39, 14, 15]
    new = ops.fork_pages(caches, t[0], t[1], t[2], parent, child, page)
    assert new.tolist() == pool.fork(parent, child, want)
    pool.check(t)
    same(caches, want, 40)
    # a child becomes a parent, and the first parent ends
    new = ops.fork_pages(caches, t[0], t[1], t[2], [11], [20], page)
    assert new.tolist() == pool.fork([11], [20], want)
    ops.free_pages(t[0], t[1], t[2], [0, 12, 30], page)
    pool.free([0, 12, 30])
    pool.check(t)
    same(caches, want, 40)
    ops.free_pages(t[0], t[1], t[2], list(range(40)), page)
    pool.free(range(40))
    pool.check(t)
    assert not t[2].any()


def test_fork_when_pages_run_out(gpu):
    pool = Pool(4, 12, 4, 7, 16, {0: 40, 1: 32})
    caches = make_caches(gpu, 2, 7, (2, 64), 16, torch.float16)
    want, t = host(caches, 7), pool.gpu(gpu)
    new = ops.fork_pages(caches, *t, [0, 1, 0, 0], [2, 3, 4, 5], 16)
    assert new.tolist() == pool.fork([0, 1, 0, 0], [2, 3, 4, 5], want) and new.tolist()[1:] == [-1, 6, -2] \
        or new.tolist().count(-2) == 1
    pool.check(t)
    same(caches, want, 7)
    assert t[1][5] == 32  # the child without a page ends with the full ones


@pytest.mark.parametrize("pages", [1, 15, 16, 17, 1000, 16384, 16385, 40000])
def test_forks_take_the_lowest_free_pages(gpu, pages):
    """Scans of every length; more forks than one launch's arguments hold."""
    r = np.random.default_rng(pages)
    ref = (r.random(pages) < 0.97).astype(np.int32)
    table = np.full((602, 3), -1, np.int32)
    table[0, 0] = int(np.flatnonzero(ref)[0]) if ref.any() else -1
    key_len = np.zeros(602, np.int32)
    key_len[0] = 1
    free = np.flatnonzero(ref == 0)
    d = [torch.from_numpy(x.copy()).to(gpu) for x in (table, key_len, ref)]
    n = 600
    new = ops.fork_pages([torch.zeros(pages * 2, 4, dtype=torch.float16, device=gpu)], *d, [0] * n,
                         list(range(1, n + 1)), 2).cpu().numpy()
    k = min(n, len(free))
    assert np.array_equal(new[:k], free[:k]) and (new[k:] == -2).all()
    assert int(d[2].sum()) == int(ref.sum()) + k
    assert np.array_equal(d[0].cpu().numpy()[1:k + 1, 0], free[:k])


def test_shared_pages_are_given_back_once_each(gpu):
    """64 sequences over one set of pages, all freed in one call; a count that is already 0 stays 0."""
    table = np.tile(np.arange(8, dtype=np.int32), (64, 1))
    table[3, 2] = 9
    ref = np.array([64] * 8 + [0, 0, 5], np.int32)
    ref[2] = 63
    d = [torch.from_numpy(x).to(gpu) for x in (table, np.full(64, 100, np.int32), ref)]
    ops.free_pages(*d, list(range(64)), 16)
    assert (d[0] == -1).all() and not d[1].any()
    assert d[2].tolist() == [0] * 10 + [5]


@pytest.mark.parametrize("page", [1, 5, 16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 4), (17, 16), (40, 33), (1 << 40, 0), (7, 1 << 40)])
def test_free_outside_a_window(gpu, page, window, sinks):
    pool = Pool(6, 5, 130, 400, page, {0: 100, 1: 33, 2: 16, 3: 1})
    t = pool.gpu(gpu)
    ops.free_pages(*t, [0, 1, 2, 3, 4], page, window=window, sinks=sinks)
    pool.free([0, 1, 2, 3, 4], window, sinks)
    pool.check(t)


def test_bad_table_entries_are_left_alone(gpu):
    """Entries outside the cache: not shared, not counted, -1 afterwards."""
    table = np.array([[0, 99, -5, 1], [-1] * 4], np.int32)
    d = [torch.from_numpy(x) .to(gpu) for x in (table, np.array([14, 0], np.int32), np.array([1, 1, 0], np.int32))]
    cache = torch.randn(3 * 4, 8, device=gpu)
    before = cache.clone()
    new = ops.fork_pages([cache], *d, [0], [1], 4)
    assert new.tolist() == [2] and d[0][1].tolist() == [0, -1, -1, 2] and d[2].tolist() == [2, 1, 1]
    before[8:10] = before[4:6]
    assert torch.equal(cache, before)
    ops.free_pages(*d, [0], 4)
    assert d[0][0].tolist() == [-1] * 4 and d[2].tolist() == [1, 0, 1]
    d[1][0] = -7  # a length below zero: a child without pages
    assert ops.fork_pages([cache], *d, [0], [1], 4).tolist() == [-1] and d[0][1].tolist() == [-1] * 4


def plain_compact(table, ref, pages):
    used = int((ref > 0).sum())
    src = [p for p in range(used, pages) if ref[p] > 0]
    dst = [p for p in range(used) if ref[p] <= 0]
    place = {p: p for p in range(pages) if ref[p] > 0}
    place.update(zip(src, dst))
    t = np.vectorize(lambda e: place.get(int(e), -1), otypes=[np.int32])(table)
    out = np.maximum(ref, 0) * 0 + ref
    out[dst] = ref[src]
    out[src] = 0
    return t, out, src, dst


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("row,page", SHAPES)
@pytest.mark.parametrize("share", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("in_place", [True, False])
def test_compact_pages(gpu, dt, row, page, share, in_place):
    pages = 61
    r = np.random.default_rng(int(100 * share))
    ref = (r.random(pages) < share) * r.integers(1, 4, pages)
    ref = ref.astype(np.int32)
    table = r.integers(-2, pages + 3, (7, 9)).astype(np.int32)  # stale and bad entries among them
    caches = make_caches(gpu, 3, pages, row, page, dt)
    want = host(caches, pages)
    t, out, src, dst = plain_compact(table, ref, pages)
    for w in want:
        w[dst] = w[src]
    dt_, dr = torch.from_numpy(table).to(gpu), torch.from_numpy(ref).to(gpu)
    to, ro = (None, None) if in_place else (torch.full_like(dt_, 77), torch.full_like(dr, 77))
    moved = ops.compact_pages(caches, dt_, dr, page, to, ro)
    assert moved.tolist() == [len(src)]
    to, ro = (dt_, dr) if in_place else (to, ro)
    assert np.array_equal(to.cpu().numpy(), t) and np.array_equal(ro.cpu().numpy(), out)
    if not in_place:
        assert np.array_equal(dt_.cpu().numpy(), table) and np.array_equal(dr.cpu().numpy(), ref)
    same(caches, want, pages)
    again = ops.compact_pages(caches, to, ro, page)
    assert again.tolist() == [0]
    same(caches, want, pages)


@pytest.mark.parametrize("pages", [1, 16, 17, 16384, 16400, 50001])
def test_compact_scans_of_every_length(gpu, pages):
    r = np.random.default_rng(pages)
    ref = (r.random(pages) < 0.4).astype(np.int32)
    table = r.integers(0, pages, (3, 11)).astype(np.int32)
    t, out, src, dst = plain_compact(table, ref, pages)
    cache = torch.arange(pages, device=gpu, dtype=torch.float32)[:, None].repeat(1, 4)
    want = cache.cpu().clone()
    want[dst] = want[src]
    d = [torch.from_numpy(x).to(gpu) for x in (table, ref)]
    assert ops.compact_pages([cache], *d, 1).tolist() == [len(src)]
    assert torch.equal(cache.cpu(), want)
    assert np.array_equal(d[0].cpu().numpy(), t) and np.array_equal(d[1].cpu().numpy(), out)


def test_captured_fork_and_free(gpu):
    """A captured fork and release, replayed with eager work between; the parent grows meanwhile."""
    pool = Pool(8, 6, 6, 20, 16, {0: 40, 1: 17})
    caches = make_caches(gpu, 2, 20, (2, 64), 16, torch.bfloat16)
    t = pool.gpu(gpu)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        new = ops.fork_pages(caches, *t, [0, 1], [2, 3], 16)
        kept = t[0].clone()
        ops.free_pages(*t, [2, 3], 16)
    for n in (40, 41, 47, 48):
        t[1][0] = n
        pool.key_len[0] = n
        want = host(caches, 20)
        expected = pool.fork([0, 1], [2, 3], want)
        g.replay()
        torch.cuda.synchronize()
        assert new.tolist() == expected and np.array_equal(kept.cpu().numpy(), pool.table)
        same(caches, want, 20)
        pool.free([2, 3])
        pool.check(t)
