"""styx_op_kv_plan (no counterpart in the reference) against its definition,
sequence by sequence, through the C ABI.  Whole numbers: equal."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from styx_amd import _lib as L

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


class Plan:
    def __init__(self, page, n_pages, table_len, table, held, free, n_free, lens, new, pos=None, shared=None, n_rows=None):
        i32 = lambda x: np.array(x, np.int32)  # noqa: E731
        self.page, self.n_pages, self.table_len, self.B = page, n_pages, table_len, len(lens)
        self.table, self.held = i32(table).reshape(self.B, table_len), i32(held)
        self.free = np.full(n_pages, -9, np.int32)
        self.free[:len(free)] = free
        self.n_free, self.lens, self.new = n_free, i32(lens), i32(new)
        self.pos = i32(range(100, 100 + self.B) if pos is None else pos)
        self.shared = None if shared is None else i32(shared)
        self.n_rows = int(np.maximum(self.new, 0).astype(np.int64).sum()) if n_rows is None else n_rows

    def want(self, in_place):
        table, page, cap = self.table.copy(), self.page, self.table_len * self.page
        blank = lambda x: x.copy() if in_place else np.full_like(x, 77)  # noqa: E731
        out_table, free_out = blank(self.table), blank(self.free)
        n_free = min(max(self.n_free, 0), self.n_pages)
        stack = self.free[:n_free].tolist()
        held = [min(max(int(h), 0), self.table_len) for h in self.held]
        first, before, ok, need = [], 0, [], []
        for b in range(self.B):
            n, m = int(self.lens[b]), max(0, int(self.new[b]))
            first.append(min(before, 2 ** 31 - 1))
            ok.append(n >= 0 and n + m <= cap and before + m <= self.n_rows)
            need.append(held[b] if n > cap else -(-(max(n, 0) + (m if ok[b] else 0)) // page) if n >= 0 else 0)
            before += m
        stays, count = [], []
        for b in range(self.B):
            keep = min(held[b], max(need[b], int(self.shared[b]) if self.shared is not None else 0))
            for e in range(keep, held[b]):
                if 0 <= table[b, e] < self.n_pages and len(stack) < self.n_pages:
                    stack.append(int(table[b, e]))
                out_table[b, e] = -1
            stays.append(keep)
            out_table[b, :keep] = table[b, :keep]
        top, closed, held_out = len(stack), False, []
        for b in range(self.B):
            m = max(0, int(self.new[b])) if ok[b] else 0
            asks = max(0, need[b] - held[b]) if m > 0 else 0
            if asks > 0 and (closed or asks > len(stack)):
                closed, m, asks = True, 0, 0
            for e in range(held[b], held[b] + asks):
                out_table[b, e] = stack.pop()
            held_out.append(stays[b] + asks)
            count.append(m)
        free_out[:len(stack)] = stack
        free_out[len(stack):top] = -1
        rows = np.full((3, self.n_rows), -1, np.int32)
        for b in range(self.B):
            for i in range(count[b]):
                t = int(self.lens[b]) + i
                e = int(out_table[b, t // page])
                rows[:, first[b] + i] = b, self.pos[b] + i, e * page + t % page if 0 <= e < self.n_pages else -1
        return dict(table=out_table, held=np.array(held_out), free=free_out, n_free=np.array([len(stack)]),
                    first=np.array(first), count=np.array(count), seq=rows[0], pos=rows[1], at=rows[2])

    def run(self, gpu, in_place, maps=(True, True, True)):
        up = gpu.from_numpy
        ins = [up(x) for x in (self.table, self.held, self.free, np.array([self.n_free], np.int32))]
        outs = ins if in_place else [up(np.full_like(x, 77)) for x in (self.table, self.held, self.free, np.zeros(1, np.int32))]
        L_, N_, P_ = up(self.lens), up(self.new), up(self.pos)
        sh = up(self.shared) if self.shared is not None else None
        seq = [up(np.full(self.B, 55, np.int32)) for _ in range(2)]
        rows = [up(np.full(max(self.n_rows, 1), 55, np.int32)) for _ in range(3)]
        kv = L.KvCache(L.F32, self.B, 1, 64, self.page, self.n_pages, self.table_len, None, None, None)
        pages = [L.KvPages(*(b.ptr for b in x)) for x in (ins, outs)]
        L.check(gpu.lib.styx_op_kv_plan(
            gpu.h, C.byref(kv), C.byref(pages[0]), C.byref(pages[1]), sh.ptr if sh else None, L_.ptr, N_.ptr, P_.ptr,
            self.n_rows, seq[0].ptr, seq[1].ptr, *(r.ptr if m else None for r, m in zip(rows, maps))))
        gpu.sync()
        i32 = lambda b, n: b.download(np.int32, n)  # noqa: E731
        got = dict(table=i32(outs[0], self.table.size).reshape(self.table.shape), held=i32(outs[1], self.B),
                   free=i32(outs[2], self.n_pages), n_free=i32(outs[3], 1), first=i32(seq[0], self.B), count=i32(seq[1], self.B))
        for name, r, m in zip(("seq", "pos", "at"), rows, maps):
            got[name] = i32(r, self.n_rows) if m else None
        return got

    def check(self, gpu):
        for in_place in (False, True):
            want, got = self.want(in_place), self.run(gpu, in_place)
            for k in want:
                assert np.array_equal(got[k], want[k]), (in_place, k, got[k], want[k])
        return want


def ordinary(rng, B, page, table_len, most, spare, ended=0.1, cut=0.2, shared=True):
    cap = table_len * page
    lens = rng.integers(0, cap // 2 + 1, B)
    held = -(-lens // page)
    lens = np.where(rng.random(B) < cut, (lens * rng.random(B)).astype(int), lens)
    new = np.minimum(rng.integers(0, most + 1, B), cap - lens)
    gone = rng.random(B) < ended
    lens[gone], new[gone] = -1, 0
    n_pages = int(held.sum()) + spare
    perm = rng.permutation(n_pages)
    table = np.full((B, table_len), -1)
    at = 0
    for b in range(B):
        table[b, :held[b]] = perm[at:at + held[b]]
        at += held[b]
    own = np.where(rng.random(B) < 0.3, (held * rng.random(B)).astype(int), 0) if shared else None
    return Plan(page, n_pages, table_len, table, held, perm[at:], spare, lens, new, shared=own)


@pytest.mark.parametrize("B", [1, 2, 63, 64, 65, 300, 1024, 1025, 2500])
@pytest.mark.parametrize("most", [1, 70])
def test_ordinary_steps(gpu, B, most):
    rng = np.random.default_rng(B + most)
    p = ordinary(rng, B, 16, 12, most, 6 * B + 5)
    assert p.check(gpu)["count"].sum() > 0 or B < 3


@pytest.mark.parametrize("page", [1, 7, 16, 100, 512])
def test_page_sizes(gpu, page):
    ordinary(np.random.default_rng(page), 40, page, 9, 3 * page + 1, 200, shared=False).check(gpu)


@pytest.mark.parametrize("spare", [0, 1, 5, 20])
@pytest.mark.parametrize("B", [10, 1500])
def test_not_enough_pages(gpu, spare, B):
    """The first that cannot be served and all after it that ask for pages get none; what comes back is handed on."""
    rng = np.random.default_rng(spare + B)
    p = ordinary(rng, B, 4, 20, 30, spare, ended=0.05, cut=0.05)
    want = p.check(gpu)
    assert (want["count"] < np.maximum(p.new, 0)).any()


def test_a_long_step_of_prompts(gpu):
    p = Plan(16, 4000, 600, np.full((5, 600), -1), [0] * 5, np.arange(4000), 4000, [0] * 5, [9000, 1, 0, 5003, 17])
    want = p.check(gpu)
    assert want["count"].tolist() == [9000, 1, 0, 5003, 17]


@pytest.mark.parametrize("wrong", [0.0, 0.3])
@pytest.mark.parametrize("sizes", [[40000, 0, 3, 1], [17, 16, 15, 0, 33, 20001, 5, 9000], [31] * 900 + [700] * 40])
def test_many_pages_change_hands(gpu, sizes, wrong):
    """Ended sequences' pages, entries outside the pool among them, come back and go to as many that begin."""
    rng = np.random.default_rng(len(sizes))
    ended, T = len(sizes), max(sizes)
    B = 2 * ended
    held = np.zeros(B, int)
    held[::2] = sizes
    n_pages = int(held.sum()) + 9
    table = np.full((B, T), -1)
    pages, at = rng.permutation(n_pages), 0
    for b in range(0, B, 2):
        table[b, :held[b]] = pages[at:at + held[b]]
        at += held[b]
    table[rng.random(table.shape) < wrong] = n_pages
    lens, new = np.where(np.arange(B) % 2 == 0, -1, 0), np.zeros(B, int)
    new[1::2] = [2 * n - (n % 3 == 1) for n in sizes[::-1]]
    want = Plan(2, n_pages, T, table, held, pages[at:], 9, lens, new).check(gpu)
    assert (want["count"][1::2] == new[1::2]).all() == (wrong == 0)


def test_what_does_not_fit_is_refused(gpu):
    """Slots past cap, rows past n_rows, lengths past cap, and impossible numbers of pages."""
    big = 2 ** 31 - 1
    B, T = 9, 4
    table = np.arange(B * T).reshape(B, T)
    lens = [8, 8, 33, 32, 0, -5, big, 10, 10]
    new = [2, 30, 4, 0, -7, 3, big, big, 4]
    held = [1, 1, 4, 9, -3, 2, 4, 2, 2]
    for n_rows in (0, 1, 40, 50):
        Plan(8, 64, T, table, held, range(36, 60), 24, lens, new, shared=[0, -4, 1, 2, 1, 1, 0, 9, 0], n_rows=n_rows).check(gpu)
    for n_free in (-4, 90):
        Plan(8, 64, T, table, held, range(64), n_free, lens, new, n_rows=50).check(gpu)


def test_entries_outside_the_pool_and_a_full_stack(gpu):
    table = [[0, -1, 70, 3], [5, 64, 6, -9], [8, 9, 10, 11]]
    Plan(8, 64, 4, table, [4, 4, 4], range(20, 40), 20, [3, -1, 25], [1, 0, 3]).check(gpu)
    # more entries come back than there are places
    Plan(8, 12, 4, [[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11]], [4, 4, 4], range(10), 10, [3, -1, 25], [1, 0, 3]).check(gpu)
    # the entry of a new row is not one of the pool's
    want = Plan(8, 64, 4, table, [4, 4, 4], range(20, 40), 20, [9, 9, 9], [2, 2, 2]).check(gpu)
    assert want["at"].tolist()[:4] == [-1] * 4


def test_maps_that_are_not_asked_for(gpu):
    p = ordinary(np.random.default_rng(5), 30, 16, 8, 20, 100)
    want = p.want(True)
    for maps in [(False, False, False), (True, False, False), (False, True, False), (False, False, True)]:
        got = p.run(gpu, True, maps)
        assert all(got[k] is None or np.array_equal(got[k], want[k]) for k in want)


def test_refusals(gpu):
    z = gpu.zeros(4096)
    a = [z.ptr + 256 * i for i in range(12)]
    kv = L.KvCache(L.F32, 2, 1, 64, 8, 4, 4, None, None, None)
    ins, outs = L.KvPages(*a[:4]), L.KvPages(*a[4:8])

    def call(kv=kv, i=ins, o=outs, n=1, len_=a[8], new=a[9], pos=a[10], first=a[11], count=a[11] + 64, at=a[11] + 128):
        return gpu.lib.styx_op_kv_plan(gpu.h, C.byref(kv) if kv else None, C.byref(i) if i else None, C.byref(o) if o else None,
                                       None, len_, new, pos, n, first, count, None, at, at)

    assert call() == 0 and call(o=ins) == 0 and call(n=0) == 0
    for b in [dict(kv=None), dict(i=None), dict(o=None), dict(i=L.KvPages(None, *a[1:4])), dict(o=L.KvPages(*a[4:7], None)),
              dict(o=L.KvPages(a[0], *a[5:8])), dict(o=L.KvPages(*a[0:3], a[7])), dict(n=-1), dict(len_=None), dict(new=None),
              dict(pos=None), dict(first=None), dict(count=None), dict(kv=L.KvCache(L.F32, 0, 1, 64, 8, 4, 4, None, None, None)),
              dict(kv=L.KvCache(L.F32, 2, 1, 64, 0, 4, 4, None, None, None)),
              dict(kv=L.KvCache(L.F32, 2, 1, 64, 1 << 16, 1 << 16, 4, None, None, None)),
              dict(kv=L.KvCache(L.F32, 3, 1, 64, 1, 4, 1 << 30, None, None, None))]:
        assert call(**b) == -1, b
    gpu.sync()
