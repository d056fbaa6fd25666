"""styx_op_kv_weigh (no counterpart in the reference) against its definition in
64 bits, through the C ABI.

Tolerance of a slot: each weight e^(s - lse) has the score's error ds, those of
the scale and the difference (2 E (|s| + |lse|)) and of the exponential (8 E),
relative; m of them added: m E more; the decayed value two roundings."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from chunk_cases import E, Chunked
from styx_amd import _lib as L

pytestmark = pytest.mark.gpu

TYPES = {"f32": (False, False), "f16": (True, True), "mixed": (True, False)}


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


def lse_of(c):
    """What attention would have left, rounded to f32."""
    lse = np.full((c.n_rows, c.nh), 3.25, np.float32)
    for b in range(c.B):
        if c.taken(b):
            for i in range(int(c.counts[b])):
                for j in range(c.nkv):
                    with np.errstate(invalid="ignore"):
                        lse[c.first[b] + i, j * c.gqa:(j + 1) * c.gqa] = c.attend(b, i, j)[2]
    return lse


def run(gpu, c, lse, last, decay=0.9, with_acc=True, in_place=False, with_pos=True, seed=0):
    rng = np.random.default_rng(seed)
    kv, ch, q = c.buffers(gpu)
    shape = (c.B, c.nkv, c.cap)
    acc = np.exp(rng.standard_normal(shape)).astype(np.float32)
    where = rng.integers(0, 1000, shape).astype(np.int32)
    pos = rng.integers(0, 5000, c.B).astype(np.int32)
    a, w, p, l = (gpu.from_numpy(x) for x in (acc, where, pos, lse))
    before = acc if in_place else np.full(shape, -3.0, np.float32)
    o = a if in_place else gpu.from_numpy(before)
    L.check(gpu.lib.styx_op_kv_weigh(
        gpu.h, C.byref(kv), C.byref(ch), p.ptr if with_pos else None, c.nh, L.F16 if c.q16 else L.F32, q.ptr, c.ld, c.scale,
        c.window, l.ptr, last, decay, a.ptr if with_acc else None, o.ptr, w.ptr if with_pos else None))
    gpu.sync()
    return acc, where, pos, before, o.download(np.float32).reshape(shape), w.download(np.int32).reshape(shape)


def check(c, lse, last, got, decay=0.9, with_acc=True, with_pos=True):
    acc, where, pos, before, out, where_out = got
    want_where, want, tol = where.copy(), before.astype(np.float64), np.zeros(out.shape)
    for b in range(c.B):
        if not c.taken(b):
            continue
        n, m, rows = int(c.lens[b]), int(c.counts[b]), c.rows(b)
        for j in range(c.nkv):
            s = np.zeros(n + m)
            t = np.zeros(n + m)
            for i in range(max(0, m - last), m):
                x, ds, see = c.scores(b, i, j, rows)
                le = lse[c.first[b] + i, j * c.gqa:(j + 1) * c.gqa, None].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    w = np.where(np.isneginf(le), 0.0, np.exp(x - le))
                    t[see] += (w * (ds + (2 * np.abs(x) + 2 * np.abs(le) + 8 + last * c.gqa) * E)).sum(0)
                s[see] += w.sum(0)
            if with_acc:
                s[:n] += decay * acc[b, j, :n].astype(np.float64)
                t[:n] += 2 * E * decay * acc[b, j, :n]
            want[b, j, :n + m] = s
            tol[b, j, :n + m] = t + 2 * E * np.abs(s) + 1e-37
            if with_pos:
                want_where[b, j, n:n + m] = pos[b] + np.arange(m)
    assert np.array_equal(where_out, want_where)
    d = np.abs(out - want)
    ok = (d <= tol) | (np.isnan(want) & np.isnan(out))
    assert ok.all(), (np.argwhere(~ok)[:5], out[~ok][:5], want[~ok][:5])


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gqa", [1, 3, 8, 16])
def test_ragged_batch(gpu, types, hd, gqa):
    c = Chunked(np.random.default_rng(hd + gqa), *TYPES[types], [0, 0, 5, -1, 130, 63, 300], [1, 37, 1, 4, 66, 2, 17], 2, gqa,
                hd, 16)
    lse = lse_of(c)
    check(c, lse, 8, run(gpu, c, lse, 8))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("last", [0, 1, 5, 64, 1000, 2 ** 31 - 1])
def test_how_many_tokens_count(gpu, types, last):
    c = Chunked(np.random.default_rng(1), *TYPES[types], [33, 500], [100, 70], 1, 4, 64, 48)
    lse = lse_of(c)
    check(c, lse, min(last, 200), run(gpu, c, lse, last))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("window", [1, 40, 100, 2 ** 31 - 1])
def test_window(gpu, types, window):
    c = Chunked(np.random.default_rng(2), *TYPES[types], [33, 500], [100, 70], 1, 4, 64, 100, window=window)
    lse = lse_of(c)
    check(c, lse, 90, run(gpu, c, lse, 90))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_in_place_without_weights_and_without_positions(gpu, types):
    c = Chunked(np.random.default_rng(3), *TYPES[types], [20, 3000], [9, 1], 2, 2, 128, 64)
    lse = lse_of(c)
    check(c, lse, 4, run(gpu, c, lse, 4, in_place=True))
    check(c, lse, 4, run(gpu, c, lse, 4, with_acc=False), with_acc=False)
    check(c, lse, 4, run(gpu, c, lse, 4, with_pos=False), with_pos=False)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_missing_pages_skipped_sequences_and_gaps(gpu, types):
    c = Chunked(np.random.default_rng(4), *TYPES[types], [90, 0, 10, -1], [20, 40, 4, 2], 1, 4, 64, 16, first=[40, 0, 62, 61],
                n_rows=64, ld=4 * 64 + 40)
    assert not c.taken(2)
    c.table[0, [0, 3]] = -1
    c.table[1, :2] = c.n_pages
    lse = lse_of(c)
    assert np.isneginf(lse[0]).all()  # a token that sees nothing
    check(c, lse, 100, run(gpu, c, lse, 100))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_not_finite(gpu, types):
    """NaN behind the last row changes nothing; in a row that is seen, only the weights that it has part in."""
    c = Chunked(np.random.default_rng(5), *TYPES[types], [70], [10], 1, 4, 64, 16)
    own = c.rows(0)
    rest = np.ones(len(c.k), bool)
    rest[own] = False
    c.k[rest] = np.nan
    lse = lse_of(c)
    check(c, lse, 10, run(gpu, c, lse, 10))
    lse[3] = np.nan  # one token's outputs were NaN: so is what it sees
    got = run(gpu, c, lse, 10)
    assert np.isnan(got[4][0, 0, :74]).all() and np.isfinite(got[4][0, 0, 74:80]).all()


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens,counts,gqa", [([70], [10], 4), ([3000, 40], [60, 5], 8), ([40000], [40], 4)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_token_without_weights_adds_nothing_whatever_its_query_holds(gpu, types, hd, lens, counts, gqa, bad):
    """Tokens with lse -infinity whose q is not finite: the others' weights alone, where waves share blocks of slots and not."""
    c = Chunked(np.random.default_rng(hd), *TYPES[types], lens, counts, 1, gqa, hd, 16)
    q = c.q.copy()
    lse = np.full((c.n_rows, c.nh), 4, np.float32)
    dead = [0, 3, counts[0] - 1]
    lse[dead] = -np.inf
    c.q[dead] = bad
    got = run(gpu, c, lse, 1000, with_acc=False)
    assert np.isfinite(got[4]).all()
    c.q = q
    lse[dead] = 1e5  # (e^-1e5 is 0, too; check's bound would be 0 times infinity)
    check(c, lse, max(counts), got, with_acc=False)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales(gpu, types, scale):
    c = Chunked(np.random.default_rng(8), *TYPES[types], [130], [9], 2, 4, 64, 16)
    c.scale = abs(scale)
    q = c.q
    c.q = -q if scale < 0 else q
    lse = lse_of(c)
    c.q, c.scale = q, scale
    got = run(gpu, c, lse, 5)
    c.q, c.scale = (-q if scale < 0 else q), abs(scale)  # (the bound's sums take a positive scale)
    check(c, lse, 5, got)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_more_work_than_workgroups(gpu, types):
    """More sequences than a wave has lanes, waiting ones among them, more slots than one round of workgroups takes."""
    rng = np.random.default_rng(9)
    lens = [int(n) for n in rng.integers(0, 700, 150)]
    lens[7] = lens[149] = -1
    c = Chunked(rng, *TYPES[types], lens, [1] * 150, 12, 1, 64, 64)
    lse = lse_of(c)
    check(c, lse, 1, run(gpu, c, lse, 1))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 45])
def test_many_blocks_of_slots(gpu, types, hd, window):
    """More than 512 blocks of 32 slots, each a wave's; missing pages, unseen rows that are not finite, several tiles of rows."""
    c = Chunked(np.random.default_rng(hd), *TYPES[types], [500, 33, 0], [12, 5, 70], 40, 3, hd, 24, window=window)
    c.table[0, 4:6] = -1
    rest = np.ones(len(c.k), bool)
    rest[np.concatenate([c.rows(b)[c.rows(b) >= 0] for b in range(3)])] = False
    c.k[rest] = np.nan
    lse = lse_of(c)
    check(c, lse, 30, run(gpu, c, lse, 30))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("lens,nkv", [([1000, 2900], 2), ([1000, 3200], 2), ([1000, 7000], 2), ([1000, 7300], 2)])
def test_blocks_shared_by_waves_or_not(gpu, types, lens, nkv):
    """Just fewer and just more blocks than waves share them for: the same weights to rounding."""
    c = Chunked(np.random.default_rng(17), *TYPES[types], lens, [11, 30], nkv, 12, 64, 100)
    lse = lse_of(c)
    check(c, lse, 25, run(gpu, c, lse, 25))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_results_repeat(gpu, types):
    c = Chunked(np.random.default_rng(6), *TYPES[types], [700, 90], [80, 40], 2, 8, 128, 64)
    lse = lse_of(c)
    assert np.array_equal(run(gpu, c, lse, 50)[4], run(gpu, c, lse, 50)[4])


def test_refusals(gpu):
    c = Chunked(np.random.default_rng(7), True, True, [9], [3], 2, 4, 64, 16)
    kv, ch, q = c.buffers(gpu)
    z = gpu.zeros(4096)

    def call(kv=kv, ch=ch, pos=z.ptr, nh=8, tq=L.F16, q=q.ptr, ldq=512, window=0, lse=z.ptr, last=1, acc_in=None, acc=z.ptr,
             where=z.ptr):
        return gpu.lib.styx_op_kv_weigh(gpu.h, C.byref(kv) if kv else None, C.byref(ch) if ch else None, pos, nh, tq, q, ldq,
                                        0.1, window, lse, last, 1.0, acc_in, acc, where)

    assert call() == 0
    for b in [dict(kv=None), dict(ch=None), dict(pos=None), dict(nh=7), dict(nh=34), dict(tq=3), dict(q=None), dict(ldq=504),
              dict(ldq=514), dict(q=q.ptr + 4), dict(window=-1), dict(last=-1), dict(lse=None), dict(acc=None)]:
        assert call(**b) == -1, b
    assert call(pos=None, where=None) == 0
    assert call(ch=L.KvChunk(1 << 27, ch.first, ch.count, ch.len)) == -1
    gpu.sync()
