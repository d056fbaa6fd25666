"""styx_op_attn_chunk (no counterpart in the reference) against its definition
in 64 bits, through the C ABI.  Tolerances: chunk_cases.Chunked.attend."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from chunk_cases import E, E16, TINY16, Chunked, check_chunk, run_chunk
from styx_amd import _lib as L

pytestmark = pytest.mark.gpu

TYPES = {"f32": (False, False), "f16": (True, True), "mixed": (True, False)}  # cache, q in 16 bits


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gqa", [1, 3, 8, 16])
def test_ragged_batch(gpu, types, hd, gqa):
    """Sequences of no rows and of many, one token and many, waiting ones between them."""
    rng = np.random.default_rng(hd + gqa)
    c = Chunked(rng, *TYPES[types], [0, 0, 5, -1, 130, 63, 1, 300], [1, 37, 1, 4, 66, 2, 0, 17], 2, gqa, hd, 16)
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("page", [1, 7, 100, 512])
def test_pages_that_end_inside_a_tile(gpu, types, page):
    c = Chunked(np.random.default_rng(page), *TYPES[types], [211, 64], [45, 64], 1, 4, 128, page)
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("window", [1, 2, 31, 64, 200, 431, 432, 1 << 30, 2 ** 31 - 1])
def test_window(gpu, types, window):
    c = Chunked(np.random.default_rng(window % 97), *TYPES[types], [0, 150, 400], [140, 33, 1], 2, 2, 64, 32, window=window)
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("lens,counts", [([2000], [1]), ([5000, 3], [2, 1]), ([0], [600]), ([1500, 900, 0, 40], [16, 128, 1, 300])])
def test_long_contexts(gpu, types, lens, counts):
    """Few tokens over many rows (split over workgroups), and prompts of several tiles."""
    c = Chunked(np.random.default_rng(len(lens)), *TYPES[types], lens, counts, 2, 8, 128, 64)
    check_chunk(c, *run_chunk(gpu, c), tokens=lambda n: range(n) if n < 20 else sorted({0, 1, n // 3, n // 2, n - 2, n - 1}))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_many_sequences_of_one_token(gpu, types):
    lens = [(37 * b) % 500 for b in range(150)]
    c = Chunked(np.random.default_rng(3), *TYPES[types], lens, [1] * 150, 1, 4, 64, 16)
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_rows_in_any_order_with_gaps_and_strides(gpu, types):
    """Sequences' rows in no order with rows of none between them, rows farther apart than they are long, no lse."""
    c = Chunked(np.random.default_rng(5), *TYPES[types], [9, 70, 0], [5, 20, 3], 2, 4, 64, 16, first=[30, 7, 1], n_rows=40,
                ld=2 * 4 * 64 + 72)
    out, lse = run_chunk(gpu, c, lse=False, ldo=2 * 4 * 64 + 24)
    check_chunk(c, out)
    assert (lse == 7.5).all()


@pytest.mark.parametrize("types", sorted(TYPES))
def test_skipped_sequences(gpu, types):
    """Lengths, counts and rows outside their ranges: nothing of the sequence is read or written."""
    big = 2 ** 31 - 1
    lens, counts = [10, -1, 40, 10, 10, big, 5, 10, 5], [4, 4, 30, 4, -3, 4, big, 4, 0]
    first = [0, 4, 8, -1, 12, 16, 20, 61, 24]
    c = Chunked(np.random.default_rng(6), *TYPES[types], [10] * 9, [4] * 9, 1, 2, 64, 8, first=first, n_rows=64, table_len=8)
    c.lens, c.counts = np.array(lens, np.int32), np.array(counts, np.int32)
    assert [c.taken(b) for b in range(9)] == [True] + [False] * 8
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
def test_full_cache(gpu, types):
    c = Chunked(np.random.default_rng(8), *TYPES[types], [50, 0], [14, 64], 1, 4, 128, 16, table_len=4, spare=0)
    assert c.cap == 64
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128])
def test_missing_pages(gpu, types, hd):
    """Entries outside the pool: their rows are not seen; a token that sees nothing gets 0 and -infinity."""
    c = Chunked(np.random.default_rng(9), *TYPES[types], [90, 0, 200], [20, 40, 3], 1, 4, hd, 16)
    c.table[0, [0, 3]] = -1
    c.table[0, 6] = c.n_pages
    c.table[1, :2] = -7
    c.table[2, 1:] = 2 ** 31 - 1
    out, lse = run_chunk(gpu, c)
    check_chunk(c, out, lse)
    f = int(c.first[1])
    assert (out[f:f + 32] == 0).all() and np.isneginf(lse[f:f + 32]).all() and np.isfinite(lse[f + 32]).all()


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_what_is_not_seen_has_no_influence(gpu, types, bad, hd):
    """Values that are not finite behind the last row, in pages of others, outside the window, and in new rows that
    only later tokens see: the others' outputs are those of the definition."""
    c = Chunked(np.random.default_rng(10), *TYPES[types], [70, 20], [50, 9], 1, 4, hd, 16, window=60)
    rows = [c.rows(b) for b in range(2)]
    own = np.concatenate(rows)
    for p in (c.k, c.v):
        rest = np.ones(len(p), bool)
        rest[own] = False
        p[rest] = bad
        p[rows[0][:5]] = bad       # outside every token's window
        p[rows[0][70 + 41]] = bad  # seen by the tokens from 41 on
    out, lse = run_chunk(gpu, c)
    later = np.zeros(c.n_rows, bool)
    later[41:50] = True
    assert np.isfinite(out[~later]).all() and np.isfinite(lse[~later]).all()
    check_chunk(c, out, lse, tokens=lambda n: range(min(n, 41)))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("count", [1, 50])
def test_values_that_are_not_finite_reach_the_outputs(gpu, types, count):
    c = Chunked(np.random.default_rng(11), *TYPES[types], [300], [count], 1, 2, 128, 16)
    rows = c.rows(0)
    c.v[rows[17], 0, 5] = np.nan
    c.v[rows[200], 0, 9] = np.inf
    c.v[rows[300], 0, 70] = np.inf  # the first new row
    out, lse = run_chunk(gpu, c)
    out = out.reshape(count, 2, 128)
    assert not np.isfinite(out[:, :, [5, 9, 70]]).any() and np.isfinite(lse).all()
    assert np.isfinite(np.delete(out, [5, 9, 70], 2)).all()
    c.k[rows[40], 0, 3] = np.nan
    out, lse = run_chunk(gpu, c)
    assert np.isnan(out).all() and np.isnan(lse).all()


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens,counts,window", [([0, 0, 0], [1, 1, 1], 0), ([200, 0, 2000], [70, 33, 3], 1)])
def test_one_slot_gives_its_value(gpu, types, hd, lens, counts, window):
    """A weight of 1 is no rounding: 16-bit outputs are the slot's V itself, 32-bit ones to the quotient of two sums."""
    c = Chunked(np.random.default_rng(hd), *TYPES[types], lens, counts, 2, 4, hd, 16, window=window)
    out, lse = run_chunk(gpu, c)
    check_chunk(c, out, lse, tokens=FEW)
    for b in range(3):
        rows = c.rows(b)
        for i in range(counts[b]):
            want = np.repeat(c.v[rows[lens[b] + i]], 4, 0)
            got = out[c.first[b] + i].reshape(8, hd)
            if c.q16:
                assert np.array_equal(got, want), (b, i)
            else:  # a factor's own pieces or bits, over it: 2^-22 and two roundings
                want = want.astype(np.float64)
                assert (np.abs(got - want) <= (2.0 ** -22 + 4 * E) * np.abs(want)).all(), (b, i)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_large_and_equal_scores(gpu, types):
    """Scores of hundreds, whose exponentials underflow or are all 1."""
    c = Chunked(np.random.default_rng(12), *TYPES[types], [100, 80], [30, 3], 1, 4, 64, 16)
    c.q = (c.q * 40).astype(c.qt)
    c.q[30:] = 0
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("start", [0, 32, 64])
@pytest.mark.parametrize("slots", [130, 6000])
@pytest.mark.parametrize("sizes", [(1, 0.5, 1, 1.25), (1, 0.5, 1, 0.75)])
def test_a_score_far_above_those_before_it(gpu, types, hd, start, slots, sizes):
    """Slots with scores of 0, 32 of 7.75 (in units of ln 2), one of `jump`, the rest of -60: V is 1 in the 32 alone, so
    that the outputs are nothing but their small weights, whatever part of a block the large score comes in.  Queries of
    `sizes`: 1.25 moves the reference for the 32, too (7.75 times it is more than 8).

    Weights as in Chunked.attend; with 16-bit rows a factor is also off by half of f16's smallest step when it is formed
    and once more when the large score moves the reference: 2 TINY16, where the largest factor is 2^6 at least."""
    for jump in (9, 15, 23.5, 24, 24.5, 25.5, 26.5, 33):
        c = Chunked(np.random.default_rng(1), *TYPES[types], [slots - 4], [4], 2, 4, hd, 16)
        c.scale = float(np.float32(np.log(2)))
        s = np.full(slots, -60.0)
        s[:start], s[start:start + 32], s[start + 32] = 0, 7.75, jump
        rows = c.rows(0)
        c.q[:], c.k[:], c.v[:] = 0, 0, 0
        c.q.reshape(4, 8, hd)[:, :, 0] = sizes * 2
        c.k[rows, :, 0] = s[:, None]
        c.v[rows[start:start + 32]] = 1
        out, lse = run_chunk(gpu, c)
        for i, j in ((0, 0), (3, 1)):
            want, _, want_lse, tol_lse = c.attend(0, i, j)
            x, ds, see = c.scores(0, i, j, rows)
            tot = np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)
            tol = (2 * ds.max(1, keepdims=True) + 2 * (see.sum() + 40) * E) * want + 1e-30
            if c.f16:
                tol = tol + 2 * TINY16 * 2.0 ** -6 * 32 / tot
            if c.q16:
                tol = tol + E16 * want + E16 * want + TINY16
            got = out[i].reshape(8, hd)[4 * j:4 * j + 4].astype(np.float64)
            assert (np.abs(got - want) <= tol).all(), (jump, i, j, got[:, 0], want[:, 0], tol[:, 0])
            assert (np.abs(lse[i, 4 * j:4 * j + 4] - want_lse) <= tol_lse).all(), (jump, i, j)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_results_repeat(gpu, types):
    """No result depends on an order of execution or on what the workspace held."""
    c = Chunked(np.random.default_rng(13), *TYPES[types], [3000, 40, 900], [7, 100, 1], 2, 8, 128, 64)
    a, b = run_chunk(gpu, c), run_chunk(gpu, c)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


FEW = lambda n: range(n) if n < 12 else sorted({0, 1, n // 3, n // 2, n - 2, n - 1})  # noqa: E731


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gqa", [1, 5, 16])
def test_tiles_cut_into_shares(gpu, types, hd, gqa):
    """Long contexts beside short ones, one token beside many: shares that end inside tiles, hold several, or none."""
    c = Chunked(np.random.default_rng(hd * gqa), *TYPES[types], [3000, 0, 2500, 700, 1], [1, 90, 40, 3, 1], 2, gqa, hd, 48)
    check_chunk(c, *run_chunk(gpu, c), tokens=FEW)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_cut_tiles_with_missing_pages_and_values_that_are_not_finite(gpu, types, hd):
    c = Chunked(np.random.default_rng(hd), *TYPES[types], [3100, 2000], [5, 70], 1, 4, hd, 16)
    rows = c.rows(1)
    c.table[0, 20:140] = -1          # whole pieces without a row
    c.table[0, 194:] = c.n_pages + 3  # the new rows' among them
    for p in (c.k, c.v):
        rest = np.ones(len(p), bool)
        rest[np.concatenate([c.rows(b)[c.rows(b) >= 0] for b in range(2)])] = False
        p[rest] = np.nan
    c.v[rows[2040], 0, 3] = np.inf   # seen by the tokens from 40 on
    out, lse = run_chunk(gpu, c)
    check_chunk(c, out, lse, tokens=lambda n: range(min(n, 40)))
    late = out[5 + 40:75].reshape(30, 4, hd)
    assert not np.isfinite(late[:, :, 3]).any() and np.isfinite(np.delete(late, 3, 2)).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("window", [700, 2500])
def test_cut_tiles_under_a_window(gpu, types, window):
    c = Chunked(np.random.default_rng(window), *TYPES[types], [4000, 100, 3000], [3, 60, 33], 1, 8, 128, 100, window=window)
    check_chunk(c, *run_chunk(gpu, c), tokens=FEW)


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gqa,counts", [(8, [1, 2, 1]), (8, [3, 1, 4]), (1, [31, 0, 1]), (1, [5, 27, 1]), (16, [2, 1, 1]), (1, [60, 5, 0])])
@pytest.mark.parametrize("window", [0, 45, 900])
def test_few_rows(gpu, types, hd, gqa, counts, window):
    """Calls of 32, 33, 64, 65 rows and fewer: whole contexts and cut ones, missing pages, unseen values that are not finite."""
    lens = [40, 2100, 333]
    c = Chunked(np.random.default_rng(hd + gqa + sum(counts)), *TYPES[types], lens, counts, 2, gqa, hd, 24, window=window)
    c.table[1, 3:60] = -1
    for p in (c.k, c.v):
        rest = np.ones(len(p), bool)
        rest[np.concatenate([c.rows(b)[c.rows(b) >= 0] for b in range(3)])] = False
        p[rest] = np.nan
    late = c.rows(0)[lens[0] + counts[0] - 1]  # seen by the first sequence's last token alone
    c.v[late, 1, hd - 1] = np.inf
    out, lse = run_chunk(gpu, c)
    assert not np.isfinite(out[counts[0] - 1].reshape(2, gqa, hd)[1, :, hd - 1]).any()
    c.v[late, 1, hd - 1] = 0
    out[counts[0] - 1].reshape(2, gqa, hd)[1, :, hd - 1] = run_chunk(gpu, c)[0][counts[0] - 1].reshape(2, gqa, hd)[1, :, hd - 1]
    check_chunk(c, out, lse, tokens=FEW)


@pytest.mark.parametrize("types", sorted(TYPES))
def test_many_sequences_with_long_ones_among_them(gpu, types):
    """More sequences than a wave has lanes, a few of them cut, skipped ones between."""
    rng = np.random.default_rng(16)
    lens = [int(n) for n in rng.integers(0, 60, 140)]
    counts = [int(n) for n in rng.integers(0, 4, 140)]
    for b in (3, 64, 70, 139):
        lens[b], counts[b] = 2000 + b, 1 + b % 3
    lens[5], lens[100] = -1, -1
    c = Chunked(rng, *TYPES[types], lens, counts, 1, 4, 64, 32)
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("nkv", [7, 40, 300, 600])
def test_many_kv_heads(gpu, types, nkv):
    """Fewer and fewer shares for a head, down to one."""
    c = Chunked(np.random.default_rng(nkv), *TYPES[types], [900, 0], [1, 2], nkv, 1, 64, 64)
    check_chunk(c, *run_chunk(gpu, c))


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(gpu, types, scale):
    c = Chunked(np.random.default_rng(17), *TYPES[types], [130], [9], 2, 4, 64, 16, window=50)
    c.scale = scale
    c.k = (c.k * 0.2).astype(c.dt)
    out, lse = run_chunk(gpu, c)
    c2 = Chunked(np.random.default_rng(17), *TYPES[types], [130], [9], 2, 4, 64, 16, window=50)
    c2.k, c2.v, c2.table = c.k, c.v, c.table
    c2.q, c2.scale = (-c.q if scale < 0 else c.q), abs(scale)  # (the bound's sums take a positive scale)
    check_chunk(c2, out, lse)


def test_queries_of_all_sizes_on_a_16_bit_cache(gpu):
    """f32 queries from 1e-30 to 1e4 and rows of zeros: the pieces' power of two is the row's own."""
    c = Chunked(np.random.default_rng(18), True, False, [60], [40], 1, 4, 64, 16)
    size = np.float32(10.0) ** np.random.default_rng(19).uniform(-30, 2, (40, 4)).astype(np.float32)
    c.q = (c.q.reshape(40, 4, 64) * size[:, :, None]).reshape(40, -1).astype(np.float32)
    c.q[7] = 0
    check_chunk(c, *run_chunk(gpu, c))


def test_more_rows_than_the_sequences_have(gpu):
    """A chunk laid out for a larger batch: rows behind the last sequence stay as they are."""
    for types in TYPES.values():
        c = Chunked(np.random.default_rng(20), *types, [900, 40], [1, 30], 2, 4, 64, 16, n_rows=5000)
        check_chunk(c, *run_chunk(gpu, c))


def test_offsets_past_32_bits(gpu):
    """Pools of more than 2^32 bytes and 2^31 values: rows at their ends."""
    c = Chunked(np.random.default_rng(14), True, True, [40], [9], 8, 2, 128, 64)
    n_pages = (2 ** 31 + 2 ** 20) // (64 * 8 * 128)
    kv, ch, q = c.buffers(gpu)
    table = np.array([[n_pages - 1]], np.int32)
    big = [gpu.buffer(2 * n_pages * 64 * 8 * 128) for _ in range(2)]
    at = 2 * (n_pages - 1) * 64 * 8 * 128
    page = c.table[0, 0]
    for buf, x in zip(big, (c.k, c.v)):
        buf.upload(x[page * 64:(page + 1) * 64], at)
    tab = gpu.from_numpy(table)
    kv.n_pages, kv.kpool, kv.vpool, kv.page_table = n_pages, big[0].ptr, big[1].ptr, tab.ptr
    out = gpu.zeros(2 * c.n_rows * c.nh * c.hd)
    need = gpu.lib.styx_op_attn_chunk_ws_bytes(C.byref(kv), c.n_rows, c.nh)
    ws = gpu.buffer(need)
    L.check(gpu.lib.styx_op_attn_chunk(gpu.h, C.byref(kv), C.byref(ch), c.nh, L.F16, q.ptr, c.ld, c.scale, 0, out.ptr,
                                       c.ld, None, ws.ptr, need))
    gpu.sync()
    check_chunk(c, out.download(np.float16).reshape(c.n_rows, -1))
    for b in big:
        b.free()


def test_refusals(gpu):
    c = Chunked(np.random.default_rng(15), True, True, [9], [3], 2, 4, 64, 16)
    kv, ch, q = c.buffers(gpu)
    need = gpu.lib.styx_op_attn_chunk_ws_bytes(C.byref(kv), 3, 8)
    ws, out = gpu.buffer(need + 16), gpu.zeros(4 * 3 * 8 * 64)

    def call(kv=kv, ch=ch, nh=8, tq=L.F16, q=q.ptr, ldq=512, window=0, out=out.ptr, ldo=512, ws=ws.ptr, n=need):
        return gpu.lib.styx_op_attn_chunk(gpu.h, C.byref(kv) if kv else None, C.byref(ch) if ch else None, nh, tq, q, ldq,
                                          0.1, window, out, ldo, None, ws, n)

    def other(**f):
        k = L.KvCache(*(getattr(kv, n) for n, _ in kv._fields_))
        for n, v in f.items():
            setattr(k, n, v)
        return k

    assert call() == 0
    bad = [dict(kv=None), dict(ch=None), dict(nh=7), dict(nh=0), dict(nh=34), dict(tq=L.Q8_0), dict(q=None), dict(out=None),
           dict(ldq=511), dict(ldq=516), dict(ldo=504), dict(ldo=2 ** 31), dict(q=q.ptr + 2), dict(out=out.ptr + 8), dict(window=-1),
           dict(ws=None), dict(n=need - 1), dict(ws=ws.ptr + 4), dict(kv=other(hd=96)), dict(kv=other(kpool=None)),
           dict(kv=other(kpool=kv.kpool + 8)), dict(kv=other(type=L.F32)), dict(kv=other(page_tokens=0)),
           dict(kv=other(table_len=0)), dict(ch=L.KvChunk(-1, ch.first, ch.count, ch.len)),
           dict(ch=L.KvChunk(3, None, ch.count, ch.len)), dict(ch=L.KvChunk(3, ch.first, None, ch.len)),
           dict(ch=L.KvChunk(3, ch.first, ch.count, None)), dict(ch=L.KvChunk(2 ** 31 - 1, ch.first, ch.count, ch.len))]
    for b in bad:
        assert call(**b) == -1, b
    assert call(ch=L.KvChunk(0, ch.first, ch.count, ch.len)) == 0  # no rows: nothing to do
    assert gpu.lib.styx_op_attn_chunk(None, C.byref(kv), C.byref(ch), 8, L.F16, q.ptr, 512, 0.1, 0, out.ptr, 512, None,
                                      ws.ptr, need) == -1
    gpu.sync()
