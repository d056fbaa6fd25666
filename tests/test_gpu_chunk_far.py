"""The operators on new tokens where offsets pass 32 bits: pools of more than
2^31 values, accumulators and page tables of more than 2^31 bytes.  The same
data at the near end of small arrays is the measure: the places must not
change a bit (that those are right is for the operators' own tests)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from chunk_cases import Chunked
from styx_amd import _lib as L, rope_table

pytestmark = pytest.mark.gpu

TYPES = {"f32": (False, False), "f16": (True, True), "mixed": (True, False)}
VALUES = 2 ** 31 + 2 ** 22


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


@pytest.fixture(scope="module")
def big(gpu):
    """Two pools of VALUES f32 values."""
    bufs = [gpu.buffer(4 * VALUES) for _ in range(2)]
    yield bufs
    for b in bufs:
        b.free()


def far_cache(c, kv, big):
    """The cache `kv` of the Chunked c with its pages at the far end of the big pools: the same page indices from
    behind, and what was in the small pools there."""
    es, row = c.dt().itemsize, c.nkv * c.hd
    n_pages = VALUES // (c.page * row)
    shift = n_pages - c.n_pages
    at = shift * c.page * row * es
    assert shift * c.page * row > 2 ** 31 and at + es * c.k.size <= big[0].nbytes
    for buf, x in zip(big, (c.k, c.v)):
        buf.upload(x, at)
    return L.KvCache(kv.type, kv.n_seq, kv.nkv, kv.hd, kv.page_tokens, n_pages, kv.table_len, big[0].ptr, big[1].ptr,
                     kv.page_table), shift


@pytest.mark.parametrize("types", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [64, 50])
def test_rows_past_32_bits(gpu, big, types, hd, page):
    """Attention and weights, one token and a prompt."""
    c = Chunked(np.random.default_rng(hd + page), *TYPES[types], [700, 40], [1, 70], 4, 4, hd, page)
    f = L.F16 if c.q16 else L.F32
    got = []
    for far in (False, True):
        kv, ch, q = c.buffers(gpu)
        if far:
            kv, shift = far_cache(c, kv, big)
            c.bufs[2].upload(np.where(c.table >= 0, c.table + shift, -1).astype(np.int32))
        out, lse = gpu.zeros(c.q.nbytes), gpu.zeros(4 * c.n_rows * c.nh)
        n = gpu.lib.styx_op_attn_chunk_ws_bytes(C.byref(kv), c.n_rows, c.nh)
        ws, acc = gpu.buffer(n), gpu.zeros(4 * c.B * c.nkv * c.cap)
        L.check(gpu.lib.styx_op_attn_chunk(gpu.h, C.byref(kv), C.byref(ch), c.nh, f, q.ptr, c.ld, c.scale, 0, out.ptr, c.ld,
                                           lse.ptr, ws.ptr, n))
        L.check(gpu.lib.styx_op_kv_weigh(gpu.h, C.byref(kv), C.byref(ch), None, c.nh, f, q.ptr, c.ld, c.scale, 0, lse.ptr, 40,
                                         1.0, None, acc.ptr, None))
        gpu.sync()
        got.append([b.download() for b in (out, lse, acc)])
    for near, there in zip(*got):
        assert near.any() and np.array_equal(near, there)


@pytest.mark.parametrize("t_in,t_c", [(L.F32, L.F32), (L.F16, L.F16), (L.F32, L.F16)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_appended_rows_past_32_bits(gpu, big, t_in, t_c, hd):
    rng = np.random.default_rng(hd)
    n, nh, nkv, page, pages = 37, 4, 8, 16, 5
    np_of = {L.F32: np.float32, L.F16: np.float16}
    ld, row, es = (nh + 2 * nkv) * hd, nkv * hd, np_of[t_c]().itemsize
    x = gpu.from_numpy(rng.standard_normal((n, ld)).astype(np_of[t_in]))
    tab, w = gpu.from_numpy(rope_table(hd, 90, 1e4)), gpu.from_numpy((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32))
    at = rng.permutation(pages * page)[:n].astype(np.int32)
    pos = gpu.from_numpy(rng.integers(0, 90, n).astype(np.int32))
    rope, before = L.Rope(tab.ptr, 90, hd, 0), rng.standard_normal((pages * page, row)).astype(np_of[t_c])
    got = []
    for far in (False, True):
        n_pages = VALUES // (page * row) if far else pages
        first = (n_pages - pages) * page
        pools = big if far else [gpu.buffer(before.nbytes) for _ in range(2)]
        for p in pools:
            p.upload(before, first * row * es)
        rows, out = gpu.from_numpy((at + first).astype(np.int32)), gpu.zeros(4 * n * nh * hd)
        kv = L.KvCache(t_c, 1, nkv, hd, page, n_pages, 1, pools[0].ptr, pools[1].ptr, rows.ptr)
        k = x.ptr + nh * hd * np_of[t_in]().itemsize
        L.check(gpu.lib.styx_op_kv_append(
            gpu.h, C.byref(kv), n, pos.ptr, rows.ptr, nh, t_in, x.ptr, ld, k, ld, k + row * np_of[t_in]().itemsize, ld, w.ptr,
            w.ptr, 1e-6, C.byref(rope), L.F32, out.ptr, nh * hd))
        gpu.sync()
        got.append([out.download()] + [p.download(np.uint8, before.nbytes, first * row * es) for p in pools])
        assert not far or first * row > 2 ** 31 - 2 ** 22
    for near, there in zip(*got):
        assert np.array_equal(near, there)
    assert not np.array_equal(got[0][1], before.view(np.uint8).ravel())


@pytest.mark.parametrize("types", sorted(TYPES))
def test_weights_past_32_bits(gpu, types):
    """Accumulators and positions of 2^32 entries, the last head of the last sequence."""
    page, table_len = 1 << 20, 1 << 10
    c = Chunked(np.random.default_rng(1), *TYPES[types], [-1, 90], [0, 12], 2, 4, 64, 128)
    lse = np.full((c.n_rows, c.nh), 2.0, np.float32)
    got = []
    for far in (False, True):
        kv, ch, q = c.buffers(gpu)
        cap, table = c.cap, c.table
        if far:
            cap = page * table_len
            assert c.table_len == 1
            table = np.full((2, table_len), -1, np.int32)
            table[1, 0] = 0
            pools = [gpu.buffer(page * 2 * 64 * c.dt().itemsize) for _ in range(2)]
            for p, x in zip(pools, (c.k, c.v)):
                p.upload(x[c.table[1, 0] * 128:][:102])
            tab = gpu.from_numpy(table)
            kv = L.KvCache(kv.type, 2, 2, 64, page, 1, table_len, pools[0].ptr, pools[1].ptr, tab.ptr)
        acc, where, l, pos = gpu.buffer(16 * cap), gpu.buffer(16 * cap), gpu.from_numpy(lse), gpu.from_numpy(np.array([0, 7], np.int32))
        mine = np.array([[0.5] * 104, [0.25] * 104], np.float32)
        for j in range(2):
            acc.upload(mine[j], 4 * (2 + j) * cap)
            where.upload(np.full(104, 3, np.int32), 4 * (2 + j) * cap)
        L.check(gpu.lib.styx_op_kv_weigh(gpu.h, C.byref(kv), C.byref(ch), pos.ptr, c.nh, L.F16 if c.q16 else L.F32, q.ptr, c.ld,
                                         c.scale, 0, l.ptr, 5, 0.5, acc.ptr, acc.ptr, where.ptr))
        gpu.sync()
        got.append([b.download(t, 104, 4 * (2 + j) * cap) for j in range(2) for b, t in ((acc, np.float32), (where, np.int32))])
        for b in (acc, where):
            b.free()
    for near, there in zip(*got):
        assert np.array_equal(near, there)
    a, w = got[1][2:]
    assert (a[:90] > 0.125).all() and (a[102:] == 0.25).all()
    assert (w[:90] == 3).all() and (w[90:102] == 7 + np.arange(12)).all() and (w[102:] == 3).all()


def test_a_page_table_past_32_bits(gpu):
    """Three sequences of 2^29 entries: the last gets pages at the table's end, gives them back, and gets them again."""
    T = 1 << 29
    table, i32 = gpu.buffer(4 * 3 * T), lambda *x: gpu.from_numpy(np.array(x, np.int32))
    end = 4 * (3 * T - 4)
    table.upload(np.array([2, 5, -1, -1], np.int32), end)
    held, free, n_free = i32(0, 0, T - 2), i32(7, 1, 3, 6, 0, 0, 0, 0), i32(4)
    lens, first, count = i32(-1, -1, T - 2), i32(0, 0, 0), i32(0, 0, 0)
    rows = [i32(9, 9) for _ in range(3)]
    kv = L.KvCache(L.F32, 3, 1, 64, 1, 8, T, None, None, None)
    pages = L.KvPages(table.ptr, held.ptr, free.ptr, n_free.ptr)

    def plan(new, n_rows):
        asked, pos = i32(0, 0, new), i32(0, 0, 100)
        L.check(gpu.lib.styx_op_kv_plan(gpu.h, C.byref(kv), C.byref(pages), C.byref(pages), None, lens.ptr, asked.ptr, pos.ptr,
                                        n_rows, first.ptr, count.ptr, *(r.ptr for r in rows)))
        gpu.sync()
        return table.download(np.int32, 4, end).tolist(), held.download(np.int32, 3).tolist(), free.download(np.int32, 8).tolist()

    want = [2, 5, 6, 3], [0, 0, T], [7, 1, -1, -1, 0, 0, 0, 0]
    assert plan(2, 2) == want and count.download(np.int32, 3).tolist() == [0, 0, 2]
    assert [r.download(np.int32, 2).tolist() for r in rows] == [[2, 2], [100, 101], [6, 3]]
    lens.upload(np.array([-1, -1, T - 3], np.int32))
    assert plan(0, 0) == ([2, -1, -1, -1], [0, 0, T - 3], [7, 1, 5, 6, 3, 0, 0, 0])
    assert plan(1, 1) == ([2, 3, -1, -1], [0, 0, T - 2], [7, 1, 5, 6, -1, 0, 0, 0])
    table.free()
