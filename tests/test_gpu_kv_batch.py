"""The operators on a batch's paged KV cache (no counterpart in the
reference): styx_op_attn_decode_batch and styx_op_kv_evict against their
definitions in 64 bits, through the C ABI.

Tolerances of the attention: with E = 2^-24 (half a step of f32) a score's
error is at most ds = (hd + 8) E scale sum |q_i k_i| (the products' f32 sum
and the query's rounding; f16 caches: plus 2^-22 of the same sum for the two
f16 pieces of the query), a weight's relative error at most 2 ds + (n + 40) E
(numerator and sum of n terms, exponentials and factors of the merges; f16
caches: plus 2^-21), and a value sum's at most the same once more for its n
additions.  The appended row is the f64 row rounded to f32 and then to the
cache's type."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from styx_amd import _lib as L

E = 2.0 ** -24
EPS = 1e-6


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


class Case:
    """A cache with lens[b] rows in pages in no order, and the new tokens."""

    def __init__(self, rng, f16, lens, nkv, gqa, hd, page, pos=None, table_len=None, norms=True, spare=2):
        self.f16, self.nkv, self.gqa, self.nh, self.hd, self.page = f16, nkv, gqa, nkv * gqa, hd, page
        self.dt = np.float16 if f16 else np.float32
        self.lens = np.array(lens, np.int32)
        self.B = len(lens)
        used = [max(0, -(-(max(n, 0) + 1) // page)) for n in lens]
        self.table_len = table_len or max(used)
        used = [min(u, self.table_len) for u in used]
        self.cap = self.table_len * page
        self.n_pages = sum(used) + spare
        perm = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((self.B, self.table_len), -1, np.int32)
        at = 0
        for b, u in enumerate(used):
            self.table[b, :u] = perm[at:at + u]
            at += u
        shape = (self.n_pages * page, nkv, hd)
        self.k = rng.standard_normal(shape).astype(self.dt)
        self.v = rng.standard_normal(shape).astype(self.dt)
        self.pos = np.array([n + 3 if n >= 0 else 0 for n in lens] if pos is None else pos, np.int32)
        self.n_rope = int(max(self.pos.max(), 0)) + 1
        self.rope = np.empty((self.n_rope, hd // 2, 2), np.float64)
        L.load().styx_rope_table(1e6, hd, self.n_rope, self.rope.ctypes.data)
        r = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.q, self.kn, self.vn = r(self.B, self.nh, hd), r(self.B, nkv, hd), r(self.B, nkv, hd)
        self.qw = 1 + 0.1 * r(hd) if norms else None
        self.kw = 1 + 0.1 * r(hd) if norms else None
        self.scale, self.decay = 1.0 / np.sqrt(hd), 0.9
        self.acc = np.exp(rng.standard_normal((self.B, nkv, self.cap))).astype(np.float32)
        self.where = np.tile(np.arange(self.cap, dtype=np.int32) * 2, (self.B, nkv, 1))

    def rows(self, b, n):
        """Pool rows of slots [0, n), -1 in pages outside the pool."""
        t = np.arange(n)
        e = self.table[b, t // self.page]
        return np.where((e >= 0) & (e < self.n_pages), e.astype(np.int64) * self.page + t % self.page, -1)

    def seen(self, b):
        n = int(self.lens[b])
        return 0 <= n < self.cap and 0 <= self.pos[b] < self.n_rope

    def head(self, x, w, p):
        x = x.astype(np.float64)
        if w is not None:
            x = x / np.sqrt((x * x).sum() / self.hd + EPS) * w.astype(np.float64)
        h = self.hd // 2
        c, s = self.rope[p, :, 0], self.rope[p, :, 1]
        return np.concatenate([x[:h] * c - x[h:] * s, x[:h] * s + x[h:] * c])

    def kv(self, gpu):
        self.bufs = [gpu.from_numpy(x) for x in (self.k, self.v, self.table)]
        return L.KvCache(L.F16 if self.f16 else L.F32, self.B, self.nkv, self.hd, self.page, self.n_pages,
                         self.table_len, *(b.ptr for b in self.bufs))


def run_attn(gpu, c, scored=True, in_place=False, with_acc_in=True, ws_fill=None):
    """Outputs of the call: out, acc_out, slot_pos, K pool, V pool (buffers
    that the call does not write keep what is put there first)."""
    lib = gpu.lib
    kv = c.kv(gpu)
    b = {n: gpu.from_numpy(x) for n, x in dict(len=c.lens, pos=c.pos, q=c.q, k=c.kn, v=c.vn, rope=c.rope,
                                               acc=c.acc, where=c.where).items()}
    out = gpu.from_numpy(np.full((c.B, c.nh, c.hd), 7.5, np.float32))
    acc_out = b["acc"] if in_place else gpu.from_numpy(np.full(c.acc.shape, -3.0, np.float32))
    qw, kw = (gpu.from_numpy(w) if w is not None else None for w in (c.qw, c.kw))
    nbytes = lib.styx_op_attn_batch_ws_bytes(C.byref(kv), c.nh, int(scored))
    assert nbytes > 0
    ws = gpu.from_numpy(np.full(nbytes, 0xFF if ws_fill is None else ws_fill, np.uint8))
    ptr = lambda x: x.ptr if x is not None else None  # noqa: E731
    L.check(lib.styx_op_attn_decode_batch(
        gpu.h, C.byref(kv), b["len"].ptr, b["pos"].ptr, c.nh, b["q"].ptr, b["k"].ptr, b["v"].ptr, ptr(qw), ptr(kw),
        EPS, b["rope"].ptr, c.n_rope, c.scale, c.decay, b["acc"].ptr if scored and with_acc_in else None,
        acc_out.ptr if scored else None, b["where"].ptr if scored else None, out.ptr, ws.ptr, nbytes))
    gpu.sync()
    return (out.download(np.float32).reshape(c.q.shape), acc_out.download(np.float32).reshape(c.acc.shape),
            b["where"].download(np.int32).reshape(c.where.shape), c.bufs[0].download(c.dt).reshape(c.k.shape),
            c.bufs[1].download(c.dt).reshape(c.v.shape))


def check_attn(c, got, scored=True, in_place=False, with_acc_in=True):
    out, acc, where, kp, vp = got
    k, v = c.k.copy(), c.v.copy()
    want_where = c.where.copy()
    for b in range(c.B):
        n = int(c.lens[b])
        if not c.seen(b):
            assert (out[b] == 7.5).all()
            if scored:
                assert np.array_equal(acc[b], c.acc[b] if in_place else np.full_like(acc[b], -3.0))
            continue
        rows = c.rows(b, n + 1)
        there = np.nonzero(rows >= 0)[0]
        p = int(c.pos[b])
        for j in range(c.nkv):
            want_where[b, j, n] = p
            k64 = c.head(c.kn[b, j], c.kw, p)
            if rows[n] >= 0:
                # rounded to f32, then to the cache's type; f64 sums in another
                # order move the f32 rounding by at most one step
                step = (2.0 ** -11 if c.f16 else 0.0) + 2 * E
                assert np.all(np.abs(kp[rows[n], j].astype(np.float64) - k64)
                              <= step * np.abs(k64) + (2.0 ** -25 if c.f16 else 0.0))
                assert np.array_equal(vp[rows[n], j], c.vn[b, j].astype(c.dt))
                k[rows[n], j], v[rows[n], j] = kp[rows[n], j], vp[rows[n], j]
            K, V = k[rows[there], j].astype(np.float64), v[rows[there], j].astype(np.float64)
            total, total_tol = np.zeros(n + 1), np.zeros(n + 1)
            for h in range(j * c.gqa, (j + 1) * c.gqa):
                if len(there) == 0:
                    assert not out[b, h].any()
                    continue
                q = c.head(c.q[b, h], c.qw, p)
                s = K @ q * c.scale
                w = np.exp(s - s.max())
                w /= w.sum()
                size = (np.abs(K) @ np.abs(q)).max() * c.scale
                ds = size * ((c.hd + 8) * E + (2.0 ** -22 if c.f16 else 0.0))
                rel = 2 * ds + (n + 40) * E + (2.0 ** -21 if c.f16 else 0.0)
                with np.errstate(invalid="ignore"):
                    ref, tol = w @ V, (rel + (n + 40) * E) * (w @ np.abs(V))
                fine = np.isfinite(ref)
                assert np.array_equal(fine, np.isfinite(out[b, h]))
                assert np.all(np.abs(out[b, h] - ref)[fine] <= tol[fine] + 1e-30), (b, h)
                total[there] += w
                total_tol[there] += w * rel
            if scored:
                old = np.where(np.arange(n + 1) < n, c.acc[b, j, :n + 1].astype(np.float64), 0.0) if with_acc_in else 0.0
                ref = c.decay * old + total
                assert np.all(np.abs(acc[b, j, :n + 1] - ref) <= total_tol + (c.gqa + 4) * E * ref + 1e-12), (b, j)
                rest = c.acc[b, j, n + 1:] if in_place else np.full(c.cap - n - 1, -3.0, np.float32)
                assert np.array_equal(acc[b, j, n + 1:], rest)
    # every other row of the pools as it was, and the positions
    assert np.array_equal(kp.view(np.uint8), k.view(np.uint8)) and np.array_equal(vp.view(np.uint8), v.view(np.uint8))
    if scored:
        assert np.array_equal(where, want_where)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gqa", [1, 3, 8, 9, 16])
def test_attn_heads_and_types(gpu, f16, hd, gqa):
    rng = np.random.default_rng(hd + gqa)
    c = Case(rng, f16, [0, 1, 15, 16, 31, 63, 64, 200, 517], 2, gqa, hd, 48)
    check_attn(c, run_attn(gpu, c))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page", [1, 7, 16, 100, 512])
def test_attn_pages(gpu, f16, page):
    rng = np.random.default_rng(page)
    c = Case(rng, f16, [130, 7, 1023], 3, 4, 128, page, norms=False)
    check_attn(c, run_attn(gpu, c, scored=page != 7), scored=page != 7)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_attn_many_ragged_sequences(gpu, f16):
    """More sequences than lanes of a wave, among them ones that are skipped
    (length below 0, at and past the capacity, positions outside the table)."""
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(0, 300, 150)]
    pos = [n + 1 for n in lens]
    lens[3], lens[64], lens[127] = -1, 512, 100000
    pos[10], pos[149], pos[80] = -1, 2 ** 31 - 1, 400
    c = Case(rng, f16, [min(n, 511) for n in lens], 1, 5, 64, 16, pos=[min(p, 399) for p in pos], table_len=32)
    c.lens, c.pos = np.array(lens, np.int32), np.array(pos, np.int32)
    assert sum(not c.seen(b) for b in range(c.B)) == 6
    check_attn(c, run_attn(gpu, c))


@pytest.mark.gpu
@pytest.mark.parametrize("n_seq,nkv,hd,longest", [(100, 2, 64, 2000), (40, 8, 256, 150), (130, 8, 64, 90),
                                                  (300, 4, 64, 3), (3, 600, 64, 40), (2, 5, 128, 5000)])
def test_attn_shares_of_the_workgroups(gpu, n_seq, nkv, hd, longest):
    """More rows or heads than the workgroups that run at once, so that shares
    end inside a head and begin others; head counts that do not divide them."""
    rng = np.random.default_rng(n_seq)
    c = Case(rng, True, [int(x) for x in rng.integers(0, longest, n_seq)], nkv, 1, hd, 64)
    check_attn(c, run_attn(gpu, c))


@pytest.mark.gpu
def test_attn_pages_shared_by_sequences(gpu):
    """A common prefix in the same pages of three sequences, their own rows
    and the new ones in pages of their own."""
    rng = np.random.default_rng(21)
    c = Case(rng, False, [100, 75, 64], 2, 4, 64, 16)
    c.table[1, :4] = c.table[2, :4] = c.table[0, :4]
    check_attn(c, run_attn(gpu, c))


@pytest.mark.gpu
def test_attn_two_calls_on_one_stream_share_a_workspace_in_turn(gpu):
    """What a call leaves in the workspace does not reach the next one."""
    rng = np.random.default_rng(22)
    lib = gpu.lib
    cases = [Case(rng, False, [300, 20], 2, 8, 128, 64), Case(rng, True, [7], 1, 3, 64, 16),
             Case(rng, False, [5, 900, 31], 1, 16, 64, 32)]
    kvs = [c.kv(gpu) for c in cases]
    need = [lib.styx_op_attn_batch_ws_bytes(C.byref(kv), c.nh, 1) for kv, c in zip(kvs, cases)]
    ws = gpu.buffer(max(need))
    held = []
    for kv, c in zip(kvs, cases):
        b = [gpu.from_numpy(x) for x in (c.lens, c.pos, c.q, c.kn, c.vn, c.qw, c.kw, c.rope, c.acc, c.where)]
        out, acc_out = gpu.buffer(c.q.nbytes), gpu.from_numpy(np.full(c.acc.shape, -3.0, np.float32))
        held.append((b, out, acc_out))
        L.check(lib.styx_op_attn_decode_batch(
            gpu.h, C.byref(kv), b[0].ptr, b[1].ptr, c.nh, b[2].ptr, b[3].ptr, b[4].ptr, b[5].ptr, b[6].ptr, EPS,
            b[7].ptr, c.n_rope, c.scale, c.decay, b[8].ptr, acc_out.ptr, b[9].ptr, out.ptr, ws.ptr, ws.nbytes))
    gpu.sync()
    for c, (b, out, acc_out) in zip(cases, held):
        check_attn(c, (out.download(np.float32).reshape(c.q.shape), acc_out.download(np.float32).reshape(c.acc.shape),
                       b[9].download(np.int32).reshape(c.where.shape), c.bufs[0].download(c.dt).reshape(c.k.shape),
                       c.bufs[1].download(c.dt).reshape(c.v.shape)))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_attn_long_context_split(gpu, f16):
    rng = np.random.default_rng(6)
    c = Case(rng, f16, [20011, 5], 1, 8, 128, 256)
    check_attn(c, run_attn(gpu, c))


@pytest.mark.gpu
@pytest.mark.parametrize("in_place,with_acc_in", [(True, True), (False, False)])
def test_attn_accumulator_forms(gpu, in_place, with_acc_in):
    rng = np.random.default_rng(7)
    c = Case(rng, False, [90, 0, 300], 2, 8, 128, 64)
    check_attn(c, run_attn(gpu, c, in_place=in_place, with_acc_in=with_acc_in), in_place=in_place,
               with_acc_in=with_acc_in)


@pytest.mark.gpu
@pytest.mark.parametrize("scored", [True, False])
def test_attn_positions_with_and_without_weights(gpu, scored):
    """slot_pos left out of a call with weights; given to one without."""
    rng = np.random.default_rng(23)
    c = Case(rng, False, [40, 0, 77], 2, 4, 64, 32)
    kv = c.kv(gpu)
    b = [gpu.from_numpy(x) for x in (c.lens, c.pos, c.q, c.kn, c.vn, c.qw, c.kw, c.rope, c.where)]
    out, acc_out = gpu.buffer(c.q.nbytes), gpu.from_numpy(np.full(c.acc.shape, -3.0, np.float32))
    acc = gpu.from_numpy(c.acc)
    nbytes = gpu.lib.styx_op_attn_batch_ws_bytes(C.byref(kv), c.nh, int(scored))
    ws = gpu.buffer(nbytes)
    L.check(gpu.lib.styx_op_attn_decode_batch(
        gpu.h, C.byref(kv), b[0].ptr, b[1].ptr, c.nh, b[2].ptr, b[3].ptr, b[4].ptr, b[5].ptr, b[6].ptr, EPS, b[7].ptr,
        c.n_rope, c.scale, c.decay, acc.ptr if scored else None, acc_out.ptr if scored else None,
        None if scored else b[8].ptr, out.ptr, ws.ptr, nbytes))
    gpu.sync()
    where = b[8].download(np.int32).reshape(c.where.shape)
    if scored:
        assert np.array_equal(where, c.where)
        for i in range(c.B):
            where[i, :, c.lens[i]] = c.pos[i]  # (what check_attn looks for)
    else:
        want = c.where.copy()
        for i in range(c.B):
            want[i, :, c.lens[i]] = c.pos[i]
        assert np.array_equal(where, want)
    check_attn(c, (out.download(np.float32).reshape(c.q.shape), acc_out.download(np.float32).reshape(c.acc.shape), where,
                   c.bufs[0].download(c.dt).reshape(c.k.shape), c.bufs[1].download(c.dt).reshape(c.v.shape)),
               scored=scored)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_attn_rows_in_pages_outside_the_pool_are_not_seen(gpu, f16):
    """Entries below 0 and past the pool: in the middle, at the new row, and
    for a whole sequence (nothing seen: output 0, no weight)."""
    rng = np.random.default_rng(8)
    c = Case(rng, f16, [200, 100, 40], 2, 4, 128, 16)
    c.table[0, 3], c.table[0, 7] = -5, c.n_pages
    c.table[1, 100 // 16] = 2 ** 31 - 1
    c.table[2, :] = -1
    check_attn(c, run_attn(gpu, c))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_attn_stale_rows_do_not_matter(gpu, f16):
    """Rows past the new one, in the last page and in free pages, may hold
    anything: NaN and infinities there change nothing."""
    rng = np.random.default_rng(9)
    c = Case(rng, f16, [37, 0, 130], 2, 8, 64, 64)
    live = np.zeros(len(c.k), bool)
    for b in range(c.B):
        live[c.rows(b, int(c.lens[b]))] = True
    c.k[~live], c.v[~live] = np.nan, np.inf
    check_attn(c, run_attn(gpu, c))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_attn_infinite_value_row(gpu, f16):
    """A V value that is infinite makes its dimension infinite (f16 caches,
    whose factors come in two pieces: not finite) for every head that weighs
    the row, and only that one."""
    rng = np.random.default_rng(10)
    c = Case(rng, f16, [50], 1, 8, 128, 16)
    c.v[c.rows(0, 50)[20], 0, 5] = np.inf
    out = run_attn(gpu, c)[0]
    assert np.isposinf(out[0, :, 5]).all() if not f16 else not np.isfinite(out[0, :, 5]).any()
    assert np.isfinite(np.delete(out, 5, axis=2)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-6, 1e-3, 300.0])
def test_attn_f16_queries_of_any_size(gpu, size):
    """Without norms a query may be far from 1: its two f16 pieces still
    carry 22 bits."""
    rng = np.random.default_rng(11)
    c = Case(rng, True, [200], 2, 4, 128, 64, norms=False)
    c.q *= np.float32(size)
    c.scale = 1.0 / size / np.sqrt(c.hd)
    check_attn(c, run_attn(gpu, c))


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("norms", [False, True])
def test_attn_appended_f16_rows_are_rounded_by_way_of_f32(gpu, norms, hd):
    """Bit for bit: of 2^18 values some ten lie so near the middle of two f16
    values that rounding the f64 row directly gives the other one.  The two f64
    rows differ by less than 2^-44 of their head's largest value (64 roundings
    of 2^-53 and the order of the sums), so values that near to the middle of
    two f32 values may go either way."""
    rng = np.random.default_rng(14)
    c = Case(rng, True, list(range(1, 65)) * 2, 2 ** 11 // hd, 1, hd, 16, norms=norms)
    kp = run_attn(gpu, c, scored=False)[3]
    direct = 0
    for b in range(c.B):
        row, p = c.rows(b, c.lens[b] + 1)[-1], int(c.pos[b])
        for j in range(c.nkv):
            k64 = c.head(c.kn[b, j], c.kw, p)
            near = 2.0 ** -44 * np.abs(k64).max()
            k32 = k64.astype(np.float32)
            sure = (k64 - near).astype(np.float32) == (k64 + near).astype(np.float32)
            assert np.array_equal(kp[row, j][sure], k32.astype(np.float16)[sure])
            direct += int(np.sum(sure & (k64.astype(np.float16) != k32.astype(np.float16))))
    assert direct > 0


@pytest.mark.gpu
@pytest.mark.parametrize("f16,hd", [(True, 256), (True, 64), (False, 128)])
def test_attn_pools_past_32_bit_offsets(gpu, f16, hd):
    """Rows more than 2^32 bytes (2^31 elements) into the pools."""
    rng = np.random.default_rng(12)
    c = Case(rng, f16, [70], 8, 2, hd, 32)
    far = 2 ** 31 // (c.nkv * c.hd * c.page) + 1  # pages before the used ones
    n_pages = far + c.n_pages
    size = np.dtype(c.dt).itemsize
    nb = n_pages * c.page * c.nkv * c.hd * size
    pools = [gpu.buffer(nb), gpu.buffer(nb)]
    off = far * c.page * c.nkv * c.hd * size
    for p, x in zip(pools, (c.k, c.v)):
        p.upload(x, off)
    table = gpu.from_numpy(np.where(c.table >= 0, c.table + far, c.table).astype(np.int32))
    kv = L.KvCache(L.F16 if f16 else L.F32, 1, c.nkv, c.hd, c.page, n_pages, c.table_len, pools[0].ptr, pools[1].ptr, table.ptr)
    b = [gpu.from_numpy(x) for x in (c.lens, c.pos, c.q, c.kn, c.vn, c.qw, c.kw, c.rope, c.acc, c.where)]
    out = gpu.buffer(c.q.nbytes)
    acc_out = gpu.from_numpy(np.full(c.acc.shape, -3.0, np.float32))
    nbytes = gpu.lib.styx_op_attn_batch_ws_bytes(C.byref(kv), c.nh, 1)
    ws = gpu.buffer(nbytes)
    L.check(gpu.lib.styx_op_attn_decode_batch(
        gpu.h, C.byref(kv), b[0].ptr, b[1].ptr, c.nh, b[2].ptr, b[3].ptr, b[4].ptr, b[5].ptr, b[6].ptr, EPS, b[7].ptr,
        c.n_rope, c.scale, c.decay, b[8].ptr, acc_out.ptr, b[9].ptr, out.ptr, ws.ptr, nbytes))
    gpu.sync()
    got = (out.download(np.float32).reshape(c.q.shape), acc_out.download(np.float32).reshape(c.acc.shape),
           b[9].download(np.int32).reshape(c.where.shape), pools[0].download(c.dt, c.k.size, off).reshape(c.k.shape),
           pools[1].download(c.dt, c.v.size, off).reshape(c.v.shape))
    check_attn(c, got)
    for p in pools:
        p.free()


# ---------------------------------------------------------------- evict ----
def run_evict(gpu, c, trigger, keep, recent, sinks, in_place=False):
    lib = gpu.lib
    kv = c.kv(gpu)
    ln, pos, acc, where = (gpu.from_numpy(x) for x in (c.lens, c.pos, c.acc, c.where))
    acc_out = acc if in_place else gpu.from_numpy(np.full(c.acc.shape, -3.0, np.float32))
    where_out = where if in_place else gpu.from_numpy(np.full(c.where.shape, -9, np.int32))
    len_out = ln if in_place else gpu.from_numpy(np.full(c.B, -77, np.int32))
    nbytes = lib.styx_op_kv_evict_ws_bytes(C.byref(kv), keep)
    assert nbytes > 0
    ws = gpu.from_numpy(np.full(nbytes, 0xFF, np.uint8))
    L.check(lib.styx_op_kv_evict(gpu.h, C.byref(kv), ln.ptr, pos.ptr, trigger, keep, recent, sinks, acc.ptr, acc_out.ptr,
                                 where.ptr, where_out.ptr, len_out.ptr, ws.ptr, nbytes))
    gpu.sync()
    return (acc_out.download(np.float32).reshape(c.acc.shape), where_out.download(np.int32).reshape(c.where.shape),
            len_out.download(np.int32, c.B), c.bufs[0].download(c.dt).reshape(c.k.shape),
            c.bufs[1].download(c.dt).reshape(c.v.shape))


def want_evict(c, trigger, keep, recent, sinks, in_place=False):
    acc = c.acc.copy() if in_place else np.full(c.acc.shape, -3.0, np.float32)
    where = c.where.copy() if in_place else np.full(c.where.shape, -9, np.int32)
    lens, k, v = c.lens.copy(), c.k.copy(), c.v.copy()
    for b in range(c.B):
        n = int(c.lens[b])
        if n < 0 or n > c.cap:
            continue
        if n <= trigger:
            acc[b, :, :n], where[b, :, :n] = c.acc[b, :, :n], c.where[b, :, :n]
            continue
        lens[b] = keep
        rows = c.rows(b, n)
        for j in range(c.nkv):
            a, p = c.acc[b, j, :n].astype(np.float64), c.where[b, j, :n].astype(np.int64)
            guarded = (p > int(c.pos[b]) - recent) | (p < sinks)
            nan = np.isnan(a)
            order = sorted(range(n), key=lambda t: (not guarded[t], not guarded[t] and nan[t],
                                                    0.0 if guarded[t] or nan[t] else -a[t], t))
            stays = np.zeros(n, bool)
            stays[order[:keep]] = True
            src = np.arange(keep)
            src[~stays[:keep]] = keep + np.nonzero(stays[keep:])[0]
            acc[b, j, :keep], where[b, j, :keep] = c.acc[b, j, src], c.where[b, j, src]
            for t in np.nonzero(src != np.arange(keep))[0]:
                if rows[t] >= 0 and rows[src[t]] >= 0:
                    k[rows[t], j], v[rows[t], j] = c.k[rows[src[t]], j], c.v[rows[src[t]], j]
    return acc, where, lens, k, v


def same(got, want):
    for g, w, name in zip(got, want, ("acc", "slot_pos", "len", "K", "V")):
        assert np.array_equal(g.view(np.uint8), w.view(np.uint8)), name


def evict_case(rng, f16, lens, nkv, hd, page, **kw):
    """Positions in no order, weights with ties."""
    c = Case(rng, f16, lens, nkv, 1, hd, page, **kw)
    c.acc = (np.exp(2 * rng.standard_normal(c.acc.shape)).round(1)).astype(np.float32)
    for b in range(c.B):
        n = min(max(int(c.lens[b]), 0), c.cap)
        for j in range(nkv):
            c.where[b, j, :n] = np.sort(rng.choice(4 * n + 8, n, replace=False))
            half = n // 2
            c.where[b, j, :half] = rng.permutation(c.where[b, j, :half])
        c.pos[b] = c.where[b, :, :n].max() if n else 0
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("f16,hd", [(False, 64), (False, 128), (False, 256), (True, 64), (True, 128), (True, 256)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_types(gpu, f16, hd, in_place):
    rng = np.random.default_rng(hd)
    # shorter than, at and past the trigger; the whole capacity; skipped ones
    c = evict_case(rng, f16, [0, 40, 64, 65, 100, 300, 511, 600], 2, hd, 24, table_len=25)
    c.lens[4], c.lens[5] = -1, c.cap + 1
    same(run_evict(gpu, c, 64, 60, 10, 3, in_place), want_evict(c, 64, 60, 10, 3, in_place))


@pytest.mark.gpu
@pytest.mark.parametrize("keep,recent,sinks,trigger", [(1, 0, 0, 1), (1, 1, 0, 1), (1000, 0, 0, 1000),
                                                       (1024, 1000, 24, 1024), (1025, 7, 7, 1500),
                                                       (3000, 100, 4, 3000), (4999, 0, 5, 4999)])
def test_evict_budgets(gpu, keep, recent, sinks, trigger):
    rng = np.random.default_rng(keep)
    c = evict_case(rng, False, [5000, 2049, 1024], 2, 64, 100)
    same(run_evict(gpu, c, trigger, keep, recent, sinks), want_evict(c, trigger, keep, recent, sinks))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "zero", "negative_zero", "nan", "inf", "denormal"])
def test_evict_weights_at_their_limits(gpu, kind):
    """Ties go to the lower slot, -0 ties with 0, NaN leaves first."""
    rng = np.random.default_rng(3)
    c = evict_case(rng, True, [700], 3, 64, 64)
    r = rng.random(c.acc.shape)
    if kind == "equal":
        c.acc[:] = 0.25
    elif kind == "zero":
        c.acc[:] = np.where(r < 0.5, 0, c.acc)
    elif kind == "negative_zero":
        c.acc[:] = np.where(r < 0.5, -0.0, 0.0)
    elif kind == "nan":
        c.acc[:] = np.where(r < 0.4, np.nan, np.where(r < 0.5, -1.0, c.acc))
    elif kind == "inf":
        c.acc[:] = np.where(r < 0.3, np.inf, np.where(r < 0.6, -np.inf, c.acc))
    else:
        c.acc[:] = (1e-44 * (1 + (r * 8).astype(int))).astype(np.float32)
    same(run_evict(gpu, c, 256, 256, 16, 4), want_evict(c, 256, 256, 16, 4))


@pytest.mark.gpu
def test_evict_positions_that_repeat_keep_no_more_than_the_budget(gpu):
    """Every row in the recent window: the lower slots stay."""
    rng = np.random.default_rng(4)
    c = evict_case(rng, False, [500], 1, 128, 16)
    c.where[:] = 90
    c.pos[:] = 90
    same(run_evict(gpu, c, 100, 100, 50, 0), want_evict(c, 100, 100, 50, 0))


@pytest.mark.gpu
def test_evict_positions_at_the_ends_of_their_type(gpu):
    rng = np.random.default_rng(14)
    c = evict_case(rng, False, [500], 2, 64, 16)
    c.where[:, :, ::7] = -2 ** 31
    c.where[:, :, 1::9] = 2 ** 31 - 1
    c.pos[:] = -2 ** 31 + 5
    same(run_evict(gpu, c, 100, 100, 50, 10), want_evict(c, 100, 100, 50, 10))


@pytest.mark.gpu
def test_evict_rows_in_pages_outside_the_pool_do_not_move(gpu):
    rng = np.random.default_rng(13)
    c = evict_case(rng, False, [400, 300], 2, 128, 32)
    c.table[0, 1], c.table[0, 9], c.table[1, 8] = -1, c.n_pages + 3, -2 ** 31
    same(run_evict(gpu, c, 128, 128, 20, 2), want_evict(c, 128, 128, 20, 2))


@pytest.mark.gpu
def test_evict_long(gpu):
    rng = np.random.default_rng(15)
    c = evict_case(rng, True, [40000, 39999], 1, 64, 512)
    same(run_evict(gpu, c, 10000, 10000, 500, 4), want_evict(c, 10000, 10000, 500, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("keep,in_place", [(1, False), (100, True), (16384, False), (16385, True), (25000, False),
                                           (36000, True)])
@pytest.mark.parametrize("weights", ["drawn", "few", "equal"])
def test_evict_caches_of_several_parts(gpu, keep, in_place, weights):
    """Past 16K slots a head is selected by several workgroups: ties that run
    over their borders, sequences that end inside a part or do not reach it."""
    rng = np.random.default_rng(keep)
    lens = [36863, 100, keep + 1, 16384 * 2 + 3, 20000]
    c = evict_case(rng, True, lens * (20 if keep == 25000 and weights == "few" else 1), 1, 64, 512, table_len=72)
    if weights == "few":
        c.acc = rng.integers(0, 3, c.acc.shape).astype(np.float32)
    elif weights == "equal":
        c.acc[:] = 1.5
    recent, sinks = min(keep // 2, 300), min(keep // 4, 4)
    same(run_evict(gpu, c, keep, keep, recent, sinks, in_place), want_evict(c, keep, keep, recent, sinks, in_place))


# ------------------------------------------------------------ refusals -----
def cache(**kw):
    d = dict(type=L.F32, n_seq=2, nkv=2, hd=128, page_tokens=16, n_pages=4, table_len=2, kpool=256, vpool=256,
             page_table=256)
    d.update(kw)
    return L.KvCache(*(d[f] for f, _ in L.KvCache._fields_))


BAD_SHAPES = [dict(type=L.Q8_0), dict(type=30), dict(n_seq=0), dict(nkv=0), dict(hd=96), dict(hd=0),
              dict(page_tokens=0), dict(n_pages=0), dict(table_len=0), dict(table_len=2 ** 28, page_tokens=2 ** 28),
              dict(n_pages=2 ** 30, page_tokens=4), dict(n_seq=2 ** 24), dict(n_seq=-1)]
# what only the eviction refuses: more than 2^26 slots
LONG = dict(table_len=2 ** 23, page_tokens=16)


@pytest.mark.parametrize("kw", BAD_SHAPES)
def test_workspace_of_refused_shapes_is_0(kw):
    lib = L.load()
    assert lib.styx_op_attn_batch_ws_bytes(C.byref(cache(**kw)), 16, 1) == 0
    assert lib.styx_op_kv_evict_ws_bytes(C.byref(cache(**kw)), 8) == 0


def test_workspace_sizes():
    lib = L.load()
    assert lib.styx_op_attn_batch_ws_bytes(None, 16, 1) == 0
    assert lib.styx_op_kv_evict_ws_bytes(None, 16) == 0
    for nh in (0, -2, 3, 34):
        assert lib.styx_op_attn_batch_ws_bytes(C.byref(cache()), nh, 1) == 0
    for keep in (0, -1, 33):
        assert lib.styx_op_kv_evict_ws_bytes(C.byref(cache()), keep) == 0
    plain = lib.styx_op_attn_batch_ws_bytes(C.byref(cache()), 16, 0)
    # scores: a float per slot (in multiples of 64) and query head
    assert lib.styx_op_attn_batch_ws_bytes(C.byref(cache()), 16, 1) == plain + 2 * 16 * 64 * 4
    assert lib.styx_op_kv_evict_ws_bytes(C.byref(cache()), 32) >= 2 * 2 * 32 * 4


def test_eviction_is_refused_past_its_longest_cache():
    lib = L.load()
    assert lib.styx_op_kv_evict_ws_bytes(C.byref(cache(**LONG)), 8) == 0
    assert lib.styx_op_attn_batch_ws_bytes(C.byref(cache(**LONG)), 16, 0) > 0
    assert lib.styx_op_kv_evict_ws_bytes(C.byref(cache(table_len=2 ** 22, page_tokens=16)), 8) > 0


def test_no_gpu_is_refused():
    lib = L.load()
    assert lib.styx_op_attn_decode_batch(None, None, *[None] * 2, 8, *[None] * 5, EPS, None, 1, 1.0, 1.0,
                                         *[None] * 5, 0) == -1
    assert lib.styx_op_kv_evict(None, None, None, None, 1, 1, 0, 0, *[None] * 6, 0) == -1


@pytest.mark.gpu
def test_attn_refusals(gpu):
    z = gpu.zeros(1 << 16)
    p = z.ptr

    def call(kv=None, nh=16, len=p, pos=p, q=p, k=p, v=p, rope=p, n_rope=4, acc_in=p, acc_out=p, out=p, ws=p,
             ws_bytes=None):
        kv = cache(kpool=p, vpool=p, page_table=p) if kv is None else kv
        if ws_bytes is None:
            ws_bytes = gpu.lib.styx_op_attn_batch_ws_bytes(C.byref(kv), nh, int(bool(acc_out)))
        rc = gpu.lib.styx_op_attn_decode_batch(gpu.h, C.byref(kv), len, pos, nh, q, k, v, None, None, EPS, rope, n_rope,
                                               0.1, 1.0, acc_in, acc_out, None, out, ws, ws_bytes)
        return rc, gpu.lib.styx_last_error().decode()

    for kw in BAD_SHAPES:
        rc, msg = call(kv=cache(**{**dict(kpool=p, vpool=p, page_table=p), **kw}))
        assert rc == -1 and "styx_op_attn_decode_batch" in msg
    for name in ("len", "pos", "q", "k", "v", "rope", "out"):
        assert call(**{name: None})[0] == -1, name
    for kw in (dict(kpool=None), dict(vpool=None), dict(page_table=None), dict(kpool=p + 4), dict(vpool=p + 8)):
        assert call(kv=cache(**{**dict(kpool=p, vpool=p, page_table=p), **kw}))[0] == -1, kw
    for nh in (0, 3, 34, -2):
        assert call(nh=nh, ws_bytes=1 << 16)[0] == -1
    assert call(n_rope=0)[0] == -1
    assert call(acc_out=None)[0] == -1
    need = gpu.lib.styx_op_attn_batch_ws_bytes(C.byref(cache()), 16, 1)
    rc, msg = call(ws_bytes=need - 1)
    assert rc == -1 and str(need) in msg
    assert call(ws=None)[0] == -1 and call(ws=p + 4)[0] == -1
    gpu.sync()


@pytest.mark.gpu
def test_evict_refusals(gpu):
    z = gpu.zeros(1 << 16)
    p = z.ptr

    def call(kv=None, trigger=8, keep=8, recent=2, sinks=2, ws=p, ws_bytes=1 << 16, **kw):
        kv = cache(kpool=p, vpool=p, page_table=p) if kv is None else kv
        a = dict(len=p, pos=p, acc_in=p, acc_out=p, pos_in=p, pos_out=p, len_out=p)
        a.update(kw)
        rc = gpu.lib.styx_op_kv_evict(gpu.h, C.byref(kv), a["len"], a["pos"], trigger, keep, recent, sinks, a["acc_in"],
                                      a["acc_out"], a["pos_in"], a["pos_out"], a["len_out"], ws, ws_bytes)
        return rc, gpu.lib.styx_last_error().decode()

    for kw in BAD_SHAPES:
        rc, msg = call(kv=cache(**{**dict(kpool=p, vpool=p, page_table=p), **kw}))
        assert rc == -1 and "styx_op_kv_evict" in msg
    for name in ("len", "pos", "acc_in", "acc_out", "pos_in", "pos_out", "len_out"):
        assert call(**{name: None})[0] == -1, name
    for kw in (dict(keep=0), dict(keep=33, trigger=33), dict(trigger=7), dict(recent=-1), dict(sinks=-1),
               dict(recent=7, sinks=2), dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1)):
        assert call(**kw)[0] == -1, kw
    rc, msg = call(kv=cache(kpool=p, vpool=p, page_table=p, **LONG))
    assert rc == -1 and "2^26" in msg
    assert call(ws_bytes=8)[0] == -1 and call(ws=None)[0] == -1 and call(ws=p + 8)[0] == -1
    gpu.sync()
