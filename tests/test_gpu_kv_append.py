"""styx_op_kv_append (no counterpart in the reference) against its definition in
64 bits, through the C ABI.  A value is the f64 result rounded to f32 and from
there to its type: off by E (1 + one step where an f64 sum in another order
moves the f32 rounding: 2 E) of its size, for f16 by E16 more (and by TINY16
below its normal numbers)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from chunk_cases import E, E16, TINY16
from styx_amd import _lib as L, rope_table

pytestmark = pytest.mark.gpu
EPS = 1e-6
NP = {L.F32: np.float32, L.F16: np.float16}


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


class Rows:
    def __init__(self, rng, t_in, t_q, t_c, n, nh, nkv, hd, n_rot, inter, norms=True, page=16, pad=0, spread=1.0):
        self.t_in, self.t_q, self.t_c = t_in, t_q, t_c
        self.n, self.nh, self.nkv, self.hd, self.n_rot, self.inter, self.page = n, nh, nkv, hd, n_rot, inter, page
        self.ld = (nh + 2 * nkv) * hd + pad
        self.qkv = (spread * rng.standard_normal((n, self.ld))).astype(NP[t_in])
        self.n_pages = -(-n // page) + 2
        self.row_at = rng.permutation(self.n_pages * page)[:n].astype(np.int32)
        self.row_pos = rng.integers(0, 500, n).astype(np.int32)
        self.table = rope_table(n_rot, 500, 1e4) if n_rot else None
        self.qw, self.kw = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) if norms else None for _ in range(2))
        self.pools = [rng.standard_normal((self.n_pages * page, nkv, hd)).astype(NP[t_c]) for _ in range(2)]

    def part(self, r, what):
        nh, nkv, hd = self.nh, self.nkv, self.hd
        a, b = dict(q=(0, nh), k=(nh, nh + nkv), v=(nh + nkv, nh + 2 * nkv))[what]
        return self.qkv[r, a * hd:b * hd].reshape(b - a, hd)

    def turned(self, r, what):
        x, w = self.part(r, what).astype(np.float64), self.qw if what == "q" else self.kw
        if w is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w
        if self.table is None:
            return x
        h = self.n_rot // 2
        i = np.arange(h)
        a, b = (2 * i, 2 * i + 1) if self.inter else (i, i + h)
        c, s = self.table[self.row_pos[r], :, 0], self.table[self.row_pos[r], :, 1]
        y = x.copy()
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, a] * s + x[:, b] * c
        return y

    def call(self, gpu, q=True, kv=True, in_place=False, ldo=None):
        B = [gpu.from_numpy(x) for x in (self.qkv, self.row_at, self.row_pos, *self.pools, np.zeros(1, np.int32))]
        tab = gpu.from_numpy(self.table) if self.table is not None else None
        qw, kw = (gpu.from_numpy(w) if w is not None else None for w in (self.qw, self.kw))
        ldo = self.ld if in_place else ldo or self.nh * self.hd
        out = B[0] if in_place else gpu.from_numpy(np.full((self.n, ldo), 7.5, NP[self.t_q]))
        c = L.KvCache(self.t_c, 1, self.nkv, self.hd, self.page, self.n_pages, 1, B[3].ptr, B[4].ptr, B[5].ptr)
        es = NP[self.t_in]().itemsize
        k = B[0].ptr + self.nh * self.hd * es
        rope = L.Rope(tab.ptr, 500, self.n_rot, int(self.inter)) if tab else None
        ptr = lambda b: b.ptr if b is not None else None  # noqa: E731
        L.check(gpu.lib.styx_op_kv_append(
            gpu.h, C.byref(c), self.n, B[2].ptr, B[1].ptr, self.nh, self.t_in, B[0].ptr if q else None, self.ld,
            k if kv else None, self.ld, k + self.nkv * self.hd * es if kv else None, self.ld, ptr(qw), ptr(kw), EPS,
            C.byref(rope) if rope else None, self.t_q, out.ptr if q else None, ldo))
        gpu.sync()
        return (out.download(NP[self.t_q]).reshape(self.n, ldo), B[3].download(NP[self.t_c]).reshape(self.pools[0].shape),
                B[4].download(NP[self.t_c]).reshape(self.pools[1].shape))

    def near(self, got, want, t):
        tol = (2 * E + (E16 if t == L.F16 else 0)) * np.abs(want) + (TINY16 if t == L.F16 else 1e-37) + 1e-14
        d = np.abs(got.astype(np.float64) - want)
        assert (d <= tol).all(), float((d - tol).max())

    def check(self, got, q=True, kv=True, in_place=False):
        out, kp, vp = got
        width = self.nh * self.hd
        left = np.ones(len(kp), bool)
        for r in range(self.n):
            there = self.table is None or 0 <= self.row_pos[r] < 500
            if q and there:
                self.near(out[r, :width].reshape(self.nh, self.hd), self.turned(r, "q"), self.t_q)
            elif q:
                assert np.array_equal(out[r, :width], self.qkv[r, :width]) if in_place else (out[r, :width] == 7.5).all()
            at = int(self.row_at[r])
            if kv and there and 0 <= at < len(kp):
                left[at] = False
                self.near(kp[at], self.turned(r, "k"), self.t_c)
                assert np.array_equal(vp[at], self.part(r, "v").astype(NP[self.t_c]))
        for p, before in zip((kp, vp), self.pools):
            assert np.array_equal(p[left], before[left])
        if in_place:
            assert np.array_equal(out[:, width:], self.qkv[:, width:])
        elif q:
            assert (out[:, width:] == 7.5).all()


TRIPLES = [(L.F32, L.F32, L.F32), (L.F32, L.F32, L.F16), (L.F32, L.F16, L.F16), (L.F16, L.F16, L.F16), (L.F16, L.F32, L.F16),
           (L.F16, L.F16, L.F32), (L.F32, L.F16, L.F32), (L.F16, L.F32, L.F32)]


@pytest.mark.parametrize("types", TRIPLES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("inter", [False, True])
def test_types_heads_and_layouts(gpu, types, hd, inter):
    r = Rows(np.random.default_rng(hd), *types, 19, 6, 2, hd, hd, inter)
    r.check(r.call(gpu))


@pytest.mark.parametrize("n_rot", [2, 6, 30, 64, 98, 126, 128])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("t", [L.F32, L.F16])
def test_part_of_the_head(gpu, n_rot, inter, t):
    r = Rows(np.random.default_rng(n_rot), t, t, t, 7, 5, 1, 128, n_rot, inter, pad=24)
    r.check(r.call(gpu, ldo=5 * 128 + 8))


@pytest.mark.parametrize("n,nh,nkv", [(1, 1, 1), (1, 64, 4), (3, 40, 40), (200, 3, 7), (1000, 8, 1)])
@pytest.mark.parametrize("t", [L.F32, L.F16])
def test_sizes(gpu, n, nh, nkv, t):
    r = Rows(np.random.default_rng(n), t, t, t, n, nh, nkv, 64, 64, False)
    r.check(r.call(gpu))


@pytest.mark.parametrize("t", [L.F32, L.F16])
@pytest.mark.parametrize("norms,n_rot", [(False, 64), (True, 0), (False, 0)])
def test_without_norms_and_without_positions(gpu, t, norms, n_rot):
    r = Rows(np.random.default_rng(1), t, t, t, 33, 4, 2, 128, n_rot, False, norms=norms)
    r.check(r.call(gpu))


@pytest.mark.parametrize("t", [L.F32, L.F16])
def test_q_alone_kv_alone_and_in_place(gpu, t):
    r = Rows(np.random.default_rng(2), t, t, t, 21, 8, 2, 128, 96, True)
    r.check(r.call(gpu, kv=False), kv=False)
    r.check(r.call(gpu, q=False), q=False)
    r.check(r.call(gpu, in_place=True), in_place=True)


@pytest.mark.parametrize("t", [L.F32, L.F16])
def test_rows_outside_the_table_or_the_pools(gpu, t):
    """A position outside the table: the row is left; a row outside the pools: q alone."""
    r = Rows(np.random.default_rng(3), t, t, t, 12, 4, 2, 64, 64, False)
    r.row_pos[[0, 5]] = [-1, 500]
    r.row_pos[7] = 2 ** 31 - 1
    r.row_at[[1, 5, 9]] = [-1, 3, r.n_pages * r.page]
    r.row_at[10] = -2 ** 31
    r.check(r.call(gpu))


@pytest.mark.parametrize("t", [L.F32, L.F16])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("norms", [False, True])
def test_rows_of_no_sequence_without_positions(gpu, t, in_place, norms):
    """No table: a row whose position is negative, as a plan marks rows of no sequence and of those that got no pages,
    is left all the same (in place it is asked for again, and a norm must not be applied twice)."""
    r = Rows(np.random.default_rng(9), t, t, t, 12, 4, 2, 64, 0, False, norms=norms, pad=8)
    r.row_pos[[0, 5, 11]] = [-1, -7, -2 ** 31]
    r.row_pos[3] = 2 ** 31 - 1  # (there is no table that it could be outside of)
    r.row_at[[0, 5]] = -1       # (the last one's place is a row of the pools)
    r.row_at[4] = -1
    out, kp, vp = r.call(gpu, in_place=in_place, ldo=4 * 64 + 8)
    left = np.ones(len(kp), bool)
    for i in range(12):
        if i in (0, 5, 11):
            assert np.array_equal(out[i], r.qkv[i]) if in_place else (out[i] == 7.5).all(), i
            continue
        r.near(out[i, :256].reshape(4, 64), r.turned(i, "q"), t)
        if i != 4:
            left[r.row_at[i]] = False
            r.near(kp[r.row_at[i]], r.turned(i, "k"), t)
            assert np.array_equal(vp[r.row_at[i]], r.part(i, "v"))
    for p, before in zip((kp, vp), r.pools):
        assert np.array_equal(p[left], before[left])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("t", [L.F32, L.F16])
def test_values_that_are_not_finite_stay_in_their_head(gpu, inter, norms, t):
    """Without the norm in their pair, and behind the dims that are turned in their dim."""
    r = Rows(np.random.default_rng(6), t, t, t, 6, 4, 2, 64, 32, inter, norms=norms)
    r.qkv[1, 64 + 5] = np.nan       # q head 1, a turned dim
    r.qkv[2, 40] = np.inf           # q head 0, one that is not
    r.qkv[3, 4 * 64 + 7] = -np.inf  # k head 0
    r.qkv[4, 6 * 64 + 9] = np.nan   # v head 0
    out, kp, vp = r.call(gpu)
    bad_q, bad_k, bad_v = (~np.isfinite(x.astype(np.float32)) for x in (out.reshape(6, 4, 64), kp[r.row_at], vp[r.row_at]))
    pair = lambda d: {d, d ^ 1} if inter else {d, (d + 16) % 32}  # noqa: E731
    # (under the norm NaN takes the whole head, an infinity makes the others 0)
    whole = set(range(64))
    for got, row, head, dims in ((bad_q, 1, 1, whole if norms else pair(5)), (bad_q, 2, 0, {40}), (bad_k, 3, 0, pair(7))):
        assert set(np.nonzero(got[row, head])[0].tolist()) == dims
        got[row, head] = False
    assert not bad_q.any() and not bad_k.any()
    assert np.argwhere(bad_v).tolist() == [[4, 0, 9]]


@pytest.mark.parametrize("t", [L.F32, L.F16])
def test_more_rows_than_workgroups_for_their_heads(gpu, t):
    r = Rows(np.random.default_rng(7), t, t, t, 2100, 5, 2, 64, 64, False)
    got = r.call(gpu)
    keep = np.random.default_rng(8).permutation(2100)[:60]
    for i in keep:
        r.near(got[0][i].reshape(5, 64), r.turned(i, "q"), t)
        r.near(got[1][r.row_at[i]], r.turned(i, "k"), t)
        assert np.array_equal(got[2][r.row_at[i]], r.part(i, "v"))


def test_small_and_zero_rows_under_the_norm(gpu):
    r = Rows(np.random.default_rng(4), L.F32, L.F32, L.F32, 9, 4, 2, 128, 128, False, spread=1e-5)
    r.qkv[4] = 0
    r.check(r.call(gpu))


def test_refusals(gpu):
    z = gpu.zeros(1 << 16)
    p = z.ptr
    kv = L.KvCache(L.F16, 1, 2, 64, 16, 2, 2, p, p, p)
    rope = L.Rope(p, 10, 64, 0)

    def call(kv=kv, n=1, pos=p, at=p + 256, nh=4, t=L.F32, q=p, ldq=256, k=p, ldk=128, v=p, ldv=128, rope=rope, tq=L.F32, o=p + 4096,
             ldo=256):
        return gpu.lib.styx_op_kv_append(gpu.h, C.byref(kv) if kv else None, n, pos, at, nh, t, q, ldq, k, ldk, v, ldv, None,
                                         None, 1e-6, C.byref(rope) if rope else None, tq, o, ldo)

    assert call(n=0) == 0
    for b in [dict(kv=None), dict(n=-1), dict(pos=None), dict(at=None), dict(nh=0), dict(nh=65537), dict(t=L.Q8_0), dict(tq=3),
              dict(q=None), dict(o=None), dict(k=None), dict(v=None), dict(q=None, o=None, k=None, v=None), dict(ldq=255),
              dict(ldq=258), dict(ldk=64), dict(ldv=130), dict(ldo=250), dict(q=p + 8), dict(o=p + 4), dict(k=p + 2),
              dict(rope=L.Rope(None, 10, 64, 0)), dict(rope=L.Rope(p, 0, 64, 0)), dict(rope=L.Rope(p, 10, 63, 0)),
              dict(rope=L.Rope(p, 10, 66, 0)), dict(rope=L.Rope(p, 10, 0, 0)), dict(rope=L.Rope(p + 8, 10, 64, 0)),
              dict(o=p, tq=L.F16), dict(o=p, ldo=260), dict(n=2 ** 31 - 1)]:
        assert call(**b) == -1, b
    gpu.sync()
