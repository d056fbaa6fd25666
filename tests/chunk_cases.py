"""Shared by the tests of the operators on new tokens of a batch: a paged cache
with its new tokens as numpy arrays, and the definitions in 64 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np

from styx_amd import _lib as L

E = 2.0 ** -24   # half a step of f32
E16 = 2.0 ** -11  # of f16
TINY16 = 2.0 ** -25  # half of f16's smallest step


class Chunked:
    """A cache whose sequences have lens[b] rows and counts[b] new ones, the new
    ones' K and V in place; rows of q in the order of `first` (default: packed)."""

    def __init__(self, rng, f16, q16, lens, counts, nkv, gqa, hd, page, first=None, n_rows=None, table_len=None, spare=2,
                 window=0, ld=None):
        self.f16, self.q16, self.nkv, self.gqa, self.nh, self.hd, self.page = f16, q16, nkv, gqa, nkv * gqa, hd, page
        self.dt, self.qt = (np.float16 if h else np.float32 for h in (f16, q16))
        self.lens, self.counts = np.array(lens, np.int32), np.array(counts, np.int32)
        self.B, self.window, self.scale = len(lens), window, 1.0 / np.sqrt(hd)
        total = [max(0, int(n)) + max(0, int(c)) for n, c in zip(lens, counts)]
        self.table_len = table_len or max(1, max(-(-t // page) for t in total))
        self.cap = self.table_len * page
        used = [min(-(-t // page), self.table_len) for t in total]
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
        c = np.maximum(self.counts, 0)
        self.first = (np.cumsum(c) - c).astype(np.int32) if first is None else np.array(first, np.int32)
        self.n_rows = int(c.sum()) if n_rows is None else n_rows
        self.ld = ld or self.nh * hd
        self.q = (2 * rng.standard_normal((self.n_rows, self.ld))).astype(self.qt)

    def heads(self, r):
        return self.q[r, :self.nh * self.hd].reshape(self.nh, self.hd).astype(np.float64)

    def rows(self, b):
        """Pool rows of the slots, -1 in pages outside the pool."""
        t = np.arange(int(self.lens[b]) + int(self.counts[b]))
        e = self.table[b, t // self.page]
        return np.where((e >= 0) & (e < self.n_pages), e.astype(np.int64) * self.page + t % self.page, -1)

    def taken(self, b):
        n, c, f = int(self.lens[b]), int(self.counts[b]), int(self.first[b])
        return n >= 0 and c > 0 and n + c <= self.cap and f >= 0 and f + c <= self.n_rows

    def seen(self, b, i, rows):
        at = int(self.lens[b]) + i
        t = np.arange(len(rows))
        return (t <= at) & (rows >= 0) & ((t > at - self.window) if self.window else True)

    def scores(self, b, i, j, rows):
        """Token i's scores over the slots it sees, for the heads of kv head j, and a bound of their
        error in f32: the sum's, the scale's roundings, and 2^-22 of the products for two f16 pieces."""
        q = self.heads(int(self.first[b]) + i)[j * self.gqa:(j + 1) * self.gqa]
        see = self.seen(b, i, rows)
        k = self.k[rows[see], j].astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            size = self.scale * (np.abs(q) @ np.abs(k).T)
            ds = (self.hd + 8) * E * size + (2.0 ** -22 * size if not self.q16 else 0)
            return q @ k.T * self.scale, ds, see

    def attend(self, b, i, j):
        """Outputs, their tolerance, lse and its tolerance for the heads of kv head j of token i.

        A weight's relative error is at most 2 ds + (n + 40) E (numerator and sum of n terms, exponentials,
        factors of merges), a value sum's once more the same for its additions; f16 q: its factors rounded to f16
        (E16, and TINY16 below its normal numbers) and the output too."""
        rows = self.rows(b)
        s, ds, see = self.scores(b, i, j, rows)
        if s.shape[1] == 0:
            z = np.zeros((self.gqa, self.hd))
            return z, z, np.full(self.gqa, -np.inf), np.zeros(self.gqa)
        v = self.v[rows[see], j].astype(np.float64)
        m = s.max(1, keepdims=True)
        p = np.exp(s - m)
        tot = p.sum(1, keepdims=True)
        out, n = (p / tot) @ v, s.shape[1]
        rel = 2 * ds.max(1, keepdims=True) + 2 * (n + 40) * E
        tol = rel * ((p / tot) @ np.abs(v)) + 1e-30
        if self.q16:
            tol += E16 * ((p / tot) @ np.abs(v)) + TINY16 * np.abs(v).sum(0) / tot + E16 * np.abs(out) + TINY16
        lse = (m + np.log(tot))[:, 0]
        return out, tol, lse, ds.max(1) + (n + 40) * E + 4 * E * np.abs(lse)

    def buffers(self, gpu):
        self.bufs = [gpu.from_numpy(x) for x in (self.k, self.v, self.table, self.first, self.counts, self.lens, self.q)]
        kv = L.KvCache(L.F16 if self.f16 else L.F32, self.B, self.nkv, self.hd, self.page, self.n_pages, self.table_len,
                       *(b.ptr for b in self.bufs[:3]))
        return kv, L.KvChunk(self.n_rows, *(b.ptr for b in self.bufs[3:6])), self.bufs[6]


def run_chunk(gpu, c, lse=True, ldo=None, fill=7.5):
    """(out [n_rows][ldo], lse [n_rows][nh]) of styx_op_attn_chunk; `fill` is what was there."""
    kv, ch, q = c.buffers(gpu)
    ldo = ldo or c.nh * c.hd
    out = gpu.from_numpy(np.full((max(c.n_rows, 1), ldo), fill, c.qt))
    l = gpu.from_numpy(np.full((max(c.n_rows, 1), c.nh), fill, np.float32))
    need = gpu.lib.styx_op_attn_chunk_ws_bytes(C.byref(kv), c.n_rows, c.nh)
    assert need > 0
    ws = gpu.from_numpy(np.full(need, 0xFF, np.uint8))
    L.check(gpu.lib.styx_op_attn_chunk(gpu.h, C.byref(kv), C.byref(ch), c.nh, L.F16 if c.q16 else L.F32, q.ptr, c.ld,
                                       c.scale, c.window, out.ptr, ldo, l.ptr if lse else None, ws.ptr, need))
    gpu.sync()
    return (out.download(c.qt).reshape(-1, ldo)[:c.n_rows], l.download(np.float32).reshape(-1, c.nh)[:c.n_rows])


def check_chunk(c, out, lse=None, fill=7.5, tokens=None):
    """Every row against its definition; rows of no sequence as they were."""
    mine = np.zeros(c.n_rows, bool)
    worst = 0.0
    for b in range(c.B):
        if not c.taken(b):
            continue
        f, n = int(c.first[b]), int(c.counts[b])
        mine[f:f + n] = True
        for i in (range(n) if tokens is None else tokens(n)):
            got = out[f + i, :c.nh * c.hd].reshape(c.nh, c.hd).astype(np.float64)
            for j in range(c.nkv):
                want, tol, wl, tl = c.attend(b, i, j)
                d = np.abs(got[j * c.gqa:(j + 1) * c.gqa] - want)
                assert (d <= tol).all(), (b, i, j, float((d - tol).max()), float(d.max()))
                worst = max(worst, float((d / (tol + 1e-300)).max()))
                if lse is not None:
                    gl = lse[f + i, j * c.gqa:(j + 1) * c.gqa].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        assert ((gl == wl) | (np.abs(gl - wl) <= tl)).all(), (b, i, j, gl, wl)
    assert (out[~mine] == fill).all()
    assert (out[:, c.nh * c.hd:] == fill).all()
    if lse is not None:
        assert (lse[~mine] == fill).all()
    return worst
