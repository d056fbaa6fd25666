"""The operators on new tokens together, through the Python package, as a program
that serves a batch runs them: prompts in parts beside single tokens, pages
handed out and taken back, eviction by the weights that prompts left, and the
single-token operators on the same cache.  Against the definitions in 64 bits
on the raw projections."""
from __future__ import annotations

import numpy as np
import pytest

from chunk_cases import E, E16
from styx_amd import _lib as L, rope_table

pytestmark = pytest.mark.gpu
EPS = 1e-6
NKV, GQA, HD, PAGE, B = 2, 4, 64, 16, 5
NH = NKV * GQA
SCALE = 1.0 / np.sqrt(HD)
N_POS = 400


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


class Serving:
    """Sequences' raw q, k, v rows, and the batch that holds them."""

    def __init__(self, gpu, f16, interleaved=False, n_rot=HD, n_pages=200):
        from styx_amd import KvBatch
        self.gpu, self.f16, self.inter, self.n_rot = gpu, f16, interleaved, n_rot
        self.rng = np.random.default_rng(21)
        self.table = rope_table(n_rot, N_POS, 1e4, L.ROPE_BANDS, 4.0, 64)
        self.rope = gpu.from_numpy(self.table)
        self.qw, self.kw = ((1 + 0.1 * self.rng.standard_normal(HD)).astype(np.float32) for _ in range(2))
        self.norms = [gpu.from_numpy(w) for w in (self.qw, self.kw)]
        self.kv = KvBatch(gpu, B, NKV, HD, PAGE, n_pages, 20, L.F16 if f16 else L.F32)
        self.kv.manage()
        self.rows = [[] for _ in range(B)]  # (q, k, v) of every token so far
        self.lens, self.pos = np.full(B, -1), np.zeros(B, int)

    def turned(self, x, w, p):
        x = x.astype(np.float64)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w
        i = np.arange(self.n_rot // 2)
        a, b = (2 * i, 2 * i + 1) if self.inter else (i, i + self.n_rot // 2)
        c, s = self.table[p, :, 0], self.table[p, :, 1]
        y = x.copy()
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
        return y

    def step(self, new, last=4, shared=None):
        """plan, append, attend, weigh; the chunk's counts, outputs [rows][NH][HD] and first rows."""
        new = np.asarray(new)
        self.lens = np.where((self.lens < 0) & (new > 0), 0, self.lens)
        self.kv.set(len=self.lens, pos=self.pos)
        ch = self.kv.plan(new, shared)
        n, width = ch.n_rows, (NH + 2 * NKV) * HD
        x = self.rng.standard_normal((max(n, 1), width)).astype(np.float32)
        qkv, q = self.gpu.from_numpy(x), self.gpu.zeros(4 * n * NH * HD)
        out, lse = self.gpu.zeros(4 * n * NH * HD), self.gpu.zeros(4 * n * NH)
        k, v = 4 * NH * HD, 4 * (NH + NKV) * HD
        self.kv.append(ch, NH, qkv, (qkv, k), (qkv, v), q, self.rope, N_POS, self.n_rot, self.inter, *self.norms, EPS,
                       ldq=width, ldk=width, ldv=width)
        self.kv.attend_chunk(ch, NH, q, out, SCALE, lse=lse)
        self.kv.weigh(ch, NH, q, lse, SCALE, last, decay=0.5)
        counts = ch.counts()
        first = np.cumsum(np.maximum(new, 0)) - np.maximum(new, 0)
        for b in range(B):
            self.rows[b] += [x[first[b] + i].reshape(-1, HD) for i in range(counts[b])]
        self.lens, self.pos = self.lens + counts, self.pos + counts
        res = out.download(np.float32)[:n * NH * HD].reshape(n, NH, HD)
        for buf in (qkv, q, out, lse):
            buf.free()
        ch.free()
        return counts, res, first

    def weights(self, b, i):
        """Token i's softmax weights [NH][i + 1] over the tokens up to it, nothing evicted."""
        k = np.stack([self.turned(r[NH:NH + NKV], self.kw, t) for t, r in enumerate(self.rows[b][:i + 1])])
        q = self.turned(self.rows[b][i][:NH], self.qw, i)
        s = np.stack([k[:, h // GQA] @ q[h] * SCALE for h in range(NH)])
        w = np.exp(s - s.max(1, keepdims=True))
        return w / w.sum(1, keepdims=True)

    def want(self, b, i):
        w = self.weights(b, i)
        v = np.stack([r[NH + NKV:] for r in self.rows[b][:i + 1]]).astype(np.float64)
        return np.stack([w[h] @ v[:, h // GQA] for h in range(NH)])

    def near(self, got, b, i):
        """q, K and V are off by their roundings (2 E; f16 caches E16 of K and V): a score by (2 + HD + 8) E |q||k|
        scale, |q|, |k| <= 1.5 sqrt(HD) under the norm (f16: E16 times as much more), a weight by twice that and
        (n + 40) E, an output by its weights' and V's (|V| < 6)."""
        ds = ((HD + 10) * E + (E16 if self.f16 else 0)) * 2.25 * HD * SCALE * 1.2 ** 2  # (the table's gain is 1)
        tol = 6 * (2 * ds + 2 * (i + 41) * E + (E16 if self.f16 else 0))
        d = np.abs(got - self.want(b, i)).max()
        assert d <= tol, (b, i, d, tol)

    def owned(self):
        """Pages of the sequences and of the stack: each once."""
        held, n_free = self.kv.held.download(np.int32, B), int(self.kv.n_free.download(np.int32, 1)[0])
        table = self.kv.table.download(np.int32).reshape(B, -1)
        pages = [int(p) for b in range(B) for p in table[b, :held[b]]]
        assert all((table[b, held[b]:] == -1).all() for b in range(B))
        pages += self.kv.free_pages.download(np.int32, n_free).tolist()
        assert sorted(pages) == list(range(self.kv.c.n_pages))
        return held, n_free


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("layout", [(False, HD), (True, HD), (False, 24)])
def test_prompts_in_parts_beside_single_tokens(gpu, f16, layout):
    s = Serving(gpu, f16, *layout)
    for new in ([40, 7, 0, 0, 0], [23, 1, 50, 0, 1], [1, 1, 30, 0, 16], [1, 1, 1, 9, 1]):
        counts, out, first = s.step(new)
        assert counts.tolist() == new
        for b in range(B):
            n = len(s.rows[b])
            for i in {0, new[b] // 2, new[b] - 1} if new[b] else ():
                s.near(out[first[b] + i], b, n - new[b] + i)
        held, _ = s.owned()
        assert held.tolist() == [-(-len(r) // PAGE) for r in s.rows]
    # accumulated weights: 0.5 of what was there and the last 4 tokens' in every step that had any
    acc = s.kv.acc.download(np.float32).reshape(B, NKV, -1)
    want = np.zeros(acc.shape)
    at = np.zeros(B, int)
    for new in ([40, 7, 0, 0, 0], [23, 1, 50, 0, 1], [1, 1, 30, 0, 16], [1, 1, 1, 9, 1]):
        for b in range(B):
            if new[b]:
                want[b] *= 0.5
                for i in range(max(0, new[b] - 4), new[b]):
                    w = s.weights(b, at[b] + i)
                    want[b, :, :w.shape[1]] += w.reshape(NKV, GQA, -1).sum(1)
                at[b] += new[b]
    # a weight's relative error: as in near(), twice (its own and its lse's)
    ds = ((HD + 10) * E + (E16 if f16 else 0)) * 2.25 * HD * SCALE * 1.2 ** 2
    assert (np.abs(acc - want) <= (4 * ds + 200 * E) * want).all()
    where = s.kv.slot_pos.download(np.int32).reshape(B, NKV, -1)
    for b in range(B):
        assert (where[b, :, :at[b]] == np.arange(at[b])).all()


@pytest.mark.parametrize("f16", [False, True])
def test_a_single_token_is_what_the_single_token_operator_gives(gpu, f16):
    """The same cache, half the sequences by either: outputs, weights and appended rows."""
    s = Serving(gpu, f16)
    s.step([40, 17, 64, 1, 33])
    acc0 = s.kv.acc.download(np.uint8)
    pools0 = [p.download(np.uint8) for p in (s.kv.kpool, s.kv.vpool)]
    where0 = s.kv.slot_pos.download(np.uint8)
    lens, pos = s.lens.copy(), s.pos.copy()
    _, out, _ = s.step([1] * B, last=1)
    acc1, where1 = s.kv.acc.download(np.float32), s.kv.slot_pos.download(np.int32)
    pools1 = [p.download(np.uint8) for p in (s.kv.kpool, s.kv.vpool)]
    for buf, x in ((s.kv.acc, acc0), (s.kv.slot_pos, where0), (s.kv.kpool, pools0[0]), (s.kv.vpool, pools0[1])):
        buf.upload(x)
    s.kv.set(len=lens, pos=pos)  # (the pages of the new rows are there)
    x = np.stack([r[-1] for r in s.rows])
    q, k, v = (gpu.from_numpy(np.ascontiguousarray(x[:, a:b])) for a, b in ((0, NH), (NH, NH + NKV), (NH + NKV, NH + 2 * NKV)))
    o = gpu.zeros(4 * B * NH * HD)
    s.kv.attend(NH, q, k, v, o, s.rope, N_POS, SCALE, *s.norms, EPS, decay=0.5)
    got = o.download(np.float32).reshape(B, NH, HD)
    for b in range(B):
        s.near(out[b], b, len(s.rows[b]) - 1)
        s.near(got[b], b, len(s.rows[b]) - 1)
    # (the same rows up to the rounding of f64 sums in another order: a step of f32, or of f16)
    for p, want in zip((s.kv.kpool, s.kv.vpool), pools1):
        t = np.float16 if f16 else np.float32
        a, b = p.download(np.uint8).view(t), want.view(t)
        # (memory that no call has written holds anything, NaN among it)
        differ = a.view(np.uint16 if f16 else np.uint32) != b.view(np.uint16 if f16 else np.uint32)
        a, b = a[differ].astype(np.float64), b[differ].astype(np.float64)
        assert (np.abs(a - b) <= 2 * (E16 if f16 else E) * np.abs(b)).all()
    assert np.array_equal(s.kv.slot_pos.download(np.int32), where1)
    ds = ((HD + 10) * E + (E16 if f16 else 0)) * 2.25 * HD * SCALE * 1.2 ** 2
    assert (np.abs(s.kv.acc.download(np.float32) - acc1) <= (8 * ds + 400 * E) * acc1).all()


@pytest.mark.parametrize("f16", [False, True])
def test_eviction_after_a_prompt_gives_pages_back(gpu, f16):
    """Rows leave by the weights that the prompt's last tokens left; the next plan hands their pages on."""
    s = Serving(gpu, f16, n_pages=20)
    s.step([160, 0, 100, 0, 0])
    held, free = s.owned()
    assert held.tolist() == [10, 0, 7, 0, 0] and free == 3
    counts, _, _ = s.step([1, 150, 0, 0, 0])  # no pages for the second
    assert counts.tolist() == [1, 0, 0, 0, 0] and s.lens.tolist() == [161, 0, 100, -1, -1]
    acc = s.kv.acc.download(np.float32).reshape(B, NKV, -1)[:, :, :161]
    s.kv.set(len=s.lens, pos=s.pos - 1)
    s.kv.evict(trigger=120, keep=48, recent=8, sinks=2)
    s.lens = s.kv.lengths()
    assert s.lens.tolist() == [48, 0, 100, -1, -1]
    where = s.kv.slot_pos.download(np.int32).reshape(B, NKV, -1)[0, :, :48]
    for j in range(NKV):
        guarded = set(range(161 - 8, 161)) | {0, 1}
        rest = [t for t in np.argsort(-acc[0, j], kind="stable") if int(t) not in guarded]
        assert set(where[j].tolist()) == guarded | {int(t) for t in rest[:48 - len(guarded)]}
    counts, _, _ = s.step([5, 120, 0, 0, 0])
    assert counts.tolist() == [5, 120, 0, 0, 0]
    held, free = s.owned()
    assert held.tolist() == [4, 8, 7, 0, 0] and free == 1
    # an ended sequence's pages, but for those it shares
    s.lens[2] = -1
    s.step([0] * B, shared=[0, 0, 2, 0, 0])
    assert s.kv.held.download(np.int32, B).tolist() == [4, 8, 2, 0, 0]


def test_checks_of_the_python_calls(gpu):
    from styx_amd import KvBatch
    s = Serving(gpu, False)
    s.kv.set(len=[0] * B)
    with pytest.raises(ValueError):
        KvBatch(gpu, 1, 1, 64, 8, 4, 4).plan([1])
    with pytest.raises(ValueError):
        s.kv.plan([1, 2])
    with pytest.raises(ValueError):
        s.kv.plan([1] * B, shared=[0])
    ch = s.kv.plan([3] * B)
    small, big = gpu.zeros(64), gpu.zeros(4 * 15 * NH * HD)
    for bad in (dict(q=small), dict(out=small), dict(lse=small), dict(ldq=10 ** 6)):
        with pytest.raises(ValueError):
            s.kv.attend_chunk(ch, NH, **{**dict(q=big, out=big, scale=1.0, lse=None), **bad})
    for bad in (dict(q=small), dict(k=small), dict(v=small), dict(q_out=small), dict(n_pos=N_POS + 9000), dict(q_norm=gpu.zeros(16))):
        with pytest.raises(ValueError):
            s.kv.append(ch, NH, **{**dict(q=big, k=big, v=big, q_out=big, rope=s.rope, n_pos=N_POS), **bad})
    with pytest.raises(ValueError):
        s.kv.weigh(ch, NH, big, small, 1.0, 1)
    with pytest.raises(ValueError):
        KvBatch(gpu, B, NKV, HD, PAGE, 4, 4, scored=False).weigh(ch, NH, big, big, 1.0, 1)
