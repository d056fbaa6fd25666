"""The operators of a bounded-cache answer together, as a program runs them
(attend, evict, sample, step after step, through the Python package), and the
engine's sampled generation."""
from __future__ import annotations

import numpy as np
import pytest

from styx_amd import _lib as L
from test_gpu_kv_batch import Case, check_attn, same, want_evict
from test_gpu_sample import define, params

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


@pytest.mark.parametrize("f16,hd,page", [(False, 64, 16), (True, 128, 10)])
def test_answers_within_a_budget(gpu, f16, hd, page):
    """Four sequences, one of which pauses, for 70 tokens in caches of 48
    slots: each step's output, weights, positions, rows and evictions against
    the definitions on the state before it, and the tokens sampled from the
    outputs (taken as logits)."""
    from styx_amd import KvBatch, sample
    rng = np.random.default_rng(hd)
    lens = [5, 0, 23, 11]
    slots = 48 if page == 16 else 50
    c = Case(rng, f16, lens, 2, 4, hd, page, table_len=slots // page)
    used = c.B * c.table_len
    c.n_pages = used + 1
    c.table = rng.permutation(c.n_pages)[:used].reshape(c.B, -1).astype(np.int32)
    c.k, c.v = (rng.standard_normal((c.n_pages * page, c.nkv, hd)).astype(c.dt) for _ in range(2))
    c.n_rope = 128
    c.rope = np.empty((c.n_rope, hd // 2, 2), np.float64)
    L.load().styx_rope_table(1e6, hd, c.n_rope, c.rope.ctypes.data)
    for b in range(c.B):
        c.where[b, :, :lens[b]] = np.arange(lens[b])
    kv = KvBatch(gpu, c.B, c.nkv, hd, page, c.n_pages, c.table_len, L.F16 if f16 else L.F32)
    kv.set(table=c.table)
    for buf, a in ((kv.kpool, c.k), (kv.vpool, c.v), (kv.acc, c.acc), (kv.slot_pos, c.where)):
        buf.upload(a)
    rope, qw, kw = (gpu.from_numpy(a) for a in (c.rope, c.qw, c.kw))
    out = gpu.buffer(c.q.nbytes)

    def state():
        return (kv.acc.download(np.float32).reshape(c.acc.shape), kv.slot_pos.download(np.int32).reshape(c.where.shape),
                kv.kpool.download(c.dt).reshape(c.k.shape), kv.vpool.download(c.dt).reshape(c.v.shape))

    pos, n = np.array(lens, np.int32), np.array(lens, np.int32)
    evicted = 0
    for step in range(70):
        pause = 20 <= step < 30  # sequence 2 waits for its user
        c.lens, c.pos = n.copy(), pos.copy()
        c.lens[2] = -1 if pause else n[2]
        c.q, c.kn, c.vn = (rng.standard_normal(a.shape).astype(np.float32) for a in (c.q, c.kn, c.vn))
        kv.set(len=c.lens, pos=c.pos)
        out.upload(np.full(c.q.shape, 7.5, np.float32))
        b = [gpu.from_numpy(a) for a in (c.q, c.kn, c.vn)]
        kv.attend(c.nh, *b, out, rope, c.n_rope, c.scale, qw, kw, 1e-6, c.decay)
        o = out.download(np.float32).reshape(c.q.shape)
        acc, where, k, v = state()
        check_attn(c, (o, acc, where, k, v), in_place=True)
        c.acc, c.where, c.k, c.v = acc, where, k, v
        # the next tokens
        u = rng.random(c.B).astype(np.float32)
        par = [(0.8, 0, 0.9, 0.0), (1.0, 5, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 50, 0.95, 0.05)]
        tok, _, left = sample(gpu, out, c.nh * hd, par, u)
        for i, x in enumerate(o.reshape(c.B, -1)):
            assert (tok[i], left[i]) == tuple(np.array(define(x, params(par)[i], u[i]))[[0, 2]].astype(int)), (step, i)
        grown = np.where(c.lens >= 0, 1, 0).astype(np.int32)
        n, pos = n + grown, pos + grown
        # a cache of more than 40 rows goes back to 32
        c.lens, c.pos = n.copy(), (pos - 1).astype(np.int32)
        kv.set(len=c.lens, pos=c.pos)
        kv.evict(40, 32, recent=8, sinks=2)
        want = want_evict(c, 40, 32, 8, 2, in_place=True)
        acc, where, k, v = state()
        new = kv.lengths()
        same((acc, where, new, k, v), want)
        evicted += int((new < n).sum())
        c.acc, c.where, c.k, c.v, n = acc, where, k, v, new
        # what must stay is there: the newest 8 positions and the first 2
        for s in range(c.B):
            for j in range(c.nkv):
                have = set(where[s, j, :n[s]].tolist())
                assert len(have) == n[s]
                assert {int(p) for p in range(max(0, pos[s] - 8), pos[s])} | set(range(min(2, pos[s]))) <= have
    assert evicted >= 4 * 3
    kv.free()


def test_the_package_checks_what_it_is_given(gpu):
    from styx_amd import KvBatch, StyxError, sample
    kv = KvBatch(gpu, 2, 1, 64, 16, 4, 2, scored=False)
    with pytest.raises(ValueError):
        kv.set(len=[1, 2, 3])
    with pytest.raises(ValueError):
        kv.set(table=np.zeros((2, 3)))
    with pytest.raises(ValueError):
        kv.evict(8, 8)
    z = gpu.zeros(2 * 4 * 64 * 4)
    small = gpu.zeros(64)
    kv.set(len=[0, -1], pos=[0, 0], table=[[0, 1], [2, 3]])
    for bad in range(5):
        a = [z] * 5
        a[bad] = small
        with pytest.raises(ValueError):
            kv.attend(4, *a, 2, 0.125)
    with pytest.raises(StyxError):
        kv.attend(17, gpu.zeros(1 << 14), z, z, gpu.zeros(1 << 14), z, 1, 0.125)
    kv.attend(4, z, z, z, z, z, 1, 0.125)
    gpu.sync()
    with pytest.raises(ValueError):
        sample(gpu, z, 300, (1.0, 0, 1.0, 0.0), [0.5, 0.5])
    with pytest.raises(ValueError):
        sample(gpu, z, 30, [(1.0, 0, 1.0, 0.0)] * 3, [0.5, 0.5])
    with pytest.raises(StyxError):
        sample(gpu, z, 30, (1.0, 0, 1.0, 0.0), [0.5], ld=20)
    kv.free()


# ------------------------------------------------------------- engine ------
def model(gpu, **kw):
    from styx_amd import MoeModel, SynthConfig
    cfg = dict(n_layers=2, n_embd=512, n_heads=8, n_kv_heads=2, head_dim=64, n_expert=32, n_expert_used=4,
               n_ff_exp=256, n_vocab=2500, exp_mix=True, seed=77)
    opts = dict(n_ctx=128)
    for k, v in kw.items():
        (opts if k in ("n_ctx", "fuse", "use_graph", "expert_budget_mb", "arena") else cfg)[k] = v
    return MoeModel.synth(gpu, SynthConfig(**cfg), **opts)


PROMPT = [11, 400, 1500, 3, 77, 9, 1024, 2499]


@pytest.mark.parametrize("kw", [{}, dict(fuse=False, use_graph=False), dict(expert_budget_mb=2, arena=False)])
def test_sampled_generation_follows_the_logits(gpu, kw):
    """Every sampled token is the definition's for the logits that the engine
    gives for the tokens before it."""
    m = model(gpu, **kw)
    rng = np.random.default_rng(3)
    u = rng.random(24).astype(np.float32)
    s = dict(temperature=0.9, top_k=60, top_p=0.9, min_p=0.01)
    toks, lps, _, _ = m.generate_sampled(PROMPT, u, **s)
    par = params([(s["temperature"], s["top_k"], s["top_p"], s["min_p"])])[0]
    m.reset()
    m.generate(PROMPT, 1)  # the prompt again, as the sampled run read it
    for i in range(len(u)):
        lg = m.forward_token(int(toks[i - 1])) if i else None
        tok, lp = m.sample(float(u[i]), **s)
        assert tok == toks[i] and np.float32(lp) == lps[i], i
        if lg is not None:
            want, wlp, _, unit = define(lg, par, u[i])
            assert tok == want
            assert abs(lp - wlp) <= 2.0 ** -24 * abs(wlp) + 2.0 ** -50 + unit
    assert len(set(toks.tolist())) > 5
    m.close()


def test_temperature_0_is_greedy(gpu):
    m = model(gpu)
    greedy, _, _ = m.generate(PROMPT, 20)
    m.reset()
    toks, lps, _, _ = m.generate_sampled(PROMPT, np.full(20, 0.7), temperature=0.0)
    assert np.array_equal(toks, greedy) and not lps.any()
    # greedy decoding goes on from where the sampled tokens end
    m.reset()
    more, _, _ = m.generate(PROMPT, 26)
    m.reset()
    m.generate_sampled(PROMPT, np.zeros(20), temperature=0.0)
    m.forward_token(int(toks[-1]), want_logits=False)
    assert m.sample(0.5, temperature=0.0)[0] == more[20]
    assert np.array_equal(m.decode(5), more[21:26])
    m.close()


def test_sampling_leaves_the_state_alone(gpu):
    m = model(gpu)
    m.forward_token(5)
    a = [m.sample(x)[0] for x in (0.1, 0.5, 0.9, 0.1, 0.5, 0.9)]
    assert a[:3] == a[3:]
    lg = m.forward_token(a[0])
    m.reset()
    m.forward_token(5)
    assert np.array_equal(lg, m.forward_token(a[0]))
    m.close()


def test_sampling_refusals(gpu):
    import ctypes as C
    from styx_amd import StyxError
    m = model(gpu, n_ctx=16)
    with pytest.raises(StyxError, match="no token forwarded"):
        m.sample(0.5)
    m.forward_token(1)
    m.sample(0.5)
    m.reset()
    with pytest.raises(StyxError, match="no token forwarded"):
        m.sample(0.5)
    m.fill_kv(4)
    with pytest.raises(StyxError, match="no token forwarded"):
        m.sample(0.5)
    m.reset()
    with pytest.raises(StyxError, match="exceeds n_ctx"):
        m.generate_sampled(PROMPT, np.zeros(10))
    with pytest.raises(StyxError, match="bad argument"):
        m.generate_sampled([], np.zeros(2))
    with pytest.raises(StyxError, match="bad argument"):
        m.generate_sampled(PROMPT, np.zeros(0))
    with pytest.raises(StyxError, match="out of range"):
        m.generate_sampled([1, 99999], np.zeros(2))
    p = L.SampleParams(1.0, 0, 1.0, 0.0)
    assert gpu.lib.styx_moe_sample(m.h, None, 0.5, None, None) == -1
    assert gpu.lib.styx_moe_sample(None, C.byref(p), 0.5, None, None) == -1
    m.close()


def test_sampling_after_stage_timing_is_refused(gpu):
    """Its replays of the head overwrite the logits with those of another
    state; the next token brings them back."""
    from styx_amd import StyxError
    m = model(gpu)
    m.generate(PROMPT, 1)
    m.forward_token(5)
    m.time_stage("lm_head", 1)
    with pytest.raises(StyxError, match="no token forwarded"):
        m.sample(0.5)
    lg = m.forward_token(6)
    assert m.sample(0.5, temperature=0.0)[0] == int(np.argmax(lg))
    m.decode(2)
    m.sample(0.5)
    m.close()
