"""styx_op_attn_decode_batch where K, q or V are not finite: NaN scores reach
the outputs and weights of their heads wherever the row lies (among others,
alone in a wave's tile or in a workgroup's piece, the only one), and an
infinite value is never lost.  Tolerances: tests/test_gpu_kv_batch.py."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_kv_batch import E, Case, run_attn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


def check(c, got, scored):
    """A head with a score that is NaN or +infinity: all NaN, its weights too.
    A score of -infinity: a row without weight (f16 caches, whose queries come
    in two pieces: or NaN)."""
    out, acc, _, kp, vp = got
    for b in range(c.B):
        n = int(c.lens[b])
        rows = c.rows(b, n + 1)
        for j in range(c.nkv):
            K, V = kp[rows, j].astype(np.float64), vp[rows, j].astype(np.float64)
            total, total_tol, broken, maybe = np.zeros(n + 1), np.zeros(n + 1), False, False
            for h in range(j * c.gqa, (j + 1) * c.gqa):
                with np.errstate(invalid="ignore"):
                    q = c.head(c.q[b, h], c.qw, int(c.pos[b]))
                    s = K @ q * c.scale
                if np.isnan(s).any() or np.isposinf(s).any():
                    assert np.isnan(out[b, h]).all(), (b, h)
                    broken = True
                    continue
                if c.f16 and np.isneginf(s).any() and np.isnan(out[b, h]).all():
                    maybe = True
                    continue
                fine = np.isfinite(s)
                if not fine.any():
                    assert not out[b, h].any(), (b, h)
                    continue
                w = np.where(fine, np.exp(s - s.max()), 0.0)
                w /= w.sum()
                size = (np.abs(K[fine]) @ np.abs(q)).max() * c.scale
                rel = 2 * size * ((c.hd + 8) * E + (2.0 ** -22 if c.f16 else 0.0)) + (n + 40) * E + \
                    (2.0 ** -21 if c.f16 else 0.0)
                ref, tol = w @ V, (rel + (n + 40) * E) * (w @ np.abs(V))
                assert np.all(np.abs(out[b, h] - ref) <= tol + 1e-30), (b, h)
                total += w
                total_tol += w * rel
            if not scored:
                continue
            got_acc = acc[b, j, :n + 1]
            if broken:
                assert np.isnan(got_acc).all(), (b, j)
            elif not (maybe and np.isnan(got_acc).all()):
                ref = c.decay * np.where(np.arange(n + 1) < n, c.acc[b, j, :n + 1].astype(np.float64), 0.0) + total
                assert np.all(np.abs(got_acc - ref) <= total_tol + (c.gqa + 4) * E * ref + 1e-12), (b, j)


# rows before the new one, and the slots whose K is not finite: an old row,
# the new one, the only one; the new row alone in a wave's tile (f32: 16 keys,
# f16: 32) and in a piece of its own; all rows of a wave, of a piece, of a head
PLACES = {"old": (50, [20]), "new": (50, [50]), "only": (0, [0]), "alone_in_16": (16, [16]),
          "alone_in_32": (32, [32]), "alone_in_piece": (64, [64]), "alone_in_later_piece": (640, [640]),
          "wave": (60, range(16, 32)), "wave_of_two": (120, range(32, 64)), "piece": (200, range(64, 128)),
          "last_piece": (70, range(64, 71)), "all": (300, range(301))}


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("place", PLACES)
def test_keys_that_are_not_finite(gpu, f16, scored, value, place):
    n, slots = PLACES[place]
    rng = np.random.default_rng(31)
    c = Case(rng, f16, [n, n], 2, 3, 128, 32, norms=False)
    rows = c.rows(0, n + 1)
    for t in slots:  # of kv head 1 of sequence 0; the others are checked beside it
        if t == n:
            c.kn[0, 1, 5] = value
        else:
            c.k[rows[t], 1, 5] = value
    with np.errstate(invalid="ignore"):
        check(c, run_attn(gpu, c, scored=scored), scored)


@pytest.mark.parametrize("f16", [False, True])
def test_a_finite_key_that_the_f16_cache_makes_infinite(gpu, f16):
    """70000 is past f16: the row is one of the above there, ordinary in f32."""
    rng = np.random.default_rng(32)
    c = Case(rng, f16, [64, 64], 1, 4, 64, 16, norms=False)
    c.kn[0, 0, 7] = 70000.0
    c.pos[:] = 0
    got = run_attn(gpu, c)
    assert np.isinf(got[3][c.rows(0, 65)[64], 0, 7]) == f16
    check(c, got, True)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("n", [0, 50, 700])
@pytest.mark.parametrize("hd,gqa", [(64, 1), (128, 5), (256, 16)])
def test_queries_that_are_nan(gpu, f16, scored, norms, n, hd, gqa):
    rng = np.random.default_rng(33)
    c = Case(rng, f16, [n, n], 2, gqa, hd, 32, norms=norms)
    c.q[0, gqa, 3] = np.nan  # the first query head of kv head 1
    check(c, run_attn(gpu, c, scored=scored), scored)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("low", [range(20, 21), range(0, 16), range(32, 64), range(64, 128), range(0, 192)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_values_of_rows_whose_factor_is_0(gpu, f16, low, value):
    """Scores 150 below the others', whose factor f32 holds as 0: what their V
    holds is still not lost, wherever these rows meet the others (in a tile,
    between waves, between pieces)."""
    rng = np.random.default_rng(34)
    c = Case(rng, f16, [200], 1, 1, 128, 16, norms=False)
    rows = c.rows(0, 201)
    q = c.head(c.q[0, 0], None, int(c.pos[0]))
    for t in low:
        c.k[rows[t], 0] = (-150.0 / (q @ q * c.scale) * q).astype(c.dt)
    keep = np.setdiff1d(np.arange(200), list(low))
    # each row alone, then all of them
    for some in ([low[0]], [low[-1]], list(low)):
        v = c.v.copy()
        c.v[rows[some], 0, 5] = value
        with np.errstate(invalid="ignore"):
            out, _, _, kp, vp = run_attn(gpu, c, scored=False)
        c.v = v
        assert not np.isfinite(out[0, 0, 5])
        K, V = (np.concatenate([p[rows[keep], 0], p[rows[200:], 0]]).astype(np.float64) for p in (kp, vp))
        s = K @ q * c.scale
        w = np.exp(s - s.max())
        w /= w.sum()
        size = (np.abs(K) @ np.abs(q)).max() * c.scale
        rel = 2 * size * ((c.hd + 8) * E + (2.0 ** -22 if f16 else 0.0)) + 240 * E + (2.0 ** -21 if f16 else 0.0)
        tol = (rel + 240 * E) * (w @ np.abs(V))
        others = np.arange(128) != 5
        assert np.all(np.abs(out[0, 0] - w @ V)[others] <= tol[others] + 1e-30)
