"""styx_op_sample (no counterpart in the reference) against its definition:
weights in whole units of 2^-44, so that which words stay and which one a
random number meets are decided by exact sums; tokens and counts are equal,
the log probability is off by its rounding to f32, the few roundings of the
quotient and the logarithm in f64, and by a unit in the weights where two
f64 exponentials round to different whole numbers (one over the word's
weight, and the words over their sum)."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

from styx_amd import _lib as L

ONE = 2.0 ** 44


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


def params(rows):
    """[(temperature, top_k, top_p, min_p)] as the device reads them."""
    a = np.zeros(len(rows), dtype=[("t", np.float32), ("k", np.int32), ("p", np.float32), ("m", np.float32)])
    for i, r in enumerate(rows):
        a[i] = r
    return a


def run(gpu, x, par, u, ld=None, extras=True, offset=0):
    """x [rows][n], laid out ld apart after `offset` floats."""
    rows, n = x.shape
    ld = ld or n
    buf = np.full(offset + rows * ld, 50.0, np.float32)
    for r in range(rows):
        buf[offset + r * ld:offset + r * ld + n] = x[r]
    b = [gpu.from_numpy(a) for a in (buf, par, np.asarray(u, np.float32))]
    tok, lp, nk = (gpu.from_numpy(np.full(rows + 1, v, t)) for v, t in ((77, np.uint32), (5.0, np.float32), (9, np.uint32)))
    nbytes = gpu.lib.styx_op_sample_ws_bytes(rows, n)
    ws = gpu.from_numpy(np.full(nbytes, 0xA5, np.uint8))
    L.check(gpu.lib.styx_op_sample(gpu.h, b[0].ptr + 4 * offset, ld, rows, n, b[1].ptr, len(par), b[2].ptr, tok.ptr,
                                   lp.ptr if extras else None, nk.ptr if extras else None, ws.ptr, nbytes))
    gpu.sync()
    tok, lp, nk = tok.download(np.uint32), lp.download(np.float32), nk.download(np.uint32)
    assert tok[rows] == 77 and lp[rows] == 5.0 and nk[rows] == 9
    return tok[:rows], lp[:rows], nk[:rows]


def define(x, par, u):
    """(token, logprob, n_kept) of one row by the definition, and how far a
    unit in every weight moves the log probability."""
    t, k, p, m = float(par["t"]), int(par["k"]), float(par["p"]), float(par["m"])
    ids = np.nonzero(x > -np.inf)[0]
    if len(ids) == 0:
        return 0xFFFFFFFF, -math.inf, 0, 0.0
    ids = ids[np.argsort(-x[ids].astype(np.float64), kind="stable")]
    if not t > 0:
        return int(ids[0]), 0.0, 1, 0.0
    v = x[ids].astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        d = np.where(v == v[0], 0.0, np.where(v[0] == np.inf, -np.inf, (v - v[0]) / t))
    w = np.rint(np.exp(d) * ONE).astype(np.int64)
    if k > 0:
        ids, w = ids[:k], w[:k]
    ids, w = ids[w > 0], w[w > 0]
    if p < 1:
        before = np.cumsum(w) - w
        keep = before.astype(np.float64) < p * float(w.sum())
        keep[0] = True
        ids, w = ids[keep], w[keep]
    if m > 0:
        keep = w.astype(np.float64) >= m * ONE
        keep[0] = True
        ids, w = ids[keep], w[keep]
    by = np.argsort(ids)
    ids, w = ids[by], w[by]
    run_, total = np.cumsum(w), int(w.sum())
    f = float(u) * float(total)
    at = min(int(f) if f > 0 else 0, total - 1)
    i = int(np.searchsorted(run_, at, side="right"))
    return int(ids[i]), math.log(int(w[i]) / total), len(ids), 1.0 / int(w[i]) + len(ids) / total


def check(gpu, x, par, u, **kw):
    got = run(gpu, x, par, u, **kw)
    for r in range(len(x)):
        tok, lp, nk, unit = define(x[r], par[0 if len(par) == 1 else r], u[r])
        assert got[0][r] == tok, (r, got[0][r], tok, got[2][r], nk)
        if kw.get("extras", True):
            assert got[2][r] == nk, (r, got[2][r], nk)
            assert got[1][r] == lp or abs(got[1][r] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -50 + unit, (r, got[1][r], lp)
    return got


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (1.3, 0, 0.95, 0.0), (1.0, 40, 1.0, 0.0), (0.9, 0, 1.0, 0.05),
            (1.0, 50, 0.9, 0.1), (0.0, 5, 0.5, 0.5), (2.0, 1000, 0.999, 0.001), (0.3, 1, 0.3, 0.0), (5.0, 0, 0.5, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 2047, 2048, 2049, 8192, 50257, 151936])
def test_settings_over_sizes(gpu, n):
    rng = np.random.default_rng(n)
    x = (2.5 * rng.standard_normal((len(SETTINGS), n))).astype(np.float32)
    check(gpu, x, params(SETTINGS), rng.random(len(SETTINGS)).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 33, 300, 1100])
def test_rows_with_settings_of_their_own(gpu, rows):
    rng = np.random.default_rng(rows)
    n = 5003 if rows < 1000 else 2500
    x = (2.0 * rng.standard_normal((rows, n))).astype(np.float32)
    par = params([SETTINGS[int(i)] for i in rng.integers(0, len(SETTINGS), rows)])
    check(gpu, x, par, rng.random(rows).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("step", [1 / 16, 1.0, 100.0])
def test_ties_go_to_the_lower_index(gpu, step):
    """Logits in steps: the border of top-k and top-p runs through words of
    one logit; a step of 100 makes them all equal."""
    rng = np.random.default_rng(1)
    x = (np.round(2 * rng.standard_normal((len(SETTINGS), 20000)) / step) * step + 0.0).astype(np.float32)
    if step == 100.0:
        x[:] = 3.25
    check(gpu, x, params(SETTINGS), rng.random(len(SETTINGS)).astype(np.float32))


@pytest.mark.gpu
def test_zeros_of_both_signs_are_one_logit(gpu):
    rng = np.random.default_rng(2)
    x = np.where(rng.random((4, 700)) < 0.5, -0.0, 0.0).astype(np.float32)
    check(gpu, x, params([(0.0, 0, 1, 0), (1.0, 5, 1, 0), (1.0, 0, 0.3, 0), (1.0, 7, 0.5, 0)]),
          rng.random(4).astype(np.float32))


@pytest.mark.gpu
def test_masked_words_infinities_and_nan(gpu):
    rng = np.random.default_rng(3)
    n, k = 3001, len(SETTINGS)
    rows = []
    for kind in range(6):
        x = (2 * rng.standard_normal((k, n))).astype(np.float32)
        if kind == 0:
            x[rng.random((k, n)) < 0.9] = -np.inf
        elif kind == 1:
            x[rng.random((k, n)) < 0.5] = np.nan
        elif kind == 2:
            x[:] = -np.inf
            x[:, 1234] = -80.0
        elif kind == 3:
            x[:, [7, 100, 2999]] = np.inf
        elif kind == 4:
            x[:] = np.where(rng.random((k, n)) < 0.5, -np.inf, np.nan)
        else:  # the type's ends
            x[rng.random((k, n)) < 0.3] = np.finfo(np.float32).min
            x[:, 5] = np.finfo(np.float32).max
        rows.append(x)
    x = np.concatenate(rows)
    u = rng.random(len(x)).astype(np.float32)
    got = check(gpu, x, params(SETTINGS * 6), u)
    assert (got[0][4 * k:5 * k] == 0xFFFFFFFF).all()


@pytest.mark.gpu
def test_settings_at_their_limits(gpu):
    inf, nan = math.inf, math.nan
    rng = np.random.default_rng(4)
    s = [(1.0, -3, 1.0, -1.0), (nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0), (inf, 0, 1.0, 0.0), (inf, 0, 0.5, 0.0),
         (1e-38, 0, 0.5, 0.0), (1e-45, 0, 1.0, 0.0), (1.0, 2 ** 31 - 1, 0.9, 0.0), (1.0, 0, 0.0, 0.0),
         (1.0, 0, -1.0, 0.0), (1.0, 0, nan, nan), (1.0, 0, 1e-30, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 7.0),
         (1.0, 0, 1.0, inf), (1.0, 4000, 0.99, 1e-20), (1.0, 3999, 1.0, 0.0), (1e30, 0, 0.9999, 0.0),
         (1.0, 1, 0.0, 2.0), (1.0, 2, 2.0, 0.0)]
    x = (3 * rng.standard_normal((len(s), 4000))).astype(np.float32)
    check(gpu, x, params(s), rng.random(len(s)).astype(np.float32))


@pytest.mark.gpu
def test_random_numbers_at_their_limits(gpu):
    rng = np.random.default_rng(5)
    u = np.array([0.0, -0.0, 2.0 ** -24, 1 - 2.0 ** -24, 1.0, 1.5, -0.5, math.nan, math.inf], np.float32)
    x = (rng.standard_normal((len(u), 3000))).astype(np.float32)
    for s in ((1.0, 0, 1.0, 0.0), (1.0, 30, 0.9, 0.0)):
        got = run(gpu, x, params([s]), u)
        for r in range(len(u)):
            # nan: 0; infinity: the last word that is left
            v = {True: 0.0}.get(math.isnan(u[r]), min(float(u[r]), 1.0))
            assert got[0][r] == define(x[r], params([s])[0], v)[0], (r, u[r])


@pytest.mark.gpu
def test_strides_offsets_and_outputs_left_out(gpu):
    rng = np.random.default_rng(6)
    x = (2 * rng.standard_normal((5, 1003))).astype(np.float32)
    u = rng.random(5).astype(np.float32)
    for ld, off in ((1003, 0), (1003, 1), (1005, 3), (4096, 2)):
        check(gpu, x, params([(0.8, 30, 0.9, 0.0)]), u, ld=ld, offset=off)
    check(gpu, x, params([(0.8, 30, 0.9, 0.0)]), u, extras=False)


@pytest.mark.gpu
@pytest.mark.parametrize("mean", [-1e30, -300.0, 0.0, 1e6, 1e30])
def test_logits_far_from_zero(gpu, mean):
    """Only the differences to the largest logit count: rows whose logits are
    large against the temperature, of both signs."""
    rng = np.random.default_rng(10)
    x = (mean + 2 * max(1.0, abs(mean) * 2.0 ** -22) * rng.standard_normal((len(SETTINGS), 9000))).astype(np.float32)
    check(gpu, x, params(SETTINGS), rng.random(len(SETTINGS)).astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 7, 8, 9, 40])
def test_top_k_about_the_number_of_blocks(gpu, k):
    """Rows of a few blocks of words whose best words lie together, apart, at
    the ends, or number fewer than k."""
    rng = np.random.default_rng(k)
    n = 8 * 2048 - 5
    x = rng.standard_normal((6, n)).astype(np.float32)
    x[0, :50] += 20
    x[1, ::2048] += 20
    x[2, -9:] += 20
    x[3, [0, n - 1]] = 30
    x[4, :] = -np.inf
    x[4, [5, 3000, 9000]] = [1.0, 1.0, 0.5]
    x[5, 2000:2100] = 8.0
    u = rng.random(6).astype(np.float32)
    check(gpu, x, params([(1.0, k, 1.0, 0.0)]), u)
    check(gpu, x, params([(0.7, k, 0.8, 0.05)]), u)
    check(gpu, x, params([(0.01, k, 0.999, 0.0)]), u)


@pytest.mark.gpu
def test_the_most_rows(gpu):
    rng = np.random.default_rng(11)
    x = (2 * rng.standard_normal((65535, 7))).astype(np.float32)
    par, u = params([(0.8, 5, 0.9, 0.02)]), rng.random(65535).astype(np.float32)
    tok, lp, left = run(gpu, x, par, u)
    for r in [0, 1, 65534, *rng.integers(0, 65535, 2000).tolist()]:
        want = define(x[r], par[0], u[r])
        assert (tok[r], left[r]) == (want[0], want[2]), r


@pytest.mark.gpu
def test_the_longest_rows(gpu):
    """2^19 - 1 words, all of one logit among them: sums just below 2^63, and
    a border list that is the whole row."""
    rng = np.random.default_rng(7)
    n = 2 ** 19 - 1
    x = np.stack([np.full(n, 2.0), rng.standard_normal(n), np.where(rng.random(n) < 0.5, 1.0, 1.25)]).astype(np.float32)
    for s in ((1.0, 0, 1.0, 0.0), (1.0, 0, 0.75, 0.0), (1.0, 300000, 0.9, 0.0)):
        check(gpu, x, params([s]), rng.random(3).astype(np.float32))


@pytest.mark.gpu
def test_the_same_call_gives_the_same_answer(gpu):
    """(No sum depends on the order in which it was formed.)"""
    rng = np.random.default_rng(8)
    x = (1.0 * rng.standard_normal((40, 50257))).astype(np.float32)
    u = rng.random(40).astype(np.float32)
    par = params([(1.5, 0, 0.98, 0.0)])
    first = run(gpu, x, par, u)
    for _ in range(3):
        again = run(gpu, x, par, u)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
def test_frequencies_follow_the_weights(gpu):
    """4096 evenly spaced random numbers meet each word as often as its share
    of the weight says, to one."""
    rng = np.random.default_rng(9)
    row = (1.5 * rng.standard_normal(50)).astype(np.float32)
    m = 4096
    x = np.tile(row, (m, 1))
    tok, _, _ = run(gpu, x, params([(0.8, 0, 1.0, 0.0)]), ((np.arange(m) + 0.5) / m).astype(np.float32))
    p = np.exp((row.astype(np.float64) - row.max()) / np.float64(np.float32(0.8)))
    p /= p.sum()
    assert np.all(np.abs(np.bincount(tok, minlength=50) - m * p) <= 1.0 + 1e-3)


# ------------------------------------------------------------- refusals ----
def test_workspace_of_refused_shapes_is_0():
    f = L.load().styx_op_sample_ws_bytes
    for rows, n in ((0, 10), (-1, 10), (65536, 10), (1, 0), (1, -5), (1, 2 ** 19)):
        assert f(rows, n) == 0
    assert f(1, 1) > 0 and f(65535, 100) > 0 and f(1, 2 ** 19 - 1) >= 2 * (2 ** 19 - 1)


def test_no_gpu_is_refused():
    assert L.load().styx_op_sample(None, None, 1, 1, 1, None, 1, None, None, None, None, None, 0) == -1


@pytest.mark.gpu
def test_refusals(gpu):
    p = gpu.zeros(1 << 16).ptr

    def call(ld=100, rows=2, n=100, n_params=1, logits=p, par=p, u=p, tok=p, ws=p, ws_bytes=None):
        if ws_bytes is None:
            ws_bytes = gpu.lib.styx_op_sample_ws_bytes(rows, n)
        return gpu.lib.styx_op_sample(gpu.h, logits, ld, rows, n, par, n_params, u, tok, None, None, ws, ws_bytes)

    for kw in (dict(ld=99), dict(rows=0), dict(rows=65536), dict(n=0), dict(n=2 ** 19, ld=2 ** 19), dict(n_params=0),
               dict(n_params=3), dict(logits=None), dict(par=None), dict(u=None), dict(tok=None), dict(ws=None),
               dict(ws=p + 4), dict(ws_bytes=16)):
        assert call(**kw) == -1, kw
        assert "styx_op_sample" in gpu.lib.styx_last_error().decode()
    gpu.sync()
