"""Instances of styx_op_attn_decode_batch's kernels that other tests leave
out: without weights, with nothing to do, and batches of more rows than the
Infinity Cache holds."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_kv_batch import Case, check_attn, run_attn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


@pytest.mark.parametrize("n_seq", [1, 3, 64, 65, 200])
@pytest.mark.parametrize("scored", [True, False])
def test_batches_of_skipped_sequences_alone(gpu, n_seq, scored):
    c = Case(np.random.default_rng(n_seq), False, [-1] * n_seq, 2, 4, 64, 16, table_len=3)
    check_attn(c, run_attn(gpu, c, scored=scored), scored=scored)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gqa", [1, 8, 9])
def test_attention_without_weights(gpu, f16, hd, gqa):
    rng = np.random.default_rng(hd + gqa)
    c = Case(rng, f16, [0, 5, 31, 64, 333, 1025], 2, gqa, hd, 48)
    check_attn(c, run_attn(gpu, c, scored=False), scored=False)



@pytest.mark.parametrize("scored", [True, False])
@pytest.mark.parametrize("f16,hd,gqa", [(False, 64, 1), (False, 128, 4), (False, 256, 1), (True, 64, 2), (True, 128, 9),
                                        (True, 256, 3)])
def test_batches_past_the_infinity_cache(gpu, f16, hd, gqa, scored):
    """More than 256 MB of rows, read past the caches."""
    nkv = 2 if gqa > 4 else 4
    rng = np.random.default_rng(hd)
    rows = 272 * 2 ** 20 // (2 * nkv * hd * (2 if f16 else 4))
    c = Case(rng, f16, [4, 5], nkv, gqa, hd, 100)
    lens = np.array([rows * 2 // 3, rows - rows * 2 // 3], np.int32)
    # the drawn rows again and again (a page more for the new rows)
    pages = (lens + 1 + 99) // 100
    c.lens, c.pos, c.table_len, c.cap = lens, np.array([3, 7], np.int32), int(pages.max()), int(pages.max()) * 100
    c.n_pages = int(pages.sum())
    base = rng.standard_normal(1 << 20).astype(c.dt)
    c.k = np.resize(base, (c.n_pages * 100, nkv, hd))
    c.v = np.resize(base[::-1], c.k.shape)
    perm = rng.permutation(c.n_pages).astype(np.int32)
    c.table = np.full((2, c.table_len), -1, np.int32)
    c.table[0, :pages[0]], c.table[1, :pages[1]] = perm[:pages[0]], perm[pages[0]:]
    c.acc = np.exp(rng.standard_normal((2, nkv, c.cap))).astype(np.float32)
    c.where = np.tile(np.arange(c.cap, dtype=np.int32), (2, nkv, 1))
    assert c.k.nbytes > 136 * 2 ** 20 and (c.rope.shape[0] > 7)
    check_attn(c, run_attn(gpu, c, scored=scored), scored=scored)
