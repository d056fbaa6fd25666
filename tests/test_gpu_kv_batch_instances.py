"""Instances of styx_op_attn_decode_batch's kernels that other tests leave
out: without weights, and with nothing to do."""
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
