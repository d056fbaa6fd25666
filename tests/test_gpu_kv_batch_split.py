"""What styx_op_attn_decode_batch's choices cost: of a batch's split, and of how
its rows are read."""
from __future__ import annotations

import ctypes as C
import time

import numpy as np
import pytest

from styx_amd import _lib as L

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    from styx_amd import Gpu
    g = Gpu(0)
    yield g
    g.close()


def time_call(gpu, lens, nkv, hd, f16, n_seq, spare=0):
    """Microseconds of a call among others, the best of six runs: the
    sequences of `lens` and, up to n_seq, ones that are skipped; pages that no
    sequence has behind each of theirs."""
    page, es = 512, 2 if f16 else 4
    used = [-(-(n + 1) // page) for n in lens]
    n_pages, table_len = sum(used) * (1 + spare), max(used)
    table = np.full((n_seq, table_len), -1, np.int32)
    at = 0
    for b, m in enumerate(used):
        table[b, :m] = np.arange(at, at + m) * (1 + spare)
        at += m
    ln = np.full(n_seq, -1, np.int32)
    ln[:len(lens)] = lens
    pool = np.resize(np.random.default_rng(1).standard_normal(1 << 20).astype(np.float16 if f16 else np.float32),
                     n_pages * page * nkv * hd)
    z = lambda n: gpu.zeros(4 * n)  # noqa: E731
    held = [gpu.from_numpy(x) for x in (pool, pool, table, ln, np.zeros(n_seq, np.int32))]
    q, k, v, out, rope = z(n_seq * nkv * hd), z(n_seq * nkv * hd), z(n_seq * nkv * hd), z(n_seq * nkv * hd), z(2 * hd)
    kv = L.KvCache(L.F16 if f16 else L.F32, n_seq, nkv, hd, page, n_pages, table_len, *(b.ptr for b in held[:3]))
    nbytes = gpu.lib.styx_op_attn_batch_ws_bytes(C.byref(kv), nkv, 0)
    ws = gpu.buffer(nbytes)
    best = np.inf
    for _ in range(6):
        gpu.sync()
        t = time.perf_counter()
        for _ in range(20):
            L.check(gpu.lib.styx_op_attn_decode_batch(
                gpu.h, C.byref(kv), held[3].ptr, held[4].ptr, nkv, q.ptr, k.ptr, v.ptr, None, None, 1e-6, rope.ptr, 1,
                0.1, 1.0, None, None, None, out.ptr, ws.ptr, nbytes))
        gpu.sync()
        best = min(best, (time.perf_counter() - t) / 20 * 1e6)
    for b in (*held, q, k, v, out, rope, ws):
        b.free()
    return best


def best_of_three(f, *args):
    """The arguments' times, measured in turn."""
    runs = [[f(a) for a in args] for _ in range(3)]
    return [min(t) for t in zip(*runs)]


@pytest.mark.parametrize("longs,n_long,short,n_seq,nkv,hd,f16", [(65536, 1, 1, 59, 13, 64, True),
                                                                (131072, 1, 128, 62, 8, 128, True),
                                                                (32768, 1, 128, 31, 8, 256, False)])
def test_a_split_that_is_not_taken_is_not_searched_for(gpu, longs, n_long, short, n_seq, nkv, hd, f16):
    """A long sequence among many short ones, nearly as many heads as
    workgroups run at once: no share keeps every head to whole shares, and the
    call takes as long as with skipped sequences up to 65 beside them (past 64
    no share is looked for at all, and the split is the same)."""
    lens = [longs - 1] * n_long + [short - 1] * (n_seq - n_long)
    alone, beside = best_of_three(lambda n: time_call(gpu, lens, nkv, hd, f16, n), n_seq, 65)
    print(f"{alone:.1f} us, {beside:.1f} us with skipped sequences")
    assert alone <= 1.3 * beside + 10.0


@pytest.mark.parametrize("times", [5, 8])
def test_rows_that_the_caches_hold_are_read_from_them_in_a_pool_of_any_size(gpu, times):
    """Calls in turn on the same rows, which the Infinity Cache holds: as fast
    in a pool several times its size as in one of their own."""
    lens = [4096, 700, 2000, 3500] * times
    own, large = best_of_three(lambda spare: time_call(gpu, lens, 4, 128, True, len(lens), spare), 0, 4)
    print(f"{own:.1f} us, {large:.1f} us in a large pool")
    assert large <= 1.08 * own
