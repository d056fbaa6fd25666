"""styx_op_kv_evict with each of its outputs its input or a buffer of its own,
in caches that one workgroup selects from and in longer ones."""
from __future__ import annotations

import ctypes as C
import itertools

import numpy as np
import pytest

from styx_amd import _lib as L
from test_gpu_kv_batch import evict_case, gpu, same, want_evict  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("acc_in_place,pos_in_place,len_in_place", itertools.product([False, True], repeat=3))
@pytest.mark.parametrize("keep,lens,table_len", [(60, [0, 64, 65, 300, 511, 40], 25), (9000, [17500, 9000, 100, 9001], 720)])
def test_outputs_in_place_one_by_one(gpu, keep, lens, table_len, acc_in_place, pos_in_place, len_in_place):  # noqa: F811
    rng = np.random.default_rng(keep)
    c = evict_case(rng, True, lens, 2, 64, 25, table_len=table_len)
    c.lens[-1] = -1
    kv = c.kv(gpu)
    ln, pos, acc, where = (gpu.from_numpy(x) for x in (c.lens, c.pos, c.acc, c.where))
    acc_out = acc if acc_in_place else gpu.from_numpy(np.full(c.acc.shape, -3.0, np.float32))
    where_out = where if pos_in_place else gpu.from_numpy(np.full(c.where.shape, -9, np.int32))
    len_out = ln if len_in_place else gpu.from_numpy(np.full(c.B, -77, np.int32))
    nbytes = gpu.lib.styx_op_kv_evict_ws_bytes(C.byref(kv), keep)
    ws = gpu.from_numpy(np.full(nbytes, 0xFF, np.uint8))
    L.check(gpu.lib.styx_op_kv_evict(gpu.h, C.byref(kv), ln.ptr, pos.ptr, keep, keep, 10, 4, acc.ptr, acc_out.ptr,
                                     where.ptr, where_out.ptr, len_out.ptr, ws.ptr, nbytes))
    gpu.sync()
    got = (acc_out.download(np.float32).reshape(c.acc.shape), where_out.download(np.int32).reshape(c.where.shape),
           len_out.download(np.int32, c.B), c.bufs[0].download(c.dt).reshape(c.k.shape),
           c.bufs[1].download(c.dt).reshape(c.v.shape))
    place, apart = (want_evict(c, keep, keep, 10, 4, p) for p in (True, False))
    same(got, (place[0] if acc_in_place else apart[0], place[1] if pos_in_place else apart[1], *apart[2:]))
