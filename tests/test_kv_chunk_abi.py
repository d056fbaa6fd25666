"""The C layouts of the structs of the operators on new tokens (printed by a gcc
build of the header) against their ctypes and Rust mirrors, the rope tables
against their formulas, and the sizes of workspaces.  No GPU needed."""
from __future__ import annotations

import ctypes as C
import json
import math
import shutil
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from styx_amd import Chunk, KvBatch, _lib as L, rope_table
from test_abi_drift import HDR, rust_layout, rust_structs

ROOT = Path(__file__).resolve().parent.parent
STRUCTS = {"styx_kv_chunk": "KvChunk", "styx_kv_pages": "KvPages", "styx_rope": "Rope", "styx_rope_scaling": "RopeScaling"}


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_mirrors_have_the_header_layout(name, tmp_path):
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc not available")
    cls = getattr(L, STRUCTS[name])
    fields = [f for f, _ in cls._fields_]
    src = "\n".join(["#include <stdio.h>", "#include <stddef.h>", f'#include "{HDR}"', "int main(void) {",
                     f'printf("[%zu", sizeof({name}));',
                     *[f'printf(", %zu", offsetof({name}, {f}));' for f in fields], 'printf("]"); return 0; }'])
    (tmp_path / "lay.c").write_text(src)
    subprocess.run([gcc, "-std=c11", "-o", str(tmp_path / "lay"), str(tmp_path / "lay.c")], check=True)
    size, *offs = json.loads(subprocess.run([str(tmp_path / "lay")], capture_output=True, text=True, check=True).stdout)
    assert C.sizeof(cls) == size and [getattr(cls, f).offset for f in fields] == offs
    rust = rust_structs()[name]
    assert [f for f, _ in rust] == fields
    assert rust_layout(rust, {}) == (offs, size)



def near(got, freq, gain=1.0, n_pos=200):
    """(cos, sin)(p f) gain; an angle p f is off by at most 2^-50 of itself."""
    th = np.arange(n_pos)[:, None] * np.asarray(freq)
    want = gain * np.stack([np.cos(th), np.sin(th)], -1)
    assert np.abs(got - want).max() <= 1e-15 * 8 * n_pos * max(gain, 1)


def plain(n_rot, base):
    return np.array([base ** (-2 * i / n_rot) for i in range(n_rot // 2)])


@pytest.mark.parametrize("n_rot", [2, 64, 98, 128, 256])
def test_plain_table_is_styx_rope_table(n_rot):
    want = np.empty((200, n_rot // 2, 2))
    L.load().styx_rope_table(1e6, n_rot, 200, want.ctypes.data)
    assert np.array_equal(rope_table(n_rot, 200, 1e6), want)
    near(want, plain(n_rot, 1e6))


def test_linear_and_stretched_base():
    near(rope_table(64, 200, 1e4, L.ROPE_LINEAR, 4.0), plain(64, 1e4) / 4)
    near(rope_table(64, 200, 1e4, L.ROPE_LINEAR, 4.0, gain=1.5), plain(64, 1e4) / 4, 1.5)
    near(rope_table(64, 200, 1e4, L.ROPE_BASE, 8.0), plain(64, 1e4 * 8 ** (64 / 62)))


@pytest.mark.parametrize("fast,slow,n_orig", [(32, 1, 4096), (8, 2, 8192), (32, 1, 4)])
def test_by_parts(fast, slow, n_orig):
    n_rot, base, s = 128, 1e6, 8.0
    f = plain(n_rot, base)
    pair = lambda turns: n_rot * math.log(n_orig / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(0.0, math.floor(pair(fast))), min(n_rot - 1.0, math.ceil(pair(slow)))
    if high <= low:
        high = low + 0.001
    r = np.clip((np.arange(n_rot // 2) - low) / (high - low), 0, 1)
    want = f * (1 - r) + f / np.float32(s) * r
    gain = 0.1 * math.log(s) + 1
    near(rope_table(n_rot, 200, base, L.ROPE_PARTS, s, n_orig, fast, slow), want, gain)
    near(rope_table(n_rot, 200, base, L.ROPE_PARTS, s, n_orig, fast, slow, gain=1.0), want)
    if n_orig > 1000:  # fast pairs are kept, slow ones interpolated
        turns = n_orig * f / (2 * math.pi)
        assert np.array_equal(want[turns > 2 * fast], f[turns > 2 * fast])
        assert np.allclose(want[turns < slow / 2], f[turns < slow / 2] / s, rtol=1e-12)


def test_bands():
    f = plain(128, 5e5)
    turns = 8192 * f / (2 * math.pi)
    r = np.clip((turns - 1) / 3, 0, 1)
    want = f / 8 * (1 - r) + f * r
    near(rope_table(128, 200, 5e5, L.ROPE_BANDS, 8.0, 8192), want)
    assert (want[turns > 4] == f[turns > 4]).all() and np.allclose(want[turns < 1] * 8, f[turns < 1])


def test_rope_refusals():
    ok = dict(n_rot=64, n_pos=4, base=1e4)
    rope_table(**ok)
    for bad in [dict(n_rot=0), dict(n_rot=63), dict(n_rot=-2), dict(n_pos=0), dict(base=0.0), dict(base=-1.0), dict(base=math.nan),
                dict(base=math.inf), dict(kind=5), dict(kind=-1), dict(kind=L.ROPE_LINEAR, factor=0.0),
                dict(kind=L.ROPE_LINEAR, factor=math.inf), dict(kind=L.ROPE_BASE, factor=2.0, n_rot=2),
                dict(kind=L.ROPE_PARTS, factor=2.0), dict(kind=L.ROPE_PARTS, factor=2.0, n_orig=8, fast=1.0, slow=2.0),
                dict(kind=L.ROPE_PARTS, factor=2.0, n_orig=8, base=1.0), dict(kind=L.ROPE_BANDS, factor=2.0),
                dict(kind=L.ROPE_BANDS, factor=2.0, n_orig=8, slow=-1.0), dict(gain=math.nan)]:
        with pytest.raises(L.StyxError):
            rope_table(**{**ok, **bad})


def test_workspace_sizes():
    lib = L.load()
    kv = lambda **f: C.byref(L.KvCache(*{**dict(type=L.F16, n_seq=4, nkv=2, hd=128, page=16, n_pages=100, table_len=20, k=None,  # noqa: E731
                                                v=None, t=None), **f}.values()))
    assert lib.styx_op_attn_chunk_ws_bytes(kv(), 50, 8) > 0 and lib.styx_op_attn_chunk_ws_bytes(kv(), 0, 8) > 0
    for args in [(None, 50, 8), (kv(), -1, 8), (kv(), 50, 7), (kv(), 50, 0), (kv(), 50, 34), (kv(hd=80), 50, 8), (kv(type=8), 50, 8),
                 (kv(n_seq=0), 50, 8), (kv(page=1 << 20, table_len=1 << 20), 50, 8), (kv(), 2 ** 31 - 1, 32)]:
        assert lib.styx_op_attn_chunk_ws_bytes(*args) == 0, args[1:]


@pytest.mark.parametrize("nkv,gqa,n_seq", [(1, 1, 1), (1, 16, 1), (4, 8, 24), (2, 3, 1000), (8, 16, 200000)])
def test_the_largest_attention_is_as_large_as_the_header_says(nkv, gqa, n_seq):
    kv = C.byref(L.KvCache(L.F16, n_seq, nkv, 128, 16, 100, 20, None, None, None))
    most = (2 ** 28 - 128 * nkv * (n_seq + 1)) // (nkv * gqa)
    size = L.load().styx_op_attn_chunk_ws_bytes
    assert size(kv, most, nkv * gqa) > 0
    assert size(kv, most + 128 * (n_seq + 2), nkv * gqa) == 0


def test_entry_points_refuse_a_null_gpu():
    lib = L.load()
    assert lib.styx_op_kv_plan(*[None] * 8, 0, *[None] * 5) == -1
    assert lib.styx_op_kv_append(None, None, 0, None, None, 0, 0, None, 0, None, 0, None, 0, None, None, 0.0, None, 0, None, 0) == -1
    assert lib.styx_op_attn_chunk(None, None, None, 0, 0, None, 0, 0.0, 0, None, 0, None, None, 0) == -1
    assert lib.styx_op_kv_weigh(None, None, None, None, 0, 0, None, 0, 0.0, 0, None, 0, 0.0, None, None, None) == -1


def test_a_rope_table_needs_no_memory_of_its_own():
    """The call returns, and right, in a process that can allocate no more (an exception that leaves a C function ends
    the process)."""
    src = """
import resource, numpy as np
from styx_amd import _lib as L
lib = L.load()
n_rot = 1 << 23  # 2^22 pairs: 32 MiB of frequencies
out, ref = np.zeros((2, n_rot // 2, 2)), np.zeros((2, 32, 2))
s = L.RopeScaling(L.ROPE_LINEAR, 4.0, 0, 0.0, 0.0, 0.0)
call = lambda n, o: lib.styx_rope_table_scaled(1e4, n, 2, L.C.byref(s), o.ctypes.data)
assert call(64, ref) == 0
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
limit = resource.getrlimit(resource.RLIMIT_AS)
resource.setrlimit(resource.RLIMIT_AS, (used + (8 << 20), limit[1]))
rc = call(n_rot, out)
resource.setrlimit(resource.RLIMIT_AS, limit)
assert rc == 0
assert (out[0] == [1.0, 0.0]).all() and np.abs(out[1, 0] - [np.cos(0.25), np.sin(0.25)]).max() < 1e-15
f = 0.25 * 1e4 ** (-2.0 * (n_rot // 4) / n_rot)
assert np.abs(out[1, n_rot // 4] - [np.cos(f), np.sin(f)]).max() < 1e-9
print("done")
"""
    r = subprocess.run([sys.executable, "-c", src], capture_output=True, text=True, cwd=ROOT, timeout=100)
    assert r.returncode == 0 and "done" in r.stdout, (r.returncode, r.stderr[-500:])


class Held:
    """A buffer that is there, or was freed."""
    ptr, nbytes = 4096, 1 << 20

    def __init__(self):
        self.h = 1

    def free(self):
        self.h = None


def batch_and_chunk(n_seq, n_seq_chunk):
    """A KvBatch and a Chunk of a batch of other sequences, without a GPU; a call that gets as far as the library counts."""
    kv, other, reached = KvBatch.__new__(KvBatch), KvBatch.__new__(KvBatch), []

    class Gpu:
        h = None
        buffer = staticmethod(lambda nbytes: Held())

    class Lib:
        def __getattr__(self, name):
            return lambda *a: reached.append(name) or 0
    for x, n in ((kv, n_seq), (other, n_seq_chunk)):
        x.gpu, x.lib, x.n_seq, x.nkv, x.hd, x.scored, x._ws = Gpu(), Lib(), n, 1, 64, True, Held()
        x.c = L.KvCache(L.F32, n, 1, 64, 16, 4, 4, 4096, 4096, 4096)
        x.kpool, x.vpool, x.table, x.len, x.pos, x.acc, x.slot_pos = (Held() for _ in range(7))
        x.held = x.free_pages = x.n_free = None
    return kv, Chunk(other, 3), reached


CALLS = {"append": lambda kv, ch, b: kv.append(ch, 1, b, b, b, b, None),
         "attend_chunk": lambda kv, ch, b: kv.attend_chunk(ch, 1, b, b, 1.0),
         "weigh": lambda kv, ch, b: kv.weigh(ch, 1, b, b, 1.0, 1)}


@pytest.mark.parametrize("call", sorted(CALLS))
@pytest.mark.parametrize("n_seq,n_seq_chunk", [(4, 2), (2, 4)])
def test_a_chunk_of_other_sequences_is_refused(call, n_seq, n_seq_chunk):
    """Its arrays have as many entries as its own batch has sequences: a larger batch would read behind them."""
    kv, ch, reached = batch_and_chunk(n_seq, n_seq_chunk)
    with pytest.raises(ValueError, match="sequences"):
        CALLS[call](kv, ch, Held())
    assert not reached


@pytest.mark.parametrize("call", sorted(CALLS))
@pytest.mark.parametrize("freed", ["chunk", "batch"])
def test_a_freed_chunk_is_refused(call, freed):
    """And one whose lengths were freed with the batch that planned it."""
    kv, ch, reached = batch_and_chunk(4, 4)
    CALLS[call](kv, ch, Held())
    assert any("styx_op" in name for name in reached)
    reached.clear()
    if freed == "chunk":
        ch.free()
    else:
        ch.len.free()
    with pytest.raises(ValueError, match="freed"):
        CALLS[call](kv, ch, Held())
    assert not reached
