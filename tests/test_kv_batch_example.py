"""The step of a batch's loop that the integration guide shows, run on the CPU against
the operators' rules for lengths.  No GPU needed."""
from __future__ import annotations

import re
from pathlib import Path

import numpy as np

from styx_amd import _lib as L

ROOT = Path(__file__).resolve().parent.parent


class Lengths:
    """What KvBatch's calls do to the lengths: attend gives rows to the
    sequences that it does not skip, evict cuts those past the trigger."""

    def __init__(self, gpu, n_seq, nkv, hd, page_tokens, n_pages, table_len, type_):
        self.cap = page_tokens * table_len
        self.rows = None  # rows that there are, beside the lengths that the caller sets

    def set(self, len=None, pos=None, table=None):
        if len is not None:
            self.len = np.array(len)
        if pos is not None:
            self.pos = np.array(pos)

    def attend(self, nh, q, k, v, out, rope, n_rope, scale, q_norm, k_norm):
        assert self.rows is None
        took = (self.len >= 0) & (self.len < self.cap) & (self.pos >= 0) & (self.pos < n_rope)
        self.rows = np.where(took, self.len + 1, self.len)

    def evict(self, trigger, keep, recent, sinks):
        assert np.array_equal(self.len, self.rows), "the lengths are not those of the rows"
        self.len = np.where((self.len > trigger) & (self.len <= self.cap), keep, self.len)

    def lengths(self):
        return self.len.copy()


def test_the_example_advances_the_sequences_that_took_a_token(monkeypatch):
    blocks = re.findall(r"```python\n(.*?)```", (ROOT / "INTEGRATION.md").read_text(), re.S)
    code = [b for b in blocks if "KvBatch(" in b]
    assert len(code) == 1
    import styx_amd
    monkeypatch.setattr(styx_amd, "KvBatch", Lengths)
    monkeypatch.setattr(styx_amd, "sample", lambda *a: (None, None, None))
    # waiting, empty, ordinary, full, past the trigger, its position outside the rope table, past the capacity
    lens = np.array([-1, 0, 100, 4800, 4700, 7, 5000], np.int32)
    pos = np.array([0, 0, 300, 9000, 8999, 10000, 5], np.int32)
    ns = dict(L=L, np=np, gpu=None, n_seq=7, nkv=1, hd=64, page_tokens=16, n_pages=4, table_len=300, lens=lens.copy(),
              positions=pos.copy(), table=None, nh=1, q=None, k=None, v=None, out=None, rope=None, n_rope=10000,
              scale=1.0, q_norm=None, k_norm=None, logits=None, n_vocab=1, u=None)
    exec(code[0], ns)
    assert ns["lens"].tolist() == [-1, 1, 101, 4096, 4096, 7, 5000]
    assert ns["positions"].tolist() == [0, 1, 301, 9000, 9000, 10000, 5]
