"""The operators of a bounded-cache answer, measured: what a program that serves
answers from one paged KV cache runs for every new token.

Three kinds of case:

  attn    decode attention of one new token for each sequence of a batch over
          the paged cache, which also adds every row's attention weight to an
          accumulator (styx_op_attn_decode_batch)
  evict   the rows of least accumulated weight leave the cache
          (styx_op_kv_evict)
  sample  the next tokens from the logits by temperature, top-k, top-p and
          min-p and given random numbers (styx_op_sample)

Where `own` is true the framework's calls run, otherwise the same operators
in elementary torch operations.
"""
from __future__ import annotations

import ctypes as C
import math
import random

import torch

own = False

EPS = 1e-6
ROPE_BASE = 1e6
DEV = "cuda"
ONE = float(2 ** 44)  # the unit of sampling weights is 2^-44 of the largest
TYPES = {"f32": (torch.float32, 0, 4), "f16": (torch.float16, 1, 2)}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # the first answer token after a short question, one sequence: the
        # smallest call, where latency counts
        dict(name="attn_one_short", kind="attn", type="f32", n_seq=1, nkv=4, gqa=8, hd=128,
             page=512, longest=37, ragged=0, scored=True, norms=True),
        # one sequence at the longest context, 16 query heads per kv head
        dict(name="attn_one_32k", kind="attn", type="f32", n_seq=1, nkv=4, gqa=16, hd=128,
             page=512, longest=32767, ragged=0, scored=True, norms=True),
        # two dozen conversations of all lengths in a 16-bit cache of small pages
        dict(name="attn_chat_f16", kind="attn", type="f16", n_seq=24, nkv=4, gqa=8, hd=128,
             page=16, longest=4096, ragged=3, scored=True, norms=True),
        # a few long documents, wide heads, pages that are no power of two,
        # no eviction: plain batched attention
        dict(name="attn_docs_f32", kind="attn", type="f32", n_seq=6, nkv=2, gqa=8, hd=256,
             page=100, longest=20011, ragged=5, scored=False, norms=True),
        # many sequences, one query head per kv head, narrow heads
        dict(name="attn_mha_f16", kind="attn", type="f16", n_seq=40, nkv=8, gqa=1, hd=64,
             page=64, longest=8192, ragged=9, scored=True, norms=False),
        # a single conversation that has grown past its budget by a page
        dict(name="evict_one", kind="evict", type="f32", n_seq=1, nkv=4, hd=128, page=64,
             longest=1088, ragged=0, keep=1024, recent=128, sinks=4),
        # a batch, some of which have grown past the trigger
        dict(name="evict_chat_f16", kind="evict", type="f16", n_seq=32, nkv=4, hd=128, page=16,
             longest=9001, ragged=7, keep=4096, recent=512, sinks=4),
        # two very long documents cut to a quarter
        dict(name="evict_long", kind="evict", type="f32", n_seq=2, nkv=8, hd=128, page=512,
             longest=65536, ragged=0, keep=16384, recent=1024, sinks=16),
        # one answer with the whole chain of filters over a 151936-word vocabulary
        dict(name="sample_one", kind="sample", rows=1, n=151936, temperature=0.7, top_k=20,
             top_p=0.8, min_p=0.0, spread=2.5, ties=False, banned=False, mixed=False),
        # one answer, a small vocabulary, temperature alone: latency
        dict(name="sample_small", kind="sample", rows=1, n=4096, temperature=1.0, top_k=0,
             top_p=1.0, min_p=0.0, spread=2.0, ties=False, banned=False, mixed=False),
        # a batch in which every request brings its own settings
        dict(name="sample_batch", kind="sample", rows=64, n=151936, temperature=1.0, top_k=50,
             top_p=0.95, min_p=0.02, spread=2.0, ties=True, banned=False, mixed=True),
        # an odd vocabulary, flat logits (a hot temperature), banned words: a
        # nucleus of tens of thousands
        dict(name="sample_flat", kind="sample", rows=17, n=50257, temperature=1.8, top_k=0,
             top_p=0.98, min_p=0.0, spread=1.0, ties=False, banned=True, mixed=False),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "evict", "sample"])
    if kind == "sample":
        n = _logint(rng, 64, 152064)
        return dict(kind=kind, rows=_logint(rng, 1, max(1, min(256, 64 * 151936 // n))), n=n,
                    temperature=round(rng.uniform(0.2, 2.0), 3),
                    top_k=rng.choice([0, 0, 1, _logint(rng, 2, 1000)]),
                    top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)]),
                    min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]),
                    spread=round(rng.uniform(0.5, 4.0), 2), ties=rng.random() < 0.3,
                    banned=rng.random() < 0.3, mixed=rng.random() < 0.3)
    nkv, hd = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256])
    type_ = rng.choice(["f32", "f16"])
    n_seq = _logint(rng, 1, 64)
    # at most the listed 32K context's bytes
    most = 32767 * 4 * 128 * 4 // (n_seq * nkv * hd * TYPES[type_][2])
    longest = _logint(rng, 1, max(2, min(32767, most)))
    c = dict(kind=kind, type=type_, n_seq=n_seq, nkv=nkv, hd=hd,
             page=rng.choice([16, 32, 48, 64, 100, 128, 256, 512]), longest=longest,
             ragged=rng.choice([0, rng.randint(1, 1 << 20)]))
    if kind == "attn":
        return dict(c, gqa=rng.randint(1, 16), scored=rng.random() < 0.7, norms=rng.random() < 0.7)
    keep = max(1, int(longest * rng.uniform(0.2, 0.98)))
    return dict(c, keep=keep, recent=rng.randint(0, keep // 3), sinks=rng.randint(0, min(16, keep // 3)))


# ----------------------------------------------------------------- inputs --
def _lens(c):
    """Rows of each sequence before the new token: all the longest, or from
    one to the longest with that one among them."""
    if not c["ragged"]:
        return [c["longest"]] * c["n_seq"]
    r = random.Random(c["ragged"])
    lens = [r.randint(1, c["longest"]) for _ in range(c["n_seq"])]
    lens[r.randrange(c["n_seq"])] = c["longest"]
    return lens


def _cache(c, g, room):
    """A paged cache that holds the sequences with `room` rows more: pages in
    no order, table entries past a sequence's pages -1."""
    dtype, code, _ = TYPES[c["type"]]
    lens, page = _lens(c), c["page"]
    used = [-(-(n + room) // page) for n in lens]
    table_len, n_pages = max(used), sum(used)
    perm = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((c["n_seq"], table_len), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, m in enumerate(used):
        table[b, :m] = perm[at:at + m]
        at += m
    shape = (n_pages, page, c["nkv"], c["hd"])
    kpool = torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)
    vpool = torch.empty(shape, dtype=dtype, device=DEV).normal_(generator=g)
    cap = table_len * page
    return dict(type=code, n_seq=c["n_seq"], nkv=c["nkv"], hd=c["hd"], page=page, n_pages=n_pages,
                table_len=table_len, table=table, kpool=kpool, vpool=vpool, cap=cap,
                len=torch.tensor(lens, dtype=torch.int32, device=DEV))


def prepare(case, seed):
    g = torch.Generator(DEV)
    g.manual_seed(seed * 1000003 + 17)
    if case["kind"] == "sample":
        return _prepare_sample(case, g)
    attn = case["kind"] == "attn"
    s = _cache(case, g, 1 if attn else 0)
    shape = (s["n_seq"], s["nkv"], s["cap"])
    valid = torch.arange(s["cap"], device=DEV) < s["len"][:, None, None]
    # weights of a served cache: most rows little, a few very much
    s["acc_in"] = torch.exp(2.0 * torch.randn(shape, generator=g, device=DEV)) * 1e-2 * valid
    s["acc_out"] = torch.zeros(shape, device=DEV)
    # positions as after earlier evictions: gaps, and the first half in no order
    gaps = torch.randint(1, 3, shape, generator=g, device=DEV)
    where = torch.cumsum(gaps, 2) - gaps[:, :, :1]
    half = s["cap"] // 2
    mixed = torch.argsort(torch.rand((s["n_seq"], s["nkv"], half), generator=g, device=DEV), 2)
    where[:, :, :half] = where[:, :, :half].gather(2, mixed)
    s["slot_pos"] = where.to(torch.int32).contiguous()
    s["kind"] = case["kind"]
    if not attn:
        newest = torch.where(valid, where, -1).amax((1, 2))
        s.update(pos=newest.to(torch.int32), keep=case["keep"], recent=case["recent"], sinks=case["sinks"],
                 slot_pos_out=torch.zeros(shape, dtype=torch.int32, device=DEV),
                 len_out=torch.zeros(s["n_seq"], dtype=torch.int32, device=DEV))
        return s
    hd, nh = s["hd"], s["nkv"] * case["gqa"]
    n_rope = 2 * case["longest"] + 2
    inv = torch.pow(torch.tensor(ROPE_BASE, dtype=torch.float64, device=DEV),
                    -2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd)
    angle = torch.arange(n_rope, dtype=torch.float64, device=DEV)[:, None] * inv
    rnd = lambda *sh: torch.randn(sh, generator=g, device=DEV)  # noqa: E731
    s.update(nh=nh, n_rope=n_rope, rope=torch.stack([angle.cos(), angle.sin()], -1).contiguous(),
             pos=(2 * s["len"]).to(torch.int32), q=rnd(s["n_seq"], nh, hd), k=rnd(s["n_seq"], s["nkv"], hd),
             v=rnd(s["n_seq"], s["nkv"], hd), scale=1.0 / math.sqrt(hd), decay=0.99, scored=case["scored"],
             q_norm=1 + 0.1 * rnd(hd) if case["norms"] else None,
             k_norm=1 + 0.1 * rnd(hd) if case["norms"] else None,
             out=torch.zeros((s["n_seq"], nh, hd), device=DEV))
    return s


def _prepare_sample(c, g):
    rows, n = c["rows"], c["n"]
    x = c["spread"] * torch.randn((rows, n), generator=g, device=DEV)
    # the few words that the model is sure of
    sure = torch.randint(0, n, (rows, 8), generator=g, device=DEV)
    x.scatter_(1, sure, 4 * c["spread"] + c["spread"] * torch.randn((rows, 8), generator=g, device=DEV))
    if c["ties"]:  # logits that were 8-bit steps once
        x = torch.round(x * 16) / 16
    if c["banned"]:
        x.masked_fill_(torch.rand((rows, n), generator=g, device=DEV) < 0.2, -math.inf)
    settings = [c["temperature"], float(c["top_k"]), c["top_p"], c["min_p"]]
    p = torch.tensor([settings] * rows, device=DEV)
    if c["mixed"]:  # every row its own, greedy ones and unfiltered ones among them
        r = lambda: torch.rand(rows, generator=g, device=DEV)  # noqa: E731
        p[:, 0] = torch.where(r() < 0.15, 0.0, p[:, 0] * (0.5 + r()))
        p[:, 1] = torch.where(r() < 0.4, 0.0, torch.floor(1 + 2 * p[:, 1] * r()))
        p[:, 2] = torch.where(r() < 0.4, 1.0, p[:, 2] * (0.5 + 0.5 * r()))
        p[:, 3] = torch.where(r() < 0.4, 0.0, p[:, 3] * r())
    # {float temperature; int top_k; float top_p; float min_p} of every row
    params = p.view(torch.int32).clone()
    params[:, 1] = p[:, 1].to(torch.int32)
    return dict(kind="sample", rows=rows, n=n, logits=x.contiguous(), params=params.contiguous(),
                u=torch.rand(rows, generator=g, device=DEV),
                token=torch.zeros(rows, dtype=torch.int32, device=DEV), logprob=torch.zeros(rows, device=DEV),
                n_kept=torch.zeros(rows, dtype=torch.int32, device=DEV))


# -------------------------------------------------------------- own calls --
_held = {}


def _gpu():
    if "gpu" not in _held:
        from styx_amd import _lib
        from styx_amd.runtime import Gpu
        _held["gpu"], _held["L"] = Gpu(0), _lib
    return _held["gpu"], _held["L"]


def _workspace(s, nbytes):
    """The workspace that a program keeps beside its buffers."""
    if "ws" not in s:
        s["ws"] = torch.empty(max(16, nbytes()), dtype=torch.uint8, device=DEV)
    return s["ws"].data_ptr(), s["ws"].numel()


def _kv(s, L):
    if "kv" not in s:
        s["kv"] = L.KvCache(s["type"], s["n_seq"], s["nkv"], s["hd"], s["page"], s["n_pages"], s["table_len"],
                            s["kpool"].data_ptr(), s["vpool"].data_ptr(), s["table"].data_ptr())
    return C.byref(s["kv"])


def _ptr(t):
    return None if t is None else t.data_ptr()


def _own_attn(s):
    gpu, L = _gpu()
    kv = _kv(s, L)
    ws, ws_bytes = _workspace(s, lambda: gpu.lib.styx_op_attn_batch_ws_bytes(kv, s["nh"], int(s["scored"])))
    acc_in, acc_out, slot_pos = (s["acc_in"], s["acc_out"], s["slot_pos"]) if s["scored"] else (None, None, None)
    L.check(gpu.lib.styx_op_attn_decode_batch(
        gpu.h, kv, _ptr(s["len"]), _ptr(s["pos"]), s["nh"], _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]),
        _ptr(s["q_norm"]), _ptr(s["k_norm"]), EPS, _ptr(s["rope"]), s["n_rope"], s["scale"], s["decay"],
        _ptr(acc_in), _ptr(acc_out), _ptr(slot_pos), _ptr(s["out"]), ws, ws_bytes))
    return _attn_outputs(s, s["out"])


def _own_evict(s):
    gpu, L = _gpu()
    kv = _kv(s, L)
    ws, ws_bytes = _workspace(s, lambda: gpu.lib.styx_op_kv_evict_ws_bytes(kv, s["keep"]))
    L.check(gpu.lib.styx_op_kv_evict(
        gpu.h, kv, _ptr(s["len"]), _ptr(s["pos"]), s["keep"], s["keep"], s["recent"], s["sinks"],
        _ptr(s["acc_in"]), _ptr(s["acc_out"]), _ptr(s["slot_pos"]), _ptr(s["slot_pos_out"]), _ptr(s["len_out"]),
        ws, ws_bytes))
    return _evict_outputs(s)


def _own_sample(s):
    gpu, L = _gpu()
    ws, ws_bytes = _workspace(s, lambda: gpu.lib.styx_op_sample_ws_bytes(s["rows"], s["n"]))
    L.check(gpu.lib.styx_op_sample(
        gpu.h, _ptr(s["logits"]), s["n"], s["rows"], s["n"], _ptr(s["params"]), s["rows"], _ptr(s["u"]),
        _ptr(s["token"]), _ptr(s["logprob"]), _ptr(s["n_kept"]), ws, ws_bytes))
    return dict(token=s["token"], logprob=s["logprob"], n_kept=s["n_kept"])


# ------------------------------------------------------------ plain forms --
def _attn_outputs(s, out):
    """The output, and the state that the call updates."""
    got = dict(out=out, kpool=s["kpool"], vpool=s["vpool"])
    return dict(got, acc=s["acc_out"], slot_pos=s["slot_pos"]) if s["scored"] else got


def _evict_outputs(s):
    return dict(kpool=s["kpool"], vpool=s["vpool"], acc=s["acc_out"], slot_pos=s["slot_pos_out"], len=s["len_out"])


def _rows(s):
    """Row of the pools of every slot [n_seq][cap] (slots past a sequence's pages: row 0)."""
    slot = torch.arange(s["cap"], device=DEV)
    return s["table"].clamp(min=0).long()[:, slot // s["page"]] * s["page"] + slot % s["page"]


def _head(x, w, cs):
    """A head's RMSNorm and rotation, in 64 bits: the K row's rounding to the
    cache's type must not depend on the order of a sum."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    half = x.shape[-1] // 2
    a, b, c, sn = x[..., :half], x[..., half:], cs[..., 0], cs[..., 1]
    return torch.cat([a * c - b * sn, a * sn + b * c], -1)


def _plain_attn(s):
    n_seq, nkv, hd, nh = s["n_seq"], s["nkv"], s["hd"], s["nh"]
    cs = s["rope"][s["pos"].long()][:, None]
    q = _head(s["q"], s["q_norm"], cs).float()
    rows, slot, n = _rows(s), torch.arange(s["cap"], device=DEV), s["len"].long()
    kpool, vpool = s["kpool"].view(-1, nkv, hd), s["vpool"].view(-1, nkv, hd)
    at = rows.gather(1, n[:, None])[:, 0]
    kpool[at] = _head(s["k"], s["k_norm"], cs).to(kpool.dtype)
    vpool[at] = s["v"].to(vpool.dtype)
    k = kpool[rows].permute(0, 2, 3, 1).float()
    v = vpool[rows].permute(0, 2, 1, 3).float()
    score = torch.matmul(q.view(n_seq, nkv, nh // nkv, hd), k) * s["scale"]
    score = score.masked_fill((slot > n[:, None])[:, None, None], -math.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    out = torch.matmul(w, v).reshape(n_seq, nh, hd)
    if s["scored"]:
        old = torch.where((slot < n[:, None])[:, None], s["acc_in"], 0.0)
        seen = (slot <= n[:, None])[:, None].expand(-1, nkv, -1)
        s["acc_out"][seen] = (s["decay"] * old + w.sum(2))[seen]
        s["slot_pos"].scatter_(2, n[:, None, None].expand(-1, nkv, 1), s["pos"][:, None, None].expand(-1, nkv, 1))
    return _attn_outputs(s, out)


def _plain_evict(s):
    keep, nkv, hd = s["keep"], s["nkv"], s["hd"]
    slot, n, pos = torch.arange(s["cap"], device=DEV), s["len"][:, None, None], s["pos"][:, None, None]
    valid, act = slot < n, n > keep
    guarded = (s["slot_pos"] > pos - s["recent"]) | (s["slot_pos"] < s["sinks"])
    key = torch.where(guarded, math.inf, s["acc_in"].double())
    key = torch.where(valid, key, -math.inf)
    order = torch.sort(key, dim=2, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(2, order, slot.expand_as(order))
    kept = valid & ((rank < keep) | ~act)
    hole, mover = act & ~kept & (slot < keep), act & kept & (slot >= keep)
    movers = torch.sort((~mover).int(), dim=2, stable=True).indices
    nth = (torch.cumsum(hole.int(), 2) - 1).clamp(min=0)
    src = torch.where(hole, movers.gather(2, nth), slot)
    stays = slot < torch.where(act, keep, n)
    stays = stays.expand_as(kept)
    s["acc_out"][stays] = s["acc_in"].gather(2, src)[stays]
    s["slot_pos_out"][stays] = s["slot_pos"].gather(2, src)[stays]
    rows = _rows(s)
    b, j, to = hole.nonzero(as_tuple=True)
    for pool in (s["kpool"].view(-1, nkv, hd), s["vpool"].view(-1, nkv, hd)):
        pool[rows[b, to], j] = pool[rows[b, src[b, j, to]], j]
    s["len_out"].copy_(torch.where(act, keep, n)[:, 0, 0])
    return _evict_outputs(s)


def _plain_sample(s):
    """In 64 bits: which word a random number meets is decided by sums next to a border."""
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    p = s["params"].view(torch.float32).double()
    temperature, top_k = p[:, :1], s["params"][:, 1:2]
    top_p, min_p = p[:, 2:3], p[:, 3:4]
    rank = torch.arange(s["n"], device=DEV)
    v, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = ~(temperature > 0)
    top_k = torch.where(greedy, 1, top_k)
    d = torch.where(v == v[:, :1], 0.0, (v - v[:, :1]) / torch.where(greedy, 1.0, temperature))
    w = torch.round(torch.exp(d) * ONE).long()
    w = torch.where(v == -math.inf, 0, w)
    w = torch.where((top_k > 0) & (rank >= top_k), 0, w)
    run = torch.cumsum(w, 1)
    inside = (run - w).double() < top_p * run[:, -1:].double()
    w = torch.where((rank == 0) | ~(top_p < 1) | inside, w, 0)
    w = torch.where((rank == 0) | ~(min_p > 0) | (w.double() >= min_p * ONE), w, 0)
    n_kept = (w > 0).sum(1)
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    run = torch.cumsum(by_index, 1)
    total = run[:, -1:]
    t = torch.minimum((s["u"].double()[:, None] * total.double()).long().clamp(min=0), total - 1)
    token = (run <= t).sum(1)
    none = total[:, 0] == 0
    chosen = by_index.gather(1, token.clamp(max=s["n"] - 1)[:, None])[:, 0]
    logprob = torch.where(none, -math.inf, torch.log(chosen.double() / total[:, 0].double()))
    return dict(token=torch.where(none, -1, token).to(torch.int32), logprob=logprob.float(),
                n_kept=n_kept.to(torch.int32))


def run(state):
    if state["kind"] == "attn":
        return _own_attn(state) if own else _plain_attn(state)
    if state["kind"] == "evict":
        return _own_evict(state) if own else _plain_evict(state)
    return _own_sample(state) if own else _plain_sample(state)


# ------------------------------------------------------------------- work --
def work(case):
    """Cache rows, weights and logits read once, what changes written once."""
    if case["kind"] == "sample":
        m = case["rows"] * case["n"]
        return dict(bytes=4.0 * m + 32.0 * case["rows"], flops=20.0 * m)
    lens, nkv, hd, es = _lens(case), case["nkv"], case["hd"], TYPES[case["type"]][2]
    if case["kind"] == "attn":
        nh, rows = nkv * case["gqa"], sum(lens)
        nb = 2.0 * rows * nkv * hd * es + case["n_seq"] * (nkv * hd * (8 + 2 * es) + 8 * nh * hd)
        if case["scored"]:
            nb += 8.0 * nkv * (rows + case["n_seq"])
        return dict(bytes=nb, flops=4.0 * nh * hd * (rows + case["n_seq"]))
    keep, recent, sinks = case["keep"], case["recent"], case["sinks"]
    nb = flops = 0.0
    for n in lens:
        if n <= keep:  # stays as it is: weights and positions to the other buffer
            nb += 16.0 * nkv * n
            continue
        # of the rows past `keep`, the recent ones stay and the others like any row
        share = (keep - recent - sinks) / max(1, n - recent - sinks)
        moved = min(recent, n - keep) + share * max(0, n - keep - recent)
        nb += nkv * (8.0 * n + 8.0 * keep + 4.0 * moved * hd * es)
        flops += 4.0 * nkv * n
    return dict(bytes=nb + 12.0 * case["n_seq"], flops=flops)


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    s = prepare(case, seed)
    return dict(attn=_exact_attn, evict=_exact_evict, sample=_exact_sample)[case["kind"]](s)


def _exact_attn(s):
    """Sequence by sequence and head by head, all in 64 bits but the two roundings that the cache's type asks for."""
    hd, nkv, g = s["hd"], s["nkv"], s["nh"] // s["nkv"]
    half = hd // 2
    lens, table = s["len"].tolist(), s["table"].tolist()
    out = torch.zeros((s["n_seq"], s["nh"], hd), dtype=torch.float64, device=DEV)
    acc, where = s["acc_out"].double(), s["slot_pos"].clone()
    kpool, vpool = s["kpool"].clone(), s["vpool"].clone()

    def turned(x, w, p):
        x = x.double()
        if w is not None:
            x = x * torch.rsqrt((x * x).sum() / hd + EPS) * w.double()
        z = torch.complex(x[:half], x[half:]) * torch.complex(s["rope"][p, :, 0], s["rope"][p, :, 1])
        return torch.cat([z.real, z.imag])

    for b, n in enumerate(lens):
        p = int(s["pos"][b])
        pages = torch.tensor(table[b][:n // s["page"] + 1], device=DEV)
        page, off = table[b][n // s["page"]], n % s["page"]
        for j in range(nkv):
            kpool[page, off, j] = turned(s["k"][b, j], s["k_norm"], p).to(kpool.dtype)
            vpool[page, off, j] = s["v"][b, j].to(vpool.dtype)
            k = kpool[pages, :, j].reshape(-1, hd)[:n + 1].double()
            v = vpool[pages, :, j].reshape(-1, hd)[:n + 1].double()
            q = torch.stack([turned(s["q"][b, j * g + h], s["q_norm"], p) for h in range(g)])
            w = torch.softmax(q @ k.T * s["scale"], -1)
            out[b, j * g:(j + 1) * g] = w @ v
            acc[b, j, :n + 1] = w.sum(0)
            acc[b, j, :n] += s["decay"] * s["acc_in"][b, j, :n].double()
            where[b, j, n] = p
    got = dict(out=out, kpool=kpool, vpool=vpool)
    return dict(got, acc=acc, slot_pos=where) if s["scored"] else got


def _exact_evict(s):
    """Sequence by sequence and head by head, by the definition."""
    keep, page = s["keep"], s["page"]
    kpool, vpool = s["kpool"].clone(), s["vpool"].clone()
    acc, where, lens = s["acc_out"].double(), s["slot_pos_out"].clone(), s["len"].tolist()
    table = s["table"].long()
    for b, n in enumerate(lens):
        for j in range(s["nkv"]):
            a, w = s["acc_in"][b, j, :n].double(), s["slot_pos"][b, j, :n]
            src = torch.arange(min(n, keep), device=DEV)
            if n > keep:
                a = a.masked_fill((w > s["pos"][b] - s["recent"]) | (w < s["sinks"]), math.inf)
                best = torch.argsort(-a, stable=True)[:keep]
                stays = torch.zeros(n, dtype=torch.bool, device=DEV)
                stays[best] = True
                to, frm = (~stays[:keep]).nonzero()[:, 0], keep + stays[keep:].nonzero()[:, 0]
                src[to] = frm
                for pool in (kpool, vpool):
                    pool[table[b, to // page], to % page, j] = pool[table[b, frm // page], frm % page, j]
            acc[b, j, :len(src)] = s["acc_in"][b, j, src].double()
            where[b, j, :len(src)] = w[src]
    return dict(kpool=kpool, vpool=vpool, acc=acc, slot_pos=where,
                len=s["len"].clamp(max=keep))


def _exact_sample(s):
    """Row by row: the words that stay as a set, then the random number's place among them in the order of the words."""
    token, logprob, n_kept = [], [], []
    params_f, params_i = s["params"].view(torch.float32).double().tolist(), s["params"].tolist()
    for r in range(s["rows"]):
        temperature, _, top_p, min_p = params_f[r]
        top_k = params_i[r][1]
        x = s["logits"][r].double()
        ids = (x > -math.inf).nonzero()[:, 0]
        ids = ids[torch.argsort(-x[ids], stable=True)]
        if len(ids) == 0:
            token, logprob, n_kept = token + [-1], logprob + [-math.inf], n_kept + [0]
            continue
        if not temperature > 0:
            ids = ids[:1]
            temperature = 1.0
        if top_k > 0:
            ids = ids[:top_k]
        w = (torch.exp((x[ids] - x[ids[0]]) / temperature) * ONE).round().long()
        ids, w = ids[w > 0], w[w > 0]
        if top_p < 1:
            before = torch.cumsum(w, 0) - w
            m = max(1, int((before.double() < top_p * float(w.sum())).sum()))
            ids, w = ids[:m], w[:m]
        if min_p > 0:
            m = max(1, int((w.double() >= min_p * ONE).sum()))
            ids, w = ids[:m], w[:m]
        by = torch.argsort(ids)
        ids, w = ids[by], w[by]
        total = int(w.sum())
        t = min(int(float(s["u"][r]) * float(total)), total - 1)
        at = int(torch.searchsorted(torch.cumsum(w, 0), t, right=True))
        token.append(int(ids[at]))
        logprob.append(math.log(int(w[at]) / total))
        n_kept.append(len(ids))
    return dict(token=torch.tensor(token, dtype=torch.int32), logprob=torch.tensor(logprob, dtype=torch.float64),
                n_kept=torch.tensor(n_kept, dtype=torch.int32))
