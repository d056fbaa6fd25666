"""The operators that bring new tokens into a batch's paged KV cache, measured:
what a program that serves prompts, parts of prompts and single tokens together
runs for every step.

Four kinds of case:

  plan    page tables from a stack of free pages, and the map from the step's
          rows to sequences, positions and rows of the cache (styx_op_kv_plan)
  append  per-head RMSNorm and rotary positions, K and V into their pages, q
          turned (styx_op_kv_append)
  attn    causal attention of each sequence's new tokens over its cached rows
          and themselves (styx_op_attn_chunk)
  weigh   the attention weights of the last tokens added to every row's
          accumulator, by which rows are evicted later (styx_op_kv_weigh)

Where `own` is true the framework's calls run, otherwise the same operators
in elementary torch operations.
"""
from __future__ import annotations

import ctypes as C
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
DEV = "cuda"
TYPES = {"f32": (torch.float32, 0, 4), "f16": (torch.float16, 1, 2)}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # a short question after a short answer, one conversation: the smallest call, where latency counts
        dict(name="attn_turn", kind="attn", type="f32", qtype="f32", n_seq=1, nkv=4, gqa=8, hd=128, page=512,
             ctx=32, new=5, ragged=0, singles=False, window=0, lse=False),
        # one long prompt from the first token on, all 16 bits
        dict(name="attn_prompt_f16", kind="attn", type="f16", qtype="f16", n_seq=1, nkv=4, gqa=8, hd=128, page=64,
             ctx=0, new=8192, ragged=0, singles=False, window=0, lse=True),
        # a step of a busy server: most sequences one token, a few a part of their prompt, contexts of all lengths
        dict(name="attn_mixed_f16", kind="attn", type="f16", qtype="f32", n_seq=24, nkv=4, gqa=8, hd=128, page=16,
             ctx=16384, new=512, ragged=3, singles=True, window=0, lse=True),
        # parts of three documents, wide heads, pages that are no power of two
        dict(name="attn_docs_f32", kind="attn", type="f32", qtype="f32", n_seq=3, nkv=2, gqa=8, hd=256, page=100,
             ctx=6007, new=1021, ragged=5, singles=False, window=0, lse=False),
        # prompts under a sliding window, one query head per kv head, narrow heads
        dict(name="attn_window_f16", kind="attn", type="f16", qtype="f16", n_seq=8, nkv=8, gqa=1, hd=64, page=64,
             ctx=4096, new=2001, ragged=9, singles=False, window=1024, lse=False),
        # the last part of a long prompt: its last 64 tokens say what may leave the cache
        dict(name="weigh_prompt_f16", kind="weigh", type="f16", qtype="f16", n_seq=1, nkv=4, gqa=8, hd=128, page=64,
             ctx=32000, new=768, ragged=0, singles=False, window=0, last=64),
        # a batch of conversations with short questions, 16 query heads per kv head
        dict(name="weigh_batch_f32", kind="weigh", type="f32", qtype="f32", n_seq=16, nkv=4, gqa=16, hd=128, page=128,
             ctx=2048, new=250, ragged=7, singles=False, window=0, last=16),
        # one token for each of four dozen sequences
        dict(name="append_tokens", kind="append", type="f16", tin="f32", qtype="f32", n_seq=48, nkv=4, gqa=8, hd=128,
             page=16, ctx=4096, new=1, ragged=11, singles=False, n_rot=128, interleaved=False, norms=True, factor=1.0),
        # a long prompt in 16 bits, neighbouring pairs of half of each head turned, positions stretched fourfold
        dict(name="append_prompt_f16", kind="append", type="f16", tin="f16", qtype="f16", n_seq=1, nkv=4, gqa=8, hd=128,
             page=64, ctx=24576, new=8192, ragged=0, singles=False, n_rot=64, interleaved=True, norms=False, factor=4.0),
        # parts of four documents, wide heads
        dict(name="append_docs_f32", kind="append", type="f32", tin="f32", qtype="f32", n_seq=4, nkv=2, gqa=8, hd=256,
             page=100, ctx=3000, new=1021, ragged=13, singles=False, n_rot=256, interleaved=False, norms=True, factor=1.0),
        # one token for each of 64 sequences, small pages, one sequence in nine has ended
        dict(name="plan_step", kind="plan", n_seq=64, page=16, ctx=8192, new=1, ragged=17, ended=0.11, cut=0.0,
             short=False),
        # a step of prompts after an eviction: pages come back and go out again
        dict(name="plan_prompts", kind="plan", n_seq=256, page=16, ctx=8192, new=2048, ragged=19, ended=0.1, cut=0.2,
             short=False),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "weigh", "append", "plan"])
    page = rng.choice([16, 32, 48, 64, 100, 128, 256, 512])
    if kind == "plan":
        n_seq = _logint(rng, 1, 512)
        new = rng.choice([1, _logint(rng, 1, min(4096, max(1, 256 * 2048 // n_seq)))])
        return dict(kind=kind, n_seq=n_seq, page=page, ctx=_logint(rng, 1, 8192), new=new,
                    ragged=rng.randint(1, 1 << 20), ended=rng.choice([0.0, 0.2]), cut=rng.choice([0.0, 0.3]),
                    short=rng.random() < 0.25)
    type_ = rng.choice(["f32", "f16"])
    qtype = type_ if type_ == "f32" else rng.choice(["f32", "f16", "f16"])
    nkv, hd, gqa = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256]), rng.randint(1, 16)
    n_seq = _logint(rng, 1, 48)
    ctx = rng.choice([0, _logint(rng, 1, 32767)])
    new = rng.choice([1, _logint(rng, 1, 4096), _logint(rng, 1, 4096)])
    c = dict(kind=kind, type=type_, qtype=qtype, nkv=nkv, gqa=gqa, hd=hd, page=page,
             ragged=rng.choice([0, rng.randint(1, 1 << 20)]), singles=rng.random() < 0.3)
    if kind == "append":
        # at most the bytes of the listed prompt: 8192 rows of 40 heads of 128 in 16 bits, read and written
        most = max(1, 8192 * 40 * 128 * 2 // ((gqa + 2) * nkv * hd * TYPES[type_][2] * n_seq))
        c.update(tin=type_ if type_ == "f32" else rng.choice(["f32", "f16"]), ctx=min(ctx, 24576), new=min(new, most),
                 n_rot=rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]), interleaved=rng.random() < 0.5,
                 norms=rng.random() < 0.5, factor=rng.choice([1.0, 1.0, 2.0, 4.0, 8.0]))
        return dict(c, n_seq=n_seq)
    # at most the cache bytes of the listed mixed step, the products of the listed prompt in the type's price
    ctx = min(ctx, 16384 * 24 * 4 * 128 * 2 // (n_seq * nkv * hd * TYPES[type_][2]))
    c["last"] = last = rng.choice([1, 16, 64, _logint(rng, 1, 256)])
    price = hd * gqa * nkv * (8 if type_ == "f32" else 2 if qtype == "f32" else 1)
    while n_seq * (min(new, last) if kind == "weigh" else new) * (ctx + new) * price > 4096 * 8192 * 128 * 32:
        if new > 1:
            new = max(1, new // 2)
        else:
            n_seq, ctx = max(1, n_seq // 2), ctx // 2
    c.update(n_seq=n_seq, ctx=ctx, new=new, window=rng.choice([0, 0, _logint(rng, 1, 4096)]))
    if kind == "attn":
        c.pop("last")
        c["lse"] = rng.random() < 0.5
    return c


# ----------------------------------------------------------------- inputs --
def _shape(c):
    """Rows that each sequence has, and its new ones."""
    if not c["ragged"]:
        return [c["ctx"]] * c["n_seq"], [c["new"]] * c["n_seq"]
    r = random.Random(c["ragged"])
    lens = [r.randint(0, c["ctx"]) for _ in range(c["n_seq"])]
    new = [r.randint(1, c["new"]) for _ in range(c["n_seq"])]
    lens[r.randrange(c["n_seq"])] = c["ctx"]
    if c.get("singles"):  # one token for most
        new = [n if r.random() < 0.2 else 1 for n in new]
    new[r.randrange(c["n_seq"])] = c["new"]
    return lens, new


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cache(c, g):
    """A paged cache that holds the sequences and their new rows: pages in no
    order, table entries past a sequence's pages -1."""
    dtype, code, _ = TYPES[c["type"]]
    lens, new = _shape(c)
    page = c["page"]
    used = [-(-(n + m) // page) for n, m in zip(lens, new)]
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
    first = [sum(new[:b]) for b in range(c["n_seq"])]
    return dict(kind=c["kind"], type=code, n_seq=c["n_seq"], nkv=c["nkv"], hd=c["hd"], nh=c["nkv"] * c["gqa"],
                page=page, n_pages=n_pages, table_len=table_len, cap=table_len * page, table=table, kpool=kpool,
                vpool=vpool, n_rows=sum(new), lens=lens, new=new, firsts=first, len=_i32(lens), count=_i32(new),
                first=_i32(first), qcode=TYPES[c["qtype"]][1], qdtype=TYPES[c["qtype"]][0])


def prepare(case, seed):
    g = torch.Generator(DEV)
    g.manual_seed(seed * 1000003 + 29)
    if case["kind"] == "plan":
        return _prepare_plan(case, g)
    s = _cache(case, g)
    if case["kind"] == "append":
        return _prepare_append(case, s, g)
    # heads as they leave the norm, some directions of them strong: a softmax with a few large weights
    q = 2.0 * torch.randn((s["n_rows"], s["nh"], s["hd"]), generator=g, device=DEV)
    s.update(q=q.to(s["qdtype"]), scale=1.0 / math.sqrt(s["hd"]), window=case["window"])
    if case["kind"] == "attn":
        s.update(out=torch.zeros_like(s["q"]),
                 lse=torch.zeros((s["n_rows"], s["nh"]), device=DEV) if case["lse"] else None)
        return s
    shape = (s["n_seq"], s["nkv"], s["cap"])
    s.update(last=case["last"], decay=0.99, lse=torch.zeros((s["n_rows"], s["nh"]), device=DEV),
             acc_in=torch.exp(2.0 * torch.randn(shape, generator=g, device=DEV)) * 1e-2,
             acc_out=torch.zeros(shape, device=DEV), slot_pos=torch.zeros(shape, dtype=torch.int32, device=DEV),
             pos=_i32([2 * n for n in s["lens"]]))
    # what attention left of the rows that count
    for b, i0, i1 in _last_parts(s):
        for j in range(s["nkv"]):
            x = _scores(s, b, j, i0, i1, _slots(s, b))
            s["lse"][s["firsts"][b] + i0:s["firsts"][b] + i1, j * case["gqa"]:(j + 1) * case["gqa"]] = \
                torch.logsumexp(x.double(), -1).float().T
    return s


def _prepare_append(c, s, g):
    n_rot, lens, new = c["n_rot"], s["lens"], s["new"]
    pos0 = [n + n // 8 for n in lens]  # rows have left the cache before
    n_pos = max(p + n for p, n in zip(pos0, new))
    base, factor, trained = 1e6, c["factor"], 8192.0
    i = torch.arange(n_rot // 2, dtype=torch.float64, device=DEV)
    freq = torch.pow(torch.tensor(base, dtype=torch.float64, device=DEV), -2.0 * i / n_rot)
    gain = 1.0
    if factor > 1:  # slow pairs interpolated, fast ones as they are, a ramp between 32 turns and 1
        turns = freq * trained / (2 * math.pi)
        keep = ((turns.log() - math.log(1.0)) / math.log(32.0)).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / factor)
        gain = 0.1 * math.log(factor) + 1
    angle = torch.arange(n_pos, dtype=torch.float64, device=DEV)[:, None] * freq
    rope = gain * torch.stack([angle.cos(), angle.sin()], -1)
    width = (s["nh"] + 2 * s["nkv"]) * s["hd"]
    dtype, tin, _ = TYPES[c["tin"]]
    qkv = torch.randn((s["n_rows"], width), generator=g, device=DEV).to(dtype)
    at, pos = [], []
    table = s["table"].tolist()
    for b, (n, m) in enumerate(zip(lens, new)):
        at += [table[b][t // s["page"]] * s["page"] + t % s["page"] for t in range(n, n + m)]
        pos += range(pos0[b], pos0[b] + m)
    s.update(tin=tin, qkv=qkv, ld=width, rope=rope.contiguous(), n_pos=n_pos, n_rot=n_rot,
             interleaved=c["interleaved"], row_at=_i32(at), row_pos=_i32(pos),
             q_norm=1 + 0.1 * torch.randn(s["hd"], generator=g, device=DEV) if c["norms"] else None,
             k_norm=1 + 0.1 * torch.randn(s["hd"], generator=g, device=DEV) if c["norms"] else None,
             q_out=torch.zeros((s["n_rows"], s["nh"], s["hd"]), dtype=s["qdtype"], device=DEV))
    return s


def _prepare_plan(c, g):
    page, n_seq = c["page"], c["n_seq"]
    lens, new = _shape(c)
    r = random.Random(c["ragged"] + 1)
    seed = int(torch.randint(0, 1 << 30, (1,), generator=g, device=DEV))
    held = [-(-n // page) for n in lens]
    shared = [0] * n_seq
    for b in range(n_seq):
        if r.random() < c["cut"]:  # rows have left since: fewer rows than pages
            lens[b] = int(lens[b] * r.random())
        if r.random() < c["ended"]:
            lens[b], new[b] = -1, 0
        if r.random() < 0.2:  # begins with pages of another's
            shared[b] = r.randint(0, held[b])
    table_len = max(max(held), -(-(c["ctx"] + c["new"]) // page))
    asked = sum(max(0, -(-(max(n, 0) + m) // page) - h) for n, m, h in zip(lens, new, held))
    n_free = asked // 2 if c["short"] else asked + n_seq
    n_pages = sum(held) + n_free + 3
    perm = np.random.default_rng(seed).permutation(n_pages).astype(np.int32)
    table = np.full((n_seq, table_len), -1, np.int32)
    at = 0
    for b, m in enumerate(held):
        table[b, :m] = perm[at:at + m]
        at += m
    free = np.full(n_pages, -1, np.int32)
    free[:n_free] = perm[at:at + n_free]
    n_rows = sum(new)
    fresh = lambda *sh: torch.full(sh, -1, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(kind="plan", n_seq=n_seq, page=page, n_pages=n_pages, table_len=table_len, n_rows=max(1, n_rows),
                table=torch.from_numpy(table).to(DEV), held=_i32(held), free=torch.from_numpy(free).to(DEV),
                n_free=_i32([n_free]), shared=_i32(shared), len=_i32(lens), n_new=_i32(new),
                pos=_i32([max(0, n) + 7 for n in lens]), table_out=fresh(n_seq, table_len), held_out=fresh(n_seq),
                free_out=fresh(n_pages), n_free_out=fresh(1), first=fresh(n_seq), count=fresh(n_seq),
                row_seq=fresh(max(1, n_rows)), row_pos=fresh(max(1, n_rows)), row_at=fresh(max(1, n_rows)))


# -------------------------------------------------------------- own calls --
_held = {}


def _gpu():
    if "gpu" not in _held:
        from styx_amd import _lib
        from styx_amd.runtime import Gpu
        _held["gpu"], _held["L"] = Gpu(0), _lib
    return _held["gpu"], _held["L"]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _kv(s, L):
    """The cache and the chunk as the program keeps them."""
    if "kv" not in s:
        s["kv"] = L.KvCache(s["type"], s["n_seq"], s["nkv"], s["hd"], s["page"], s["n_pages"], s["table_len"],
                            s["kpool"].data_ptr(), s["vpool"].data_ptr(), s["table"].data_ptr())
        s["chunk"] = L.KvChunk(s["n_rows"], s["first"].data_ptr(), s["count"].data_ptr(), s["len"].data_ptr())
    return C.byref(s["kv"]), C.byref(s["chunk"])


def _own_attn(s):
    gpu, L = _gpu()
    kv, chunk = _kv(s, L)
    if "ws" not in s:  # the workspace that a program keeps beside its buffers
        nbytes = gpu.lib.styx_op_attn_chunk_ws_bytes(kv, s["n_rows"], s["nh"])
        s["ws"] = torch.empty(max(16, nbytes), dtype=torch.uint8, device=DEV)
    row = s["nh"] * s["hd"]
    L.check(gpu.lib.styx_op_attn_chunk(gpu.h, kv, chunk, s["nh"], s["qcode"], _ptr(s["q"]), row, s["scale"],
                                       s["window"], _ptr(s["out"]), row, _ptr(s["lse"]), _ptr(s["ws"]),
                                       s["ws"].numel()))
    return _attn_outputs(s, s["out"], s["lse"])


def _own_weigh(s):
    gpu, L = _gpu()
    kv, chunk = _kv(s, L)
    L.check(gpu.lib.styx_op_kv_weigh(gpu.h, kv, chunk, _ptr(s["pos"]), s["nh"], s["qcode"], _ptr(s["q"]),
                                     s["nh"] * s["hd"], s["scale"], s["window"], _ptr(s["lse"]), s["last"], s["decay"],
                                     _ptr(s["acc_in"]), _ptr(s["acc_out"]), _ptr(s["slot_pos"])))
    return dict(acc=s["acc_out"], slot_pos=s["slot_pos"])


def _own_append(s):
    gpu, L = _gpu()
    if "kv" not in s:
        s["kv"] = L.KvCache(s["type"], s["n_seq"], s["nkv"], s["hd"], s["page"], s["n_pages"], s["table_len"],
                            s["kpool"].data_ptr(), s["vpool"].data_ptr(), s["table"].data_ptr())
        s["rope_c"] = L.Rope(s["rope"].data_ptr(), s["n_pos"], s["n_rot"], int(s["interleaved"]))
    q, es = s["qkv"].data_ptr(), s["qkv"].element_size()
    k = q + s["nh"] * s["hd"] * es
    v = k + s["nkv"] * s["hd"] * es
    L.check(gpu.lib.styx_op_kv_append(gpu.h, C.byref(s["kv"]), s["n_rows"], _ptr(s["row_pos"]), _ptr(s["row_at"]),
                                      s["nh"], s["tin"], q, s["ld"], k, s["ld"], v, s["ld"], _ptr(s["q_norm"]),
                                      _ptr(s["k_norm"]), EPS, C.byref(s["rope_c"]), s["qcode"], _ptr(s["q_out"]),
                                      s["nh"] * s["hd"]))
    return dict(q=s["q_out"], kpool=s["kpool"], vpool=s["vpool"])


def _own_plan(s):
    gpu, L = _gpu()
    if "kv" not in s:
        s["pages"] = [L.KvPages(s["table" + x].data_ptr(), s["held" + x].data_ptr(), s["free" + x].data_ptr(),
                                s["n_free" + x].data_ptr()) for x in ("", "_out")]
        s["kv"] = L.KvCache(0, s["n_seq"], 1, 64, s["page"], s["n_pages"], s["table_len"], None, None, None)
    L.check(gpu.lib.styx_op_kv_plan(gpu.h, C.byref(s["kv"]), C.byref(s["pages"][0]), C.byref(s["pages"][1]),
                                    _ptr(s["shared"]), _ptr(s["len"]), _ptr(s["n_new"]), _ptr(s["pos"]), s["n_rows"],
                                    _ptr(s["first"]), _ptr(s["count"]), _ptr(s["row_seq"]), _ptr(s["row_pos"]),
                                    _ptr(s["row_at"])))
    return _plan_outputs(s)


# ------------------------------------------------------------ plain forms --
def _attn_outputs(s, out, lse):
    return dict(out=out) if s["lse"] is None else dict(out=out, lse=lse)


def _plan_outputs(s):
    return {n: s[n] for n in ("table_out", "held_out", "free_out", "n_free_out", "first", "count", "row_seq",
                              "row_pos", "row_at")}


def _slots(s, b):
    """Rows of the pools of sequence b's slots, its new ones among them."""
    slot = torch.arange(s["lens"][b] + s["new"][b], device=DEV)
    return s["table"][b].long()[slot // s["page"]] * s["page"] + slot % s["page"]


def _scores(s, b, j, i0, i1, rows):
    """[gqa][i1 - i0][slots] scaled scores of new tokens [i0, i1), -infinity where a token does not see a slot."""
    g, hd, n = s["nh"] // s["nkv"], s["hd"], s["lens"][b]
    r0 = s["firsts"][b]
    q = s["q"][r0 + i0:r0 + i1, j * g:(j + 1) * g].float().transpose(0, 1).reshape(g * (i1 - i0), hd)
    k = s["kpool"].view(-1, s["nkv"], hd)[rows, j].float()
    x = (torch.matmul(q, k.T) * s["scale"]).view(g, i1 - i0, len(rows))
    at = n + torch.arange(i0, i1, device=DEV)[:, None]
    slot = torch.arange(len(rows), device=DEV)
    unseen = slot > at
    if s["window"]:
        unseen = unseen | (slot <= at - s["window"])
    return x.masked_fill(unseen, -math.inf)


def _plain_attn(s):
    g, hd, out = s["nh"] // s["nkv"], s["hd"], torch.empty_like(s["out"])
    lse = None if s["lse"] is None else torch.empty_like(s["lse"])
    for b, n in enumerate(s["new"]):
        rows, r0 = _slots(s, b), s["firsts"][b]
        for j in range(s["nkv"]):
            v = s["vpool"].view(-1, s["nkv"], hd)[rows, j].float()
            for i0 in range(0, n, 1024):
                i1 = min(n, i0 + 1024)
                seen = s["lens"][b] + i1  # slots past it are seen by none of these
                x = _scores(s, b, j, i0, i1, rows[:seen])
                m = x.amax(-1, keepdim=True)
                w = torch.exp(x - m)
                total = w.sum(-1, keepdim=True)
                o = torch.matmul(w.view(-1, seen), v[:seen]).view(g, i1 - i0, hd) / total
                out[r0 + i0:r0 + i1, j * g:(j + 1) * g] = o.transpose(0, 1).to(out.dtype)
                if lse is not None:
                    lse[r0 + i0:r0 + i1, j * g:(j + 1) * g] = (m + torch.log(total))[..., 0].T
    return _attn_outputs(s, out, lse)


def _last_parts(s):
    """(sequence, first, last) of the tokens that count."""
    return [(b, max(0, n - s["last"]), n) for b, n in enumerate(s["new"])]


def _plain_weigh(s):
    g = s["nh"] // s["nkv"]
    for b, i0, i1 in _last_parts(s):
        rows, r0, n = _slots(s, b), s["firsts"][b], s["lens"][b]
        for j in range(s["nkv"]):
            lse = s["lse"][r0 + i0:r0 + i1, j * g:(j + 1) * g].T
            w = torch.exp(_scores(s, b, j, i0, i1, rows) - lse[..., None]).sum((0, 1))
            w[:n] += s["decay"] * s["acc_in"][b, j, :n]
            s["acc_out"][b, j, :len(rows)] = w
        s["slot_pos"][b, :, n:len(rows)] = s["pos"][b] + torch.arange(len(rows) - n, dtype=torch.int32, device=DEV)
    return dict(acc=s["acc_out"], slot_pos=s["slot_pos"])


def _turned(x, w, cs, interleaved):
    """Heads [rows][heads][hd], in 64 bits: the rounding to a cache's type must not depend on the order of a sum."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    m = 2 * cs.shape[1]
    a, b = (x[..., 0:m:2], x[..., 1:m:2]) if interleaved else (x[..., :m // 2], x[..., m // 2:m])
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    y = x.clone()
    to_a, to_b = (y[..., 0:m:2], y[..., 1:m:2]) if interleaved else (y[..., :m // 2], y[..., m // 2:m])
    to_a.copy_(a * c - b * sn)
    to_b.copy_(a * sn + b * c)
    return y


def _plain_append(s):
    nh, nkv, hd = s["nh"], s["nkv"], s["hd"]
    x = s["qkv"].view(s["n_rows"], nh + 2 * nkv, hd)
    cs, at = s["rope"][s["row_pos"].long()], s["row_at"].long()
    q = _turned(x[:, :nh], s["q_norm"], cs, s["interleaved"]).float().to(s["qdtype"])
    k = _turned(x[:, nh:nh + nkv], s["k_norm"], cs, s["interleaved"])
    s["kpool"].view(-1, nkv, hd)[at] = k.float().to(s["kpool"].dtype)
    s["vpool"].view(-1, nkv, hd)[at] = x[:, nh + nkv:].to(s["vpool"].dtype)
    return dict(q=q, kpool=s["kpool"], vpool=s["vpool"])


def _plain_plan(s):
    page, table_len, n_pages, n_rows = s["page"], s["table_len"], s["n_pages"], s["n_rows"]
    n, held, new = s["len"].long(), s["held"].long().clamp(0, table_len), s["n_new"].long().clamp(min=0)
    first = torch.cumsum(new, 0) - new
    ok = (n >= 0) & (n + new <= table_len * page) & (first + new <= n_rows)
    new = torch.where(ok, new, 0)
    need = torch.where(n < 0, 0, (n + new + page - 1) // page)
    need = torch.where(n > table_len * page, held, need)
    stays = torch.minimum(held, torch.maximum(need, s["shared"].long()))
    entry = torch.arange(table_len, device=DEV)
    entries = s["table"]
    back = (entry >= stays[:, None]) & (entry < held[:, None]) & (entries >= 0) & (entries < n_pages)
    free = s["free"][:s["n_free"].long().clamp(0, n_pages)]
    stack = torch.cat([free, entries[back]])[:n_pages]
    asks = torch.where(ok & (new > 0), (need - held).clamp(min=0), 0)
    upto = torch.cumsum(asks, 0)
    given = ok & ((asks == 0) | (upto <= len(stack)))
    asks = torch.where(given, asks, 0)
    count = torch.where(given, new, 0)
    nth = (upto - asks)[:, None] + entry - held[:, None]
    fills = (entry >= held[:, None]) & (entry < (held + asks)[:, None])
    pad = torch.cat([stack, stack.new_full((1,), -1)])  # (of an empty stack: nothing is asked of it)
    s["table_out"].copy_(torch.where(fills, pad[(len(stack) - 1 - nth).clamp(0, max(0, len(stack) - 1))],
                                     torch.where(entry < stays[:, None], entries, -1)))
    s["held_out"].copy_(stays + asks)
    left = len(stack) - asks.sum()
    at = torch.arange(len(stack), device=DEV)
    s["free_out"][:len(stack)] = torch.where(at < left, stack, -1)
    s["n_free_out"].copy_(left)
    s["first"].copy_(first)
    s["count"].copy_(count)
    r = torch.arange(n_rows, device=DEV)
    b = (torch.searchsorted(first, r, right=True) - 1).clamp(min=0)
    i = r - first[b]
    mine = i < count[b]
    slot = torch.where(mine, n[b] + i, 0)
    e = s["table_out"].long()[b, slot // page]
    s["row_seq"].copy_(torch.where(mine, b, -1))
    s["row_pos"].copy_(torch.where(mine, s["pos"].long()[b] + i, -1))
    s["row_at"].copy_(torch.where(mine & (e >= 0) & (e < n_pages), e * page + slot % page, -1))
    return _plan_outputs(s)


def run(state):
    plain = dict(attn=_plain_attn, weigh=_plain_weigh, append=_plain_append, plan=_plain_plan)
    calls = dict(attn=_own_attn, weigh=_own_weigh, append=_own_append, plan=_own_plan)
    return (calls if own else plain)[state["kind"]](state)


# ------------------------------------------------------------------- work --
def _pairs(n, i0, i1, window):
    """Slots that the new tokens [i0, i1) of a sequence of n rows see, summed."""
    if not window:
        return sum(n + i + 1 for i in range(i0, i1))
    return sum(min(window, n + i + 1) for i in range(i0, i1))


def work(case):
    """Rows, heads, weights and entries read once, what changes written once."""
    lens, new = _shape(case)
    if case["kind"] == "plan":
        pages = sum(-(-(n + m) // case["page"]) for n, m in zip(lens, new))
        return dict(bytes=12.0 * sum(new) + 8.0 * pages + 36.0 * case["n_seq"], flops=8.0 * sum(new))
    nkv, hd, nh, es = case["nkv"], case["hd"], case["nkv"] * case["gqa"], TYPES[case["type"]][2]
    qs, rows = TYPES[case["qtype"]][2], sum(new)
    if case["kind"] == "append":
        tin = TYPES[case["tin"]][2]
        angles = set()
        for n, m in zip(lens, new):
            angles.update(range(n + n // 8, n + n // 8 + m))
        nb = rows * hd * (nh * (tin + qs) + 2 * nkv * (tin + es)) + len(angles) * 8 * case["n_rot"]
        return dict(bytes=float(nb), flops=8.0 * rows * (nh + nkv) * hd)
    w = case["window"]
    if case["kind"] == "attn":
        kept = sum(min(n, w - 1) + m if w else n + m for n, m in zip(lens, new))
        nb = 2 * kept * nkv * hd * es + 2 * rows * nh * hd * qs + (4 * rows * nh if case["lse"] else 0)
        pairs = sum(_pairs(n, 0, m, w) for n, m in zip(lens, new))
        return dict(bytes=float(nb), flops=4.0 * hd * nh * pairs)
    tail = [max(0, m - case["last"]) for m in new]
    kept = sum(min(n + i0, w - 1) + m - i0 if w else n + m for n, m, i0 in zip(lens, new, tail))
    count = sum(m - i0 for m, i0 in zip(new, tail))
    nb = kept * nkv * hd * es + count * nh * (hd * qs + 4) + 4 * nkv * (2 * sum(lens) + 2 * rows)
    return dict(bytes=float(nb), flops=2.0 * hd * nh * sum(_pairs(n, i0, m, w) for n, m, i0 in zip(lens, new, tail)))


# ------------------------------------------------------------------ exact --
def exact(case, seed):
    s = prepare(case, seed)
    return dict(attn=_exact_attn, weigh=_exact_weigh, append=_exact_append, plan=_exact_plan)[case["kind"]](s)


def _exact_rows(s, b, pool, j):
    """Slots [0, len + count) of a sequence's kv head from its pages, in 64 bits."""
    n = s["lens"][b] + s["new"][b]
    pages = s["table"][b, :-(-n // s["page"])].long()
    return pool[pages, :, j].reshape(-1, s["hd"])[:n].double()


def _exact_weights(s, b, h, i0, i1, k):
    """One query head's scores of new tokens [i0, i1) in 64 bits: exponents beside their largest, which is returned too."""
    r0, n = s["firsts"][b], s["lens"][b]
    x = s["q"][r0 + i0:r0 + i1, h].double() @ k.T * s["scale"]
    back = (n + torch.arange(i0, i1, device=DEV))[:, None] - torch.arange(len(k), device=DEV)
    x[back < 0] = -math.inf
    if s["window"]:
        x[back >= s["window"]] = -math.inf
    return x


def _exact_attn(s):
    g = s["nh"] // s["nkv"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(out.shape[:2], dtype=torch.float64, device=DEV)
    for b, m in enumerate(s["new"]):
        r0 = s["firsts"][b]
        for h in range(s["nh"]):
            k, v = (_exact_rows(s, b, s[p], h // g) for p in ("kpool", "vpool"))
            for i0 in range(0, m, 2048):
                i1 = min(m, i0 + 2048)
                x = _exact_weights(s, b, h, i0, i1, k)
                lse[r0 + i0:r0 + i1, h] = torch.logsumexp(x, -1)
                out[r0 + i0:r0 + i1, h] = torch.softmax(x, -1) @ v
    return dict(out=out) if s["lse"] is None else dict(out=out, lse=lse)


def _exact_weigh(s):
    g = s["nh"] // s["nkv"]
    acc, where = s["acc_out"].double(), s["slot_pos"].clone()
    for b, (n, m) in enumerate(zip(s["lens"], s["new"])):
        i0 = max(0, m - s["last"])
        r0 = s["firsts"][b]
        for j in range(s["nkv"]):
            k = _exact_rows(s, b, s["kpool"], j)
            acc[b, j, :n] = s["decay"] * s["acc_in"][b, j, :n].double()
            acc[b, j, n:n + m] = 0
            for h in range(j * g, j * g + g):
                x = _exact_weights(s, b, h, i0, m, k) - s["lse"][r0 + i0:r0 + m, h].double()[:, None]
                acc[b, j, :n + m] += x.exp().sum(0)
            for i in range(m):
                where[b, j, n + i] = int(2 * n + i)
    return dict(acc=acc, slot_pos=where)


def _exact_append(s):
    nh, nkv, hd, half = s["nh"], s["nkv"], s["hd"], s["n_rot"] // 2
    kpool, vpool = s["kpool"].double(), s["vpool"].double()
    z = torch.view_as_complex(s["rope"])[s["row_pos"].long()]
    i = torch.arange(half, device=DEV)
    a, b = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + half)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / hd + EPS) * w.double()
        t = torch.complex(x[..., a], x[..., b]) * z
        x = x.clone()
        x[..., a], x[..., b] = t.real, t.imag
        return x

    out = torch.stack([turned(s["qkv"][:, h * hd:(h + 1) * hd], s["q_norm"]) for h in range(nh)], 1)
    at = s["row_at"].long()
    for j in range(nkv):
        c = (nh + j) * hd
        kpool.view(-1, nkv, hd)[at, j] = turned(s["qkv"][:, c:c + hd], s["k_norm"])
        vpool.view(-1, nkv, hd)[at, j] = s["qkv"][:, c + nkv * hd:c + (nkv + 1) * hd].double()
    return dict(q=out, kpool=kpool, vpool=vpool)


def _exact_plan(s):
    """Sequence by sequence, with a list as the stack of free pages."""
    page, n_pages, n_rows = s["page"], s["n_pages"], s["n_rows"]
    table, held = s["table"].cpu().numpy().copy(), s["held"].tolist()
    stack = s["free"][:int(s["n_free"])].tolist()
    lens, new, pos = s["len"].tolist(), s["n_new"].tolist(), s["pos"].tolist()
    before, first, count = 0, [], []
    for m in new:
        first.append(before)
        before += m
    need = [0 if n < 0 else -(-(n + m) // page) for n, m in zip(lens, new)]
    for b, m in enumerate(need):
        keep = max(m, int(s["shared"][b]))
        if held[b] > keep:
            stack += table[b, keep:held[b]].tolist()
            table[b, keep:held[b]] = -1
            held[b] = keep
    top, none_left = len(stack), False
    for b, m in enumerate(need):
        ask = max(0, m - held[b])
        none_left = none_left or ask > len(stack)
        if ask and none_left:
            count.append(0)
            continue
        for e in range(held[b], held[b] + ask):
            table[b, e] = stack.pop()
        held[b] += ask
        count.append(new[b])
    free = np.full(n_pages, -1, np.int32)
    free[:len(stack)] = stack
    row = np.full((3, n_rows), -1, np.int32)
    for b, (f, m) in enumerate(zip(first, count)):
        t = lens[b] + np.arange(m)
        row[0, f:f + m] = b
        row[1, f:f + m] = pos[b] + np.arange(m)
        row[2, f:f + m] = table[b, t // page] * page + t % page
    i32 = lambda x: torch.from_numpy(np.ascontiguousarray(np.asarray(x, np.int32)))  # noqa: E731
    return dict(table_out=i32(table), held_out=i32(held), free_out=i32(free), n_free_out=i32([len(stack)]),
                first=i32(first), count=i32(count), row_seq=i32(row[0]), row_pos=i32(row[1]), row_at=i32(row[2]))
