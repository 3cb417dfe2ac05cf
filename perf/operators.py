"""The attention of a decoder layer over a paged cache, as the library's users
call it between wq/wk/wv and wo, with its plain forms.

A case's "kind" is one operator:

  rope     the q and k norms, the rotary positions and the append of k and v
           to the paged cache, from the projections' fp32 outputs
  attn     the attention of each sequence's new tokens (one, or a chunk) over
           its pages of the cache
  fork     the page tables of the next step from the parents that were picked,
           and the copies of the pages that may no longer be shared
  compact  the live pages moved to the front of the pool

"sequences", "new_lo" .. "new_hi" and "ctx_lo" .. "ctx_hi" say how many
sequences a batch has and the ranges of their new and earlier tokens; the
lengths themselves follow from "shape", so that a case always has the same
work.  "pad" rows follow the last sequence's and belong to none.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "inferno.jl_amd")
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
BASE = 1e6
ORIGINAL = 8192  # tokens that the scaled rotary tables extend


def listed():
    return [
        # a decode step of one sequence: normed heads, a far position
        {"name": "rope decode 1", "kind": "rope", "sequences": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 777, "ctx_hi": 777,
         "pad": 0, "far": 131000, "page": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "layout": "half",
         "norm": True, "scaling": "none", "act": "f32", "type": "f16", "shape": 1},
        # a decode step of a padded batch, a quarter of each wide head rotated
        {"name": "rope decode 61 partial", "kind": "rope", "sequences": 61, "new_lo": 1, "new_hi": 1, "ctx_lo": 3,
         "ctx_hi": 2000, "pad": 3, "far": 0, "page": 16, "q_heads": 16, "kv_heads": 2, "dim": 256, "rot": 64,
         "layout": "half", "norm": True, "scaling": "none", "act": "bf16", "type": "bf16", "shape": 2},
        # a long prompt with a rotary table scaled for a longer context
        {"name": "rope prompt 8192", "kind": "rope", "sequences": 1, "new_lo": 8192, "new_hi": 8192, "ctx_lo": 1024,
         "ctx_hi": 1024, "pad": 0, "far": 0, "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "layout": "interleaved", "norm": False, "scaling": "yarn", "act": "f16", "type": "f16", "shape": 3},
        # one token of a short chat: the smallest call
        {"name": "attn decode 1x777", "kind": "attn", "sequences": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 776, "ctx_hi": 776,
         "pad": 0, "page": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "act": "f32", "type": "f16", "window": 0,
         "cap": 0.0, "slopes": False, "prefix": 0, "shape": 4},
        # one token over a long document
        {"name": "attn decode 1x65537", "kind": "attn", "sequences": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 65536,
         "ctx_hi": 65536, "pad": 0, "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "act": "f32", "type": "f16",
         "window": 0, "cap": 0.0, "slopes": False, "prefix": 0, "shape": 5},
        # a served batch of sequences of many lengths
        {"name": "attn decode 61 ragged", "kind": "attn", "sequences": 61, "new_lo": 1, "new_hi": 1, "ctx_lo": 200,
         "ctx_hi": 16000, "pad": 3, "page": 16, "q_heads": 32, "kv_heads": 8, "dim": 128, "act": "bf16", "type": "bf16",
         "window": 0, "cap": 0.0, "slopes": False, "prefix": 0, "shape": 6},
        # drafted tokens verified together: a few rows a sequence, capped scores in a window, wide heads
        {"name": "attn verify 9x5 window", "kind": "attn", "sequences": 9, "new_lo": 2, "new_hi": 7, "ctx_lo": 30,
         "ctx_hi": 6000, "pad": 0, "page": 32, "q_heads": 16, "kv_heads": 8, "dim": 256, "act": "f32", "type": "bf16",
         "window": 1024, "cap": 50.0, "slopes": False, "prefix": 0, "shape": 7},
        # a prompt on the library's fp32 activations
        {"name": "attn prompt 2048 f32", "kind": "attn", "sequences": 1, "new_lo": 2048, "new_hi": 2048, "ctx_lo": 0,
         "ctx_hi": 0, "pad": 0, "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "act": "f32", "type": "f16",
         "window": 0, "cap": 0.0, "slopes": False, "prefix": 0, "shape": 8},
        # chunks of several prompts, distances as biases, a prefix that sees itself whole
        {"name": "attn chunks 5 ragged", "kind": "attn", "sequences": 5, "new_lo": 33, "new_hi": 900, "ctx_lo": 1,
         "ctx_hi": 5000, "pad": 11, "page": 16, "q_heads": 24, "kv_heads": 8, "dim": 64, "act": "f16", "type": "f16",
         "window": 0, "cap": 0.0, "slopes": True, "prefix": 300, "shape": 9},
        # a chunk of a very long prompt: the largest call
        {"name": "attn chunk 4096 over 32768", "kind": "attn", "sequences": 1, "new_lo": 4096, "new_hi": 4096,
         "ctx_lo": 32768, "ctx_hi": 32768, "pad": 0, "page": 64, "q_heads": 32, "kv_heads": 8, "dim": 128, "act": "bf16",
         "type": "bf16", "window": 0, "cap": 0.0, "slopes": False, "prefix": 0, "shape": 10},
        # a few sequences, each continued several ways
        {"name": "fork 7 to 29", "kind": "fork", "parents": 7, "children": 29, "ctx_lo": 5, "ctx_hi": 3000, "room": 1,
         "page": 16, "kv_heads": 8, "dim": 128, "layers": 4, "type": "f16", "shape": 11},
        # a pool that has become half empty
        {"name": "compact 4099 pages", "kind": "compact", "pages": 4099, "full": 0.55, "sequences": 40, "page": 16,
         "kv_heads": 8, "dim": 128, "layers": 4, "type": "bf16", "shape": 12},
    ]


def _log_int(rng, lo, hi):
    return lo if lo >= hi else min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1)))) - 1)))


def draw(rng):
    kind = rng.choice(("rope", "attn", "attn", "attn", "attn", "fork", "compact"))
    kv_heads, group = rng.choice(((8, 4), (8, 3), (4, 8), (2, 8), (8, 1), (1, 16), (4, 5), (2, 2), (8, 7)))
    dim = rng.choice((64, 80, 96, 128, 128, 128, 192, 256))
    kv = rng.choice(("f16", "bf16"))
    c = {"kind": kind, "kv_heads": kv_heads, "dim": dim, "page": rng.choice((16, 16, 32, 64, 128)), "type": kv,
         "shape": rng.randrange(1 << 30)}
    if kind == "fork":
        n = _log_int(rng, 2, 48)
        return c | {"parents": n, "children": _log_int(rng, 1, 4 * n), "ctx_lo": rng.randint(0, 40),
                    "ctx_hi": _log_int(rng, 60, 4000), "room": rng.randint(0, 40), "layers": rng.randint(1, 4),
                    "page": rng.choice((16, 32))}
    if kind == "compact":
        return c | {"pages": _log_int(rng, 64, 4100), "full": rng.uniform(0.2, 0.95), "sequences": rng.randint(1, 50),
                    "layers": rng.randint(1, 4), "page": 16}
    batch = rng.choice(("decode", "decode", "verify", "chunks", "prompt"))
    sequences = {"decode": _log_int(rng, 1, 96), "verify": _log_int(rng, 1, 32), "chunks": rng.randint(2, 8), "prompt": 1}[batch]
    new = {"decode": (1, 1), "verify": (1, rng.randint(2, 16)), "chunks": (rng.randint(1, 90), rng.randint(100, 1200)),
           "prompt": (_log_int(rng, 17, 4096),) * 2}[batch]
    ctx_hi = _log_int(rng, 16, 65536 if sequences < 4 else 16384)
    c |= {"sequences": sequences, "new_lo": new[0], "new_hi": new[1],
          "ctx_lo": ctx_hi if sequences == 1 else rng.randint(0, ctx_hi), "ctx_hi": ctx_hi, "pad": rng.choice((0, 0, 5)),
          "q_heads": kv_heads * group, "act": rng.choice(("f32", kv))}
    while c["sequences"] * c["new_hi"] * (c["new_hi"] + c["ctx_hi"]) * c["q_heads"] > 4.0e9:
        c["ctx_hi"] //= 2
        c["new_hi"] = max(c["new_lo"], c["new_hi"] * 3 // 4) if c["sequences"] > 1 else max(17, c["new_hi"] * 3 // 4)
        c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])
        c["new_lo"] = min(c["new_lo"], c["new_hi"]) if c["sequences"] > 1 else c["new_hi"]
    if kind == "rope":
        while c["ctx_hi"] > 4000:
            c["ctx_hi"] //= 2
        c["ctx_lo"] = min(c["ctx_lo"], c["ctx_hi"])
        return c | {"far": rng.choice((0, 0, rng.randint(1, 500000))), "rot": rng.choice((dim, dim, dim // 2, dim // 4)),
                    "layout": rng.choice(("half", "interleaved")), "norm": rng.random() < 0.5,
                    "scaling": rng.choice(("none", "linear", "ntk", "yarn", "bands"))}
    return c | {"window": rng.choice((0, 0, 0, rng.randint(1, 4096))), "cap": rng.choice((0.0, 0.0, 30.0, 50.0)),
                "slopes": rng.random() < 0.2, "prefix": rng.choice((0, 0, 0, rng.randint(1, 600)))}


# ---- what a case's batch is --------------------------------------------------
def _lengths(case):
    """(new tokens, all tokens) of each sequence."""
    r = random.Random(case["shape"])
    new = [_log_int(r, case["new_lo"], case["new_hi"]) for _ in range(case["sequences"])]
    return new, [n + _log_int(r, case["ctx_lo"], case["ctx_hi"]) for n in new]


def _prefixes(case):
    r = random.Random(case["shape"] + 1)
    return [r.randint(0, case["prefix"]) for _ in range(case["sequences"])]


def _forks(case):
    """(tokens of each parent, each child's parent): some parents twice, some never, the last child of none."""
    r = random.Random(case["shape"])
    lens = [_log_int(r, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["parents"])]
    parents = [r.randrange(case["parents"]) for _ in range(case["children"])]
    if case["children"] > 2:
        parents[-1] = -1
    return lens, parents


def _spans(case):
    """Pages of each sequence of a pool to compact."""
    r = random.Random(case["shape"])
    used = int(case["pages"] * case["full"])
    cuts = sorted(r.randint(0, used) for _ in range(case["sequences"] - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [used])]


def _pages(tokens, page):
    return -(-tokens // page)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tables(counts, width, order):
    """Page tables of `width` entries: row s holds the next counts[s] pages of `order`, then -1."""
    rows = np.repeat(np.arange(len(counts)), counts)
    cols = np.concatenate([np.arange(n) for n in counts]) if len(rows) else rows
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    table[torch.from_numpy(rows).cuda(), torch.from_numpy(cols).cuda()] = order[:len(rows)].to(torch.int32)
    return table


def _device():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from inferno_hip import device
    return device


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, page = case["kind"], case["page"]
    s = {"case": case}

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def pool(pages):
        return normal(pages, case["kv_heads"], page, case["dim"], dtype=DTYPES[case["type"]])

    if kind in ("fork", "compact"):
        if kind == "fork":
            lens, parents = _forks(case)
            counts = [_pages(n, page) for n in lens]
            most = max(counts + [1]) + _pages(case["room"], page) + 1
            pages = sum(counts) + case["children"] * (_pages(case["room"], page) + 1) + 5
            order = torch.randperm(pages, generator=g, device="cuda")
            s["table"], s["lens"], s["parents"] = _tables(counts, most, order), _ints(lens), _ints(parents)
        else:
            pages, counts = case["pages"], _spans(case)
            order = torch.randperm(pages, generator=g, device="cuda")
            s["table"] = _tables(counts, max(counts), order)
            s["table"][-1, :counts[0]] = s["table"][0, :counts[0]]  # the last sequence has become a fork of the first
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda")
        flat = s["table"].reshape(-1)
        s["refs"].scatter_add_(0, flat.clamp(min=0).long(), (flat >= 0).to(torch.int32))
        s["k"] = torch.stack([pool(pages) for _ in range(case["layers"])])
        s["v"] = torch.stack([pool(pages) for _ in range(case["layers"])])
        if own:
            s["cache"] = _device().KVCache(s["k"], s["v"])
        return s

    new, lens = _lengths(case)
    counts = [_pages(n, page) for n in lens]
    pages = sum(counts) + 3
    s["table"] = _tables(counts, max(counts), torch.randperm(pages, generator=g, device="cuda"))
    s["k"], s["v"] = pool(pages), pool(pages)
    s["starts"], s["lens"] = _ints([0] + list(np.cumsum(new))), _ints(lens)
    s["live"], s["tokens"], s["most_new"], s["most_len"] = sum(new), sum(new) + case["pad"], max(new), max(lens)
    heads, dim = case["q_heads"], case["dim"]
    s["out"] = torch.zeros(s["tokens"], heads, dim, dtype=DTYPES[case["act"]], device="cuda")
    if kind == "rope":
        qkv = 1.5 * normal(s["tokens"], heads + 2 * case["kv_heads"], dim)
        s["q"], s["x"], s["y"] = qkv[:, :heads], qkv[:, heads:heads + case["kv_heads"]], qkv[:, heads + case["kv_heads"]:]
        s["q_norm"], s["k_norm"] = (1 + 0.1 * normal(dim), 1 + 0.1 * normal(dim)) if case["norm"] else (None, None)
        at = np.concatenate([np.arange(b - a, b) for a, b in zip(new, lens)] + [np.zeros(case["pad"], np.int64)])
        s["positions"] = _ints(at + case["far"]) if case["far"] else None
        turns, s["mscale"] = _turns(case["rot"], case["scaling"])
        s["turns"] = torch.from_numpy(turns).cuda()
    else:
        s["q"] = (1.5 * normal(s["tokens"], heads, dim)).to(DTYPES[case["act"]])
        s["prefix"] = _ints(_prefixes(case)) if case["prefix"] else None
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if case["slopes"] else None
        # slots that no token has filled hold what the allocation left there
        full = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        at = torch.arange(s["most_len"], device="cuda")
        ids, seen = s["table"][:, at // page].clamp(min=0).long(), at < s["lens"][:, None]
        full.view(-1).index_put_(((ids * page + at % page)[seen],), torch.tensor(True, device="cuda"))
        s["k"].masked_fill_(~full[:, None, :, None], float("nan"))
        s["v"].masked_fill_(~full[:, None, :, None], float("nan"))
    if own:
        D = _device()
        s["cache"] = D.KVCache(s["k"], s["v"])
        s["batch"] = D.KVBatch(s["starts"], s["lens"], s["table"], s["tokens"])
        if kind == "attn":
            s["workspace"] = D.attn_workspace(heads, s["cache"], s["batch"])
    return s


def _turns(rot, scaling):
    """Turns per position of each rotated pair, in 64 bits, and the factor on the rotated values."""
    i = np.arange(rot // 2, dtype=np.float64)
    f = BASE ** (-2 * i / rot)
    factor, m = 4.0, 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "ntk":
        f = (BASE * factor ** (rot / (rot - 2))) ** (-2 * i / rot)
    elif scaling == "yarn":
        low, high = (rot * math.log(ORIGINAL / (b * 2 * math.pi)) / (2 * math.log(BASE)) for b in (32, 1))
        low, high = max(math.floor(low), 0), min(math.ceil(high), rot - 1)
        keep = 1 - np.clip((i - low) / max(high - low, 0.001), 0, 1)
        f, m = f / factor * (1 - keep) + f * keep, 0.1 * math.log(factor) + 1
    elif scaling == "bands":
        smooth = np.clip((ORIGINAL * f / (2 * math.pi) - 1) / 3, 0, 1)
        f = f / factor * (1 - smooth) + f * smooth
    return f / (2 * math.pi), m


# ---- the operators -------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    return {"rope": _rope, "attn": _attn, "fork": _fork, "compact": _compact}[kind](state)


def _rope(s):
    c = s["case"]
    if own:
        D = _device()
        D.rope_kv(s["q"], s["x"], s["y"], s["turns"], s["cache"], s["batch"], layout=c["layout"], mscale=s["mscale"],
                  q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, positions=s["positions"], out=s["out"])
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    live, page = s["live"], c["page"]
    seq = torch.searchsorted(s["starts"], torch.arange(live, device="cuda", dtype=torch.int32), right=True) - 1
    at = s["lens"][seq] - s["starts"][seq + 1] + torch.arange(live, device="cuda")
    pos = at if s["positions"] is None else s["positions"][:live]
    t = pos.double()[:, None] * s["turns"]
    t = (t - t.round()) * (2 * math.pi)
    cos, sin = (s["mscale"] * t.cos()).float()[:, None], (s["mscale"] * t.sin()).float()[:, None]

    def turned(x, w):
        x = x[:live]
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        r = c["rot"]
        if c["layout"] == "half":
            a, b = x[..., :r // 2], x[..., r // 2:r]
            y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
        else:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        return torch.cat((y, x[..., r:]), -1)

    s["out"][:live] = turned(s["q"], s["q_norm"]).to(s["out"].dtype)
    ids = s["table"][seq, at // page].long()
    s["k"][ids, :, at % page] = turned(s["x"], s["k_norm"]).to(s["k"].dtype)
    s["v"][ids, :, at % page] = s["y"][:live].to(s["v"].dtype)
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _attn(s):
    c = s["case"]
    if own:
        return _device().attn_paged(s["q"], s["cache"], s["batch"], window=c["window"], softcap=c["cap"],
                                    prefix_lens=s["prefix"], slopes=s["slopes"], out=s["out"], workspace=s["workspace"])
    S, H, G, D, page = c["sequences"], c["kv_heads"], c["q_heads"] // c["kv_heads"], c["dim"], c["page"]
    Q, C, T = s["most_new"], s["most_len"], s["tokens"]
    lens, starts = s["lens"].long(), s["starts"].long()
    new = starts[1:] - starts[:-1]
    at, i = torch.arange(C, device="cuda"), torch.arange(Q, device="cuda")
    seen = at < lens[:, None]
    ids = s["table"][:, at // page].clamp(min=0).long()

    def cached(pool):
        return torch.where(seen[:, :, None, None], pool[ids, :, at % page].float(), 0.0)  # S, C, H, D

    q = s["q"][(starts[:-1, None] + i).clamp(max=T - 1)].float().view(S, Q, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(S, H, G * Q, D)
    p = torch.matmul(q, cached(s["k"]).permute(0, 2, 3, 1).contiguous()).mul_(D ** -0.5)
    if c["cap"]:
        p = p.div_(c["cap"]).tanh_().mul_(c["cap"])
    apart = (lens - new)[:, None, None] + i[:, None] - at  # S, Q, C
    p = p.view(S, H, G, Q, C)
    if s["slopes"] is not None:
        p -= s["slopes"].view(1, H, G, 1, 1) * apart.abs()[:, None, None]
    visible = apart >= 0
    if s["prefix"] is not None:
        visible |= at < s["prefix"][:, None, None]
    if c["window"]:
        visible &= apart < c["window"]
    visible &= seen[:, None]
    p.masked_fill_(~visible[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(p.view(S, H, G * Q, C), cached(s["v"]).permute(0, 2, 1, 3).contiguous()).view(S, H, G, Q, D) / total
    t = torch.arange(T, device="cuda")
    seq = torch.searchsorted(starts, t, right=True) - 1
    inside = seq < S
    seq = seq.clamp(max=S - 1)
    o = o.permute(0, 3, 1, 2, 4)[seq, (t - starts[seq]).clamp(max=Q - 1)].reshape(T, H * G, D)
    s["out"].copy_(torch.where(inside[:, None, None], o, s["out"].float()))
    return s["out"]


def _held(table, pages):
    flat = table.reshape(-1)
    return torch.zeros(pages, dtype=torch.int32, device="cuda").scatter_add_(0, flat.clamp(min=0).long(), (flat >= 0).to(torch.int32))


def _copied(s, copies):
    pairs = copies[copies[:, 0] >= 0].long()
    for pool in (s["k"], s["v"]):
        pool[:, pairs[:, 1]] = pool[:, pairs[:, 0]]


def _fork(s):
    c = s["case"]
    if own:
        D = _device()
        refs = s["refs"].clone()
        table, lens, copies = D.kv_fork(s["table"], s["lens"], s["parents"], refs, c["page"], room=c["room"])
        D.kv_copy(s["cache"], copies)
        return {"table": table, "lens": lens, "refs": refs, "copies": copies, "k": s["k"], "v": s["v"]}
    page, width, pages = c["page"], s["table"].shape[1], s["refs"].numel()
    parents = s["parents"].long()
    alive, p, j = parents >= 0, parents.clamp(min=0), torch.arange(width, device="cuda")
    first = alive & ~(parents[:, None] == parents).tril(-1).any(1)
    lens = torch.where(alive, s["lens"][p], 0)
    full, need = lens // page, ((lens + c["room"] + page - 1) // page).clamp(max=width)
    row = s["table"][p]
    keep = alive[:, None] & (row >= 0) & (first[:, None] | (j < full[:, None]))
    table = torch.where(keep, row, -1)
    refs = s["refs"] - _held(s["table"], pages) + _held(table, pages)
    fresh = ~keep & (j < need[:, None])
    rank = (fresh.reshape(-1).cumsum(0) - 1).view_as(fresh)
    free = refs == 0
    order = torch.argsort((~free).to(torch.int32), stable=True)
    got = torch.where(rank < free.sum(), order[rank.clamp(0, pages - 1)], -1).to(torch.int32)
    given = torch.where(fresh, got, -1)
    refs = refs + _held(given, pages)
    table = torch.where(fresh, got, table)
    at = full.clamp(max=width - 1)[:, None].long()
    pairs = torch.cat((row.gather(1, at), table.gather(1, at)), 1)
    copied = (alive & ~first & (lens % page != 0))[:, None] & (pairs >= 0).all(1, keepdim=True)
    copies = torch.where(copied, pairs, -1)
    _copied(s, copies)
    return {"table": table, "lens": lens, "refs": refs, "copies": copies, "k": s["k"], "v": s["v"]}


def _compact(s):
    if own:
        D = _device()
        refs, table = s["refs"].clone(), s["table"].clone()
        copies, moved = D.kv_compact(table, refs)
        D.kv_copy(s["cache"], copies, moved)
        return {"table": table, "refs": refs, "copies": copies, "moved": moved, "k": s["k"], "v": s["v"]}
    pages = s["refs"].numel()
    at, used = torch.arange(pages, device="cuda"), s["refs"] > 0
    n = used.sum()
    move, hole = used & (at >= n), ~used & (at < n)
    rank = move.cumsum(0) - 1
    holes = torch.argsort((~hole).to(torch.int32), stable=True)
    to = torch.where(move, holes[rank.clamp(min=0)], at)
    table = torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].to(torch.int32), s["table"])
    refs = torch.zeros_like(s["refs"]).scatter_add_(0, to, s["refs"])
    copies = torch.full((pages // 2 + 1, 2), -1, dtype=torch.int32, device="cuda")
    copies[torch.where(move, rank, pages // 2)] = torch.where(move[:, None], torch.stack((at, to), 1), -1).to(torch.int32)
    copies = copies[:pages // 2]
    _copied(s, copies)
    return {"table": table, "refs": refs, "copies": copies, "moved": move.sum().to(torch.int32).reshape(1), "k": s["k"], "v": s["v"]}


# ---- what a pass cannot do without ------------------------------------------------
def work(case):
    size = 4 if case.get("act") == "f32" else 2
    if case["kind"] in ("rope", "attn"):
        new, lens = _lengths(case)
        head = case["dim"] * (case["q_heads"] * size if case["kind"] == "attn" else case["q_heads"] * 4)
        if case["kind"] == "rope":
            kv = case["kv_heads"] * case["dim"]
            per = head + 2 * kv * 4 + case["q_heads"] * case["dim"] * size + 2 * kv * 2
            return {"bytes": sum(new) * per, "flops": sum(new) * 3 * case["rot"] * (case["q_heads"] + case["kv_heads"])}
        pairs = keys = 0
        for n, m, pre in zip(new, lens, _prefixes(case)):
            a = np.arange(m - n, m)
            low = np.maximum(a - case["window"] + 1, 0) if case["window"] else np.zeros_like(a)
            high = np.maximum(a + 1, min(pre, m))
            pairs += int((high - low).sum())
            keys += int(high.max() - low.min())
        return {"bytes": 2 * sum(new) * head + keys * 2 * case["kv_heads"] * case["dim"] * 2,
                "flops": 4 * case["dim"] * case["q_heads"] * pairs}
    page = case["page"] * case["kv_heads"] * case["dim"] * 2 * 2 * case["layers"]
    if case["kind"] == "fork":
        lens, parents = _forks(case)
        moved = sum(1 for c, p in enumerate(parents) if p >= 0 and p in parents[:c] and lens[p] % case["page"])
        ints = sum(_pages(n, case["page"]) for n in lens) + sum(_pages(lens[p], case["page"]) for p in parents if p >= 0)
    else:
        counts = _spans(case)
        used = sum(counts) - (min(counts[0], counts[-1]) if len(counts) > 1 else 0)
        moved, ints = used * (case["pages"] - used) // case["pages"], 2 * case["pages"]
    return {"bytes": 2 * moved * page + 4 * ints, "flops": 0}


# ---- from the definitions, in 64 bits -----------------------------------------------
def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"rope": _exact_rope, "attn": _exact_attn, "fork": _exact_fork, "compact": _exact_compact}[case["kind"]](s)


def _exact_rope(s):
    c = s["case"]
    new, lens = _lengths(c)
    k, v, out = s["k"].double(), s["v"].double(), s["out"].double()
    row = 0
    for n, m, pages in zip(new, lens, s["table"].cpu().tolist()):
        at = torch.arange(m - n, m, device="cuda")
        # e^(i angle) of every (token, pair), on complex numbers
        spin = torch.polar(torch.full((), s["mscale"], dtype=torch.float64, device="cuda"),
                           torch.remainder((at + c["far"]).double()[:, None] * s["turns"], 1.0) * (2 * math.pi))
        for x, w, head in ((s["q"], s["q_norm"], True), (s["x"], s["k_norm"], False)):
            x = x[row:row + n].double()
            if w is not None:
                x = w.double() * x * (x.pow(2).sum(2, keepdim=True) / c["dim"] + EPS).pow(-0.5)
            r = x[..., :c["rot"]]
            z = r.unflatten(2, (2, -1)).transpose(2, 3) if c["layout"] == "half" else r.unflatten(2, (-1, 2))
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * spin[:, None])
            r = (z.transpose(2, 3) if c["layout"] == "half" else z).flatten(2)
            x = torch.cat((r, x[..., c["rot"]:]), 2)
            if head:
                out[row:row + n] = x
            else:
                keys = x
        slot = torch.tensor(pages, device="cuda")[at // c["page"]]
        k[slot, :, at % c["page"]] = keys
        v[slot, :, at % c["page"]] = s["y"][row:row + n].double()
        row += n
    return {"q": out, "k": k, "v": v}


def _exact_attn(s):
    c = s["case"]
    new, lens = _lengths(c)
    G, page = c["q_heads"] // c["kv_heads"], c["page"]
    out = s["out"].double()
    row = 0
    for n, m, pre, ids in zip(new, lens, _prefixes(c), s["table"].cpu().tolist()):
        ids = torch.tensor(ids[:_pages(m, page)], device="cuda")
        i, j = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")
        hidden = j > i
        if c["prefix"]:
            hidden = hidden & (j >= pre)
        if c["window"]:
            hidden = hidden | (j <= i - c["window"])
        for h in range(c["q_heads"]):
            k = s["k"][ids, h // G].reshape(-1, c["dim"])[:m].double()
            v = s["v"][ids, h // G].reshape(-1, c["dim"])[:m].double()
            z = s["q"][row:row + n, h].double() @ k.T / math.sqrt(c["dim"])
            if c["cap"]:
                z = c["cap"] * torch.tanh(z / c["cap"])
            if c["slopes"]:
                z = z - s["slopes"][h].double() * (i - j).abs()
            out[row:row + n, h] = torch.softmax(z.masked_fill(hidden, -math.inf), 1) @ v
        row += n
    return out


def _exact_pools(s, pairs):
    k, v = s["k"].double(), s["v"].double()
    for a, b in pairs:
        k[:, b], v[:, b] = s["k"][:, a].double(), s["v"][:, a].double()
    return k, v


def _exact_fork(s):
    c = s["case"]
    lens, parents = _forks(c)
    rows, refs, page = s["table"].cpu().tolist(), s["refs"].cpu().tolist(), c["page"]
    width, taken, out = len(rows[0]), set(), []
    for p in parents:
        held = [x for x in rows[p] if x >= 0] if p >= 0 else []
        out.append(held if p not in taken else held[:lens[p] // page])
        taken.add(p)
    for n, held in ((-1, rows), (1, out)):
        for x in (x for r in held for x in r if x >= 0):
            refs[x] += n
    free = [x for x, n in enumerate(refs) if n == 0][::-1]
    pairs = []
    for child, p in enumerate(parents):
        n = lens[p] if p >= 0 else 0
        pair, had = (-1, -1), len(out[child])
        while len(out[child]) < min(width, _pages(n + c["room"], page)):
            out[child].append(free.pop() if free else -1)
            refs[out[child][-1]] += 1
        if p >= 0 and p in parents[:child] and n % page and had < len(out[child]):
            pair = (rows[p][n // page], out[child][n // page])
        pairs.append(pair)
    k, v = _exact_pools(s, [x for x in pairs if x[0] >= 0])
    table = torch.tensor([r + [-1] * (width - len(r)) for r in out])
    return {"table": table, "lens": torch.tensor([lens[p] if p >= 0 else 0 for p in parents]), "refs": torch.tensor(refs),
            "copies": torch.tensor(pairs), "k": k, "v": v}


def _exact_compact(s):
    refs, table = s["refs"].cpu().tolist(), s["table"].cpu().tolist()
    pages, n = len(refs), sum(x > 0 for x in refs)
    movers = [x for x in range(n, pages) if refs[x] > 0]
    to = dict(zip(movers, (x for x in range(n) if refs[x] == 0)))
    for a, b in to.items():
        refs[a], refs[b] = 0, refs[a]
    k, v = _exact_pools(s, to.items())
    pairs = list(to.items()) + [(-1, -1)] * (pages // 2 - len(to))
    return {"table": torch.tensor([[to.get(x, x) for x in r] for r in table]), "refs": torch.tensor(refs),
            "copies": torch.tensor(pairs), "moved": torch.tensor([len(to)]), "k": k, "v": v}
