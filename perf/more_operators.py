"""A step of a model with recurrent layers, where the library's projections end:
the short convolution and the gated delta rule between a recurrent layer's
projections, and the choice of the next token from the lm_head's logits; as the
library's users call them, with their plain forms.

A case's "kind" is one operator:

  conv    the causal convolution over each channel's last few inputs, with the
          inputs that a sequence keeps from one call to the next
  delta   the gated delta rule: norms of q and k, decay and write strength from
          their projections, the state of every head, the gated output norm
  sample  a token per row of logits by temperature, top-k, top-p and min-p, and
          the logarithm of its share of what those left

"sequences", "new_lo" .. "new_hi" say how many sequences a batch has and the
range of their new tokens, "begin" the share of them that begin with this call;
the lengths themselves follow from "shape", so that a case always has the same
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
CHUNK = 64  # tokens that the plain form of the delta rule takes at once


def listed():
    heads = {"k_heads": 16, "v_heads": 32, "k_dim": 128, "v_dim": 128}
    return [
        # one token of a chat: the smallest call
        {"name": "conv decode 1", "kind": "conv", "sequences": 1, "new_lo": 1, "new_hi": 1, "begin": 0.0, "pad": 0,
         "channels": 6144, "width": 4, "bias": False, "silu": True, "act": "f32", "type": "f32", "shape": 1},
        # chunks of several prompts, some of which go on
        {"name": "conv chunks 5 ragged", "kind": "conv", "sequences": 5, "new_lo": 33, "new_hi": 900, "begin": 0.5, "pad": 11,
         "channels": 2560, "width": 3, "bias": True, "silu": True, "act": "f32", "type": "f16", "shape": 2},
        # a long prompt
        {"name": "conv prompt 8192", "kind": "conv", "sequences": 1, "new_lo": 8192, "new_hi": 8192, "begin": 1.0, "pad": 0,
         "channels": 8192, "width": 4, "bias": False, "silu": True, "act": "f32", "type": "bf16", "shape": 3},
        # one token of a chat, with the output norm
        {"name": "delta decode 1", "kind": "delta", "sequences": 1, "new_lo": 1, "new_hi": 1, "begin": 0.0, "pad": 0, **heads,
         "gate": True, "type": "f32", "out": "f32", "shape": 4},
        # a served batch, padded
        {"name": "delta decode 61", "kind": "delta", "sequences": 61, "new_lo": 1, "new_hi": 1, "begin": 0.0, "pad": 3, **heads,
         "gate": True, "type": "f32", "out": "f32", "shape": 5},
        # drafted tokens that are verified together
        {"name": "delta verify 9x5", "kind": "delta", "sequences": 9, "new_lo": 2, "new_hi": 7, "begin": 0.0, "pad": 0,
         **heads, "v_heads": 16, "gate": True, "type": "bf16", "out": "f32", "shape": 6},
        # chunks of several prompts beside a few short ones, narrow heads
        {"name": "delta chunks 5 ragged", "kind": "delta", "sequences": 5, "new_lo": 3, "new_hi": 900, "begin": 0.5, "pad": 11,
         "k_heads": 8, "v_heads": 24, "k_dim": 64, "v_dim": 64, "gate": False, "type": "f16", "out": "f16", "shape": 7},
        # a prompt on the library's fp32 activations
        {"name": "delta prompt 2048 f32", "kind": "delta", "sequences": 1, "new_lo": 2048, "new_hi": 2048, "begin": 1.0, "pad": 0,
         **heads, "v_heads": 16, "gate": True, "type": "f32", "out": "f32", "shape": 8},
        # a long prompt: the largest call
        {"name": "delta prompt 8192", "kind": "delta", "sequences": 1, "new_lo": 8192, "new_hi": 8192, "begin": 1.0, "pad": 0,
         **heads, "gate": True, "type": "bf16", "out": "bf16", "shape": 9},
        # one token of a chat, all filters on
        {"name": "sample 1", "kind": "sample", "rows": 1, "vocab": 151936, "type": "f32", "filters": "all", "masked": 0.0,
         "shape": 10},
        # a served batch, every request with its own settings, some tokens ruled out by a grammar
        {"name": "sample 61 mixed", "kind": "sample", "rows": 61, "vocab": 151936, "type": "bf16", "filters": "mixed",
         "masked": 0.3, "shape": 11},
        # a large batch at a temperature, without filters
        {"name": "sample 256 plain", "kind": "sample", "rows": 256, "vocab": 151936, "type": "f32", "filters": "plain",
         "masked": 0.0, "shape": 12},
    ]


def _log_int(rng, lo, hi):
    return lo if lo >= hi else min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1)))) - 1)))


def draw(rng):
    kind = rng.choice(("conv", "delta", "delta", "delta", "sample", "sample"))
    c = {"kind": kind, "shape": rng.randrange(1 << 30)}
    if kind == "sample":
        vocab = _log_int(rng, 1000, 262144)
        return c | {"rows": _log_int(rng, 1, min(256, 38_000_000 // vocab)), "vocab": vocab,
                    "type": rng.choice(("f32", "f32", "f16", "bf16")), "filters": rng.choice(("all", "mixed", "mixed", "plain")),
                    "masked": rng.choice((0.0, 0.0, 0.2, 0.9))}
    batch, kept = rng.choice(("decode", "verify", "chunks", "prompt", "prompt")), rng.choice(("f32", "f16", "bf16"))
    sequences = {"decode": _log_int(rng, 1, 64), "verify": _log_int(rng, 1, 32), "chunks": rng.randint(2, 8), "prompt": 1}[batch]
    new = {"decode": (1, 1), "verify": (1, rng.randint(2, 16)), "chunks": (rng.randint(1, 90), rng.randint(100, 900)),
           "prompt": (_log_int(rng, 17, 4096 if kept == "f32" else 8192),) * 2}[batch]
    c |= {"sequences": sequences, "new_lo": new[0], "new_hi": new[1], "begin": 0.0 if batch == "decode" else rng.choice((0.0, 0.5, 1.0)),
          "pad": rng.choice((0, 0, 5)), "type": kept}
    if kind == "conv":
        return c | {"channels": 8 * _log_int(rng, 40, 1024), "width": rng.choice((4, 4, 4, 2, 3, 5)), "bias": rng.random() < 0.3,
                    "silu": rng.random() < 0.8, "act": rng.choice(("f32", "f32", c["type"]))}
    k_heads, group = rng.choice(((16, 1), (16, 2), (8, 2), (4, 3), (2, 8), (8, 4), (3, 5)))
    dim = rng.choice((64, 80, 96, 128, 128, 128))
    return c | {"k_heads": k_heads, "v_heads": k_heads * group, "k_dim": dim, "v_dim": rng.choice((dim, dim, 64, 112)),
                "gate": rng.random() < 0.6, "out": rng.choice((c["type"], c["type"], "f32"))}


# ---- what a case's batch is --------------------------------------------------
def _lengths(case):
    """(new tokens, all tokens) of each sequence; they are equal where it begins."""
    r = random.Random(case["shape"])
    new = [_log_int(r, case["new_lo"], case["new_hi"]) for _ in range(case["sequences"])]
    return new, [n if r.random() < case["begin"] else n + r.randint(1, 5000) for n in new]


def _settings(case):
    """(temperature, top_k, top_p, min_p) of each row; None where no row has one."""
    r, n = random.Random(case["shape"]), case["rows"]
    if case["filters"] == "plain":
        return [r.choice((0.7, 1.0)) for _ in range(n)], None, None, None
    if case["filters"] == "all":
        return [0.8] * n, [50] * n, [0.95] * n, [0.02] * n
    return ([r.choice((0.0, 0.3, 0.6, 0.8, 1.0, 1.5)) for _ in range(n)], [r.choice((0, 0, 1, 20, 64, 1000)) for _ in range(n)],
            [r.choice((1.0, 0.5, 0.9, 0.95, 0.999)) for _ in range(n)], [r.choice((0.0, 0.0, 0.05, 0.2)) for _ in range(n)])


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _device():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from inferno_hip import device
    return device


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    s = {"case": case}

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(lo, hi, *shape):
        return lo + (hi - lo) * torch.rand(shape, generator=g, device="cuda")

    if kind == "sample":
        n, vocab = case["rows"], case["vocab"]
        x = 2 * normal(n, vocab)
        x += 14 * uniform(0, 1, n, vocab).pow(2) * (uniform(0, 1, n, vocab) < 2e-4)  # the few tokens that fit
        s["logits"] = x.to(DTYPES[case["type"]])
        if case["masked"]:
            out = uniform(0, 1, n, vocab) < case["masked"]
            s["logits"].masked_fill_(out, -math.inf)
            s["logits"][::2].masked_fill_(out[::2], torch.finfo(DTYPES[case["type"]]).min)
        for name, v in zip(("temperature", "top_k", "top_p", "min_p"), _settings(case)):
            s[name] = None if v is None else _ints(v) if name == "top_k" else torch.tensor(v, device="cuda")
        s["u"] = torch.rand(n, generator=g, device="cuda")
        s["tokens"], s["logprobs"] = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
        if own:
            s["workspace"] = _device().sample_workspace(n, vocab)
        return s

    new, lens = _lengths(case)
    n, slots = case["sequences"], case["sequences"] + 3
    s["starts"], s["lens"] = _ints([0] + list(np.cumsum(new))), _ints(lens)
    s["slots"] = torch.randperm(slots, generator=g, device="cuda")[:n].int()
    s["live"], s["tokens"], s["most"] = sum(new), sum(new) + case["pad"], max(new)
    begins = s["lens"] == s["starts"][1:] - s["starts"][:-1]
    if kind == "conv":
        C, W = case["channels"], case["width"]
        s["x"] = (1.5 * normal(s["tokens"], C)).to(DTYPES[case["act"]])
        s["w"], s["bias"] = 0.5 * normal(C, W), 0.1 * normal(C) if case["bias"] else None
        s["state"] = normal(slots, W - 1, C)
        s["out"] = torch.zeros(s["tokens"], C, dtype=DTYPES[case["type"]], device="cuda")
    else:
        K, H, dk, dv, T = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"], s["tokens"]
        x = 1.5 * normal(T, 2 * K * dk + H * dv)
        s["qkv"] = (x * torch.sigmoid(x)).to(DTYPES[case["type"]])  # as the short convolution leaves it
        s["q"], s["k"] = (s["qkv"][:, i * K * dk:(i + 1) * K * dk].view(T, K, dk) for i in (0, 1))
        s["v"] = s["qkv"][:, 2 * K * dk:].view(T, H, dv)
        ab = normal(T, 2 * H)
        s["a"], s["b"] = ab[:, :H], ab[:, H:]
        s["decay"] = -torch.exp(uniform(0, math.log(16), H))
        dt = torch.exp(uniform(math.log(0.001), math.log(0.1), H))
        s["dt_bias"] = dt + torch.log(-torch.expm1(-dt))
        s["z"] = normal(T, H, dv) if case["gate"] else None
        s["norm"] = 1 + 0.1 * normal(dv) if case["gate"] else None
        s["state"] = 0.3 * normal(slots, H, dk, dv)
        s["out"] = torch.zeros(T, H, dv, dtype=DTYPES[case["out"]], device="cuda")
    s["state"][s["slots"][begins].long()] = float("nan")  # whatever the slot's last owner left
    if own:
        D = _device()
        s["batch"] = D.StateBatch(s["starts"], s["slots"], s["tokens"], kv_lens=s["lens"], most=s["most"])
        if kind == "delta":
            s["layer"] = D.DeltaLayer(s["state"], case["k_heads"], s["decay"], s["dt_bias"], norm_w=s["norm"], norm_eps=EPS,
                                      l2_eps=EPS)
            s["workspace"] = D.delta_workspace(s["layer"], s["batch"], s["qkv"].dtype)
    return s


# ---- the operators -------------------------------------------------------------
def run(state):
    return {"conv": _conv, "delta": _delta, "sample": _sample}[state["case"]["kind"]](state)


def _rows(s, width):
    """Rows (sequences x width) of the new tokens, whether they are any, and which sequences begin."""
    starts = s["starts"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(width, device="cuda")
    return (starts[:-1, None] + i).clamp(max=s["tokens"] - 1), i < new[:, None], s["lens"] == new, new


def _conv(s):
    c = s["case"]
    if own:
        _device().short_conv(s["x"], s["w"], s["state"], s["batch"], bias=s["bias"], silu=c["silu"], out=s["out"])
        return {"out": s["out"], "state": s["state"]}
    W = c["width"]
    rows, live, begins, new = _rows(s, s["most"])
    slots = s["slots"].long()
    old = torch.where(begins[:, None, None], 0.0, s["state"][slots])
    x = torch.cat((old, s["x"][rows].float()), 1)  # sequences x (W - 1 + most) x channels
    y = sum(x[:, j:j + s["most"]] * s["w"][:, j] for j in range(W))
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["silu"]:
        y = y / (1 + torch.exp(-y))
    s["out"][rows[live]] = y[live].to(s["out"].dtype)
    last = new[:, None] + torch.arange(W - 1, device="cuda")
    s["state"][slots] = x.gather(1, last[:, :, None].expand(-1, -1, c["channels"]))
    return {"out": s["out"], "state": s["state"]}


def _delta(s):
    c = s["case"]
    if own:
        _device().gated_delta(s["q"], s["k"], s["v"], s["a"], s["b"], s["layer"], s["batch"], gate=s["z"], out=s["out"],
                              workspace=s["workspace"])
        return {"out": s["out"], "state": s["state"]}
    C = min(CHUNK, s["most"])
    N = -(-s["most"] // C)
    rows, live, begins, _ = _rows(s, N * C)
    slots, group, H = s["slots"].long(), c["v_heads"] // c["k_heads"], c["v_heads"]

    def chunks(x):  # tokens x heads (x dim) -> chunks x sequences x heads x C (x dim)
        x = torch.where(live[:, :, None, None], x.reshape(len(x), x.shape[1], -1)[rows].float(), 0.0)
        return x.view(-1, N, C, *x.shape[2:]).permute(1, 0, 3, 2, 4).contiguous()

    def unit(x):
        return chunks(x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)).repeat_interleave(group, 2)

    q, k, v = unit(s["q"].float()), unit(s["k"].float()), chunks(s["v"])
    x = s["a"] + s["dt_bias"]
    g = chunks(s["decay"] * (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))))[..., 0]
    beta = chunks(1 / (1 + torch.exp(-s["b"])))
    G = g.double().cumsum(-1)
    low = torch.ones(C, C, device="cuda").tril()
    fade = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(low == 0, 0).float()) * low
    kt = k.transpose(-1, -2).contiguous()
    A = (beta * torch.matmul(k, kt) * fade).tril(-1)
    P = torch.matmul(q, kt) * fade
    inv = torch.eye(C, device="cuda").expand(A.shape).clone()
    for i in range(1, C):  # (1 + A) inv = 1, a row at a time
        inv[..., i, :i] = -torch.matmul(A[..., i:i + 1, :i], inv[..., :i, :i].contiguous())[..., 0, :]
    eG, last = torch.exp(G.float())[..., None], G[..., -1:]
    rest = torch.exp((last - G).float())[..., None]
    S = torch.where(begins[:, None, None, None], 0.0, s["state"][slots])
    o = torch.empty_like(v)
    for n in range(N):  # a chunk after the other
        u = torch.matmul(inv[n], beta[n] * (v[n] - eG[n] * torch.matmul(k[n], S)))
        o[n] = eG[n] * torch.matmul(q[n], S) + torch.matmul(P[n], u)
        S = torch.exp(last[n].float())[..., None] * S + torch.matmul((k[n] * rest[n]).transpose(-1, -2).contiguous(), u)
    s["state"][slots] = S
    o = o.permute(1, 0, 3, 2, 4).reshape(-1, N * C, H, c["v_dim"])[live] * c["k_dim"] ** -0.5
    if s["z"] is not None:
        z = s["z"][rows[live]]
        o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm"] * z / (1 + torch.exp(-z))
    s["out"][rows[live]] = o.to(s["out"].dtype)
    return {"out": s["out"], "state": s["state"]}


def _sample(s):
    if own:
        _device().sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                         out=s["tokens"], logprobs=s["logprobs"], workspace=s["workspace"])
        return {"token": s["tokens"], "logprob": s["logprobs"]}
    l = s["logits"].double()
    t = s["temperature"].double()[:, None]
    most, best = l.max(1, keepdim=True)
    best = (l == most).int().argmax(1)
    w = torch.exp((l - most) / torch.where(t > 0, t, 1.0))
    if s["top_k"] is not None:
        order = torch.sort(l, dim=1, descending=True, stable=True)[1]
        v = w.gather(1, order)
        k = s["top_k"][:, None]
        v = torch.where((k <= 0) | (torch.arange(v.shape[1], device="cuda") < k), v, 0.0)
        upto, p = v.cumsum(1), s["top_p"].double()[:, None]
        keep = (p >= 1) | (upto - v < p * upto[:, -1:])
        keep &= v >= s["min_p"].double()[:, None]
        keep[:, 0] = True
        w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, v, 0.0))
    upto = w.cumsum(1)
    past = upto > s["u"].double()[:, None] * upto[:, -1:]
    token = torch.where(past.any(1), past.int().argmax(1), best)
    s["tokens"].copy_(torch.where(t[:, 0] > 0, token, best))
    chance = torch.log(w.gather(1, token[:, None]) / upto[:, -1:])[:, 0]
    s["logprobs"].copy_(torch.where(t[:, 0] > 0, chance, 0.0))
    return {"token": s["tokens"], "logprob": s["logprobs"]}


# ---- what a pass cannot do without ------------------------------------------------
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["type"] == "f32" else 2) + 24 * case["rows"], "flops": 2 * n}
    new, lens = _lengths(case)
    n, goes_on = sum(new), sum(a != b for a, b in zip(new, lens))
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "conv":
        C, W = case["channels"], case["width"]
        kept = (W - 1) * C * 4
        return {"bytes": n * C * (size + (4 if case["act"] == "f32" else 2)) + (goes_on + len(new)) * kept + W * C * 4,
                "flops": 2 * n * C * W}
    K, H, dk, dv = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"]
    row = (2 * K * dk + H * dv) * size + H * dv * (4 if case["out"] == "f32" else 2) + 8 * H + (4 * H * dv if case["gate"] else 0)
    return {"bytes": n * row + (goes_on + len(new)) * H * dk * dv * 4, "flops": 6 * n * H * dk * dv}


# ---- from the definitions, in 64 bits -----------------------------------------------
def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"conv": _exact_conv, "delta": _exact_delta, "sample": _exact_sample}[case["kind"]](s)


def _exact_conv(s):
    c = s["case"]
    new, lens = _lengths(c)
    out, state = s["out"].double(), s["state"].double()
    w, row = s["w"].double(), 0
    for n, m, slot in zip(new, lens, s["slots"].tolist()):
        x = torch.cat((torch.zeros_like(state[slot]) if n == m else state[slot], s["x"][row:row + n].double()))
        y = torch.einsum("tcj,cj->tc", x.unfold(0, c["width"], 1), w)
        if s["bias"] is not None:
            y += s["bias"].double()
        out[row:row + n] = y * torch.sigmoid(y) if c["silu"] else y
        state[slot] = x[n:]
        row += n
    return {"out": out, "state": state}


def _exact_delta(s):
    """A token after the other, each of them in all sequences that have it."""
    c = s["case"]
    new, lens = _lengths(c)
    group, D = c["v_heads"] // c["k_heads"], torch.float64
    q, k = (x.to(D) for x in (s["q"], s["k"]))
    q, k = (x * ((x ** 2).sum(-1, keepdim=True) + EPS) ** -0.5 for x in (q, k))
    q, k = (x[:, torch.arange(c["v_heads"], device="cuda") // group] for x in (q, k))
    v, beta = s["v"].to(D), torch.sigmoid(s["b"].to(D))
    alpha = torch.exp(s["decay"].to(D) * torch.nn.functional.softplus(s["a"].to(D) + s["dt_bias"].to(D), threshold=1000))
    state, out = s["state"].to(D), s["out"].to(D)
    order = sorted(range(len(new)), key=lambda i: -new[i])
    starts = s["starts"].tolist()
    first = torch.tensor([starts[i] for i in order], device="cuda")
    slots = s["slots"].long()[order]
    S = state[slots]
    S[torch.tensor([new[i] == lens[i] for i in order], device="cuda")] = 0
    has = [sum(n > t for n in new) for t in range(max(new))]  # the longest come first
    for t in range(max(new)):
        at = first[:has[t]] + t
        M = S[:has[t]]
        M *= alpha[at][..., None, None]
        kk = k[at][..., None]
        M += kk * (beta[at][..., None] * (v[at] - (kk * M).sum(2)))[..., None, :]
        out[at] = (q[at][..., None] * M).sum(2) / math.sqrt(c["k_dim"])
    state[slots] = S
    if c["gate"]:
        z, o = s["z"][:s["live"]].to(D), out[:s["live"]]
        out[:s["live"]] = o * ((o ** 2).mean(-1, keepdim=True) + EPS) ** -0.5 * s["norm"].to(D) * z * torch.sigmoid(z)
    return {"out": out, "state": state}


def _exact_sample(s):
    t, k, p, m = _settings(s["case"])
    f = np.float32
    out, share = [], []
    for i, (l, u) in enumerate(zip(s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy())):
        if t[i] <= 0:
            out.append(int(np.argmax(l)))
            share.append(0.0)
            continue
        order = np.lexsort((np.arange(len(l)), -l))
        w = np.exp((l[order] - l[order[0]]) / np.float64(f(t[i])))
        n = len(l) if k is None or k[i] <= 0 else min(k[i], len(l))
        if p is not None and p[i] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w[:n])[:-1], np.float64(f(p[i])) * w[:n].sum()))
        if m is not None:
            n = max(1, min(n, int((w >= np.float64(f(m[i]))).sum())))
        kept = np.sort(order[:n])
        upto = np.cumsum(np.exp((l[kept] - l[order[0]]) / np.float64(f(t[i]))))
        out.append(int(kept[min(np.searchsorted(upto, u * upto[-1], side="right"), n - 1)]))
        share.append(float((l[out[-1]] - l[order[0]]) / np.float64(f(t[i])) - np.log(upto[-1])))
    return {"token": torch.tensor(out, dtype=torch.int32), "logprob": torch.tensor(share, dtype=torch.float64)}
