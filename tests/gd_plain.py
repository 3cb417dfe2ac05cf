"""Plain forms, in 64 bits on the CPU, of the short convolution, the gated delta rule
and the choice of a token: the oracle of the tests, and how far a kernel may be from it."""
import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a subnormal step


def conv(x, w, bias, silu, state, new, begins, slots, starts, out):
    """(out, state, allowed error): rows and slots of no sequence as they were.  A sum of
    `width` products and a bias is off by a step of 2^-24 for each of them of what is
    summed; silu changes an error by less than 1.1, and its exponential, sum and
    quotient are a few steps off; then the result is rounded once."""
    W = w.shape[1]
    y, held = out.double().clone(), state.double().clone()
    tol = torch.zeros_like(y)
    u = HALF_STEP[out.dtype]
    for n, begin, slot, at in zip(new, begins, slots, starts):
        if n == 0 or slot < 0:
            continue
        old = torch.zeros(W - 1, x.shape[1], dtype=torch.float64) if begin else held[slot]
        rows = torch.cat((old, x[at:at + n].double()))
        for t in range(n):
            terms = rows[t:t + W] * w.double().t()
            v, size = terms.sum(0), terms.abs().sum(0)
            if bias is not None:
                v, size = v + bias.double(), size + bias.double().abs()
            e = (W + 2) * 2.0 ** -24 * size
            if silu:
                v, e = v / (1 + torch.exp(-v)), 1.1 * e + 8 * 2.0 ** -24 * (v / (1 + torch.exp(-v))).abs()
            y[at + t] = v
            tol[at + t] = e + u * (v.abs() + e) + LEAST[out.dtype]
        held[slot] = rows[n:]
    return y, held, tol


def delta(q, k, v, a, b, decay, dt_bias, state, new, begins, slots, starts, out, scale=None, norm_w=None, gate=None,
          eps=1e-6, l2_eps=1e-6):
    """(out, state) of the definition, a token after the other."""
    H, dk = v.shape[1], q.shape[2]
    group = H // q.shape[1]
    scale = dk ** -0.5 if scale is None else scale
    q, k = (x.double() / (x.double().pow(2).sum(-1, keepdim=True) + l2_eps).sqrt() for x in (q, k))
    q, k = (x.repeat_interleave(group, 1) for x in (q, k))
    g = decay.double() * torch.nn.functional.softplus(a.double() + dt_bias.double(), threshold=600)  # (e^-600 is nothing beside 600)
    alpha, beta = torch.exp(g.clamp(max=0)), torch.sigmoid(b.double())
    y, held = out.double().clone(), state.double().clone()
    for n, begin, slot, at in zip(new, begins, slots, starts):
        if n == 0 or slot < 0:
            continue
        S = torch.zeros_like(held[slot]) if begin else held[slot].clone()
        for t in range(at, at + n):
            S = alpha[t][:, None, None] * S
            d = beta[t][:, None] * (v[t].double() - (k[t][..., None] * S).sum(1))
            S = S + k[t][..., None] * d[:, None]
            o = scale * (q[t][..., None] * S).sum(1)
            if norm_w is not None:
                o = o / (o.pow(2).mean(-1, keepdim=True) + eps).sqrt() * norm_w.double()
            if gate is not None:
                z = gate[t].double()
                o = o * z / (1 + torch.exp(-z))
            y[t] = o
        held[slot] = S
    return y, held


def off(got, want):
    """2-norm of the difference over the norm, of all of it."""
    got, want = got.double().cpu(), want.double()
    size = float(want.norm())
    return float((got - want).norm()) / size if size else float(got.norm())


# Of the delta rule.  A product of operands in two fp16 parts leaves 2^-22 of its terms
# at most, an fp32 sum of 128 terms 2^-24 a term, and neither with one sign; from the
# inputs to an output follow four such products (the norms of k, K S, T X or M X, Q S),
# and a state forgets old errors with what they came from.  2^-20 of a result's norm
# holds them with room; a part or a tile that is left out changes it by 2^-11 at least.
NEAR = 2.0 ** -20


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """(token, logprob, flags) of one row, a vector of 64-bit values."""
    l = np.asarray(logits, dtype=np.float64)
    if np.isnan(l).any() or (l == np.inf).any():
        return 0, float("nan"), (1 if np.isnan(l).any() else 0) | (2 if (l == np.inf).any() else 0)
    if not np.isfinite(l).any():
        return 0, 0.0, 4
    t = 1.0 if temperature is None else temperature
    if not t > 0:
        return int(np.argmax(l)), 0.0, 0
    order = np.lexsort((np.arange(len(l)), -l))
    with np.errstate(invalid="ignore"):
        x = (l[order] - l[order[0]]) / t
    w = np.where(np.isinf(l[order]), 0.0, np.exp(np.where(np.isnan(x), 0.0, x)))
    n = len(l)
    if top_k is not None and 0 < top_k < n:
        n = top_k
    if top_p is not None and top_p < 1:
        want = max(top_p, 0.0) * w[:n].sum()
        n = 1 + int(np.searchsorted(np.cumsum(w[:n])[:-1], want))
    kept = np.zeros(len(l))
    kept[order[:n]] = w[:n]
    if min_p is not None and min_p > 0:
        kept[kept < min_p] = 0.0
        kept[order[0]] = 1.0
    upto = np.cumsum(kept)
    u = min(max(u, 0.0), 2.0) if u == u else 0.0
    past = (upto > (u if u < 1 else 2.0) * upto[-1]) & (kept > 0)
    token = int(np.argmax(past)) if past.any() else int(np.nonzero(kept)[0][-1])
    return token, float(np.log(kept[token] / upto[-1])), 0
