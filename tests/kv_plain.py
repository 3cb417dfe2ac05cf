"""Plain forms, in 64 bits on the CPU, of the paged-cache operators: the oracle
of the tests, and how far a kernel may be from it."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def gathered(pool, pages, n, head):
    """The first n tokens of one head: n x dim, in 64 bits."""
    page = pool.shape[2]
    ids = torch.tensor([pages[j // page] for j in range(n)], dtype=torch.long)
    at = torch.tensor([j % page for j in range(n)], dtype=torch.long)
    return pool[ids, head, at].double()


def attention(q, k, v, starts, lens, table, scale, cap=0.0, window=0, prefix=None, slopes=None, fill=None):
    """(out, allowed error) of every row; rows of no sequence hold `fill`'s.  All on the CPU.

    The error allowed: a score is a sum of dim products, each rounded to 32 bits
    (2^-23 a step, as the matrix cores may cut), of operands split into parts that
    leave 2^-22 at most; the cap and the bias add a few steps of their size.  An
    error e of every score changes a softmax average by 2 e max |v| at most; the
    sums over n keys add n steps.  Where the weights are rounded to 16 bits, each
    is off by half a step, and so is the output."""
    T, H, D = q.shape
    G = H // k.shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64) if fill is None else fill.double().clone()
    tol = torch.zeros(T, H, D, dtype=torch.float64)
    u = HALF_STEP[q.dtype]
    f32 = 2.0 ** -23
    for s in range(len(lens)):
        n, m = starts[s + 1] - starts[s], lens[s]
        pre = prefix[s] if prefix is not None else 0
        for h in range(H):
            kk, vv = gathered(k, table[s], m, h // G), gathered(v, table[s], m, h // G)
            for i in range(n):
                t, p = starts[s] + i, m - n + i
                see = [j for j in range(m) if (j <= p or j < pre) and (window == 0 or p - j < window)]
                if not see:
                    out[t, h] = 0
                    continue
                x = q[t, h].double()
                a = kk[see]
                z = a @ x * scale
                size = float((a.abs() @ x.abs()).max()) * abs(scale)
                e = (D + 8) * f32 * size + 2.0 ** -22 * size
                if cap:
                    z = cap * torch.tanh(z / cap)
                    e += 8 * f32 * cap
                if slopes is not None:
                    far = torch.tensor([abs(p - j) for j in see], dtype=torch.float64)
                    z = z - float(slopes[h]) * far
                    e += 4 * f32 * float(slopes[h]) * float(far.max())
                e += 8 * f32 * float(z.abs().max() + 1)
                w = torch.softmax(z, 0)
                out[t, h] = w @ vv[see]
                most = float(vv[see].abs().max())
                tol[t, h] = (2 * e + (len(see) + 16) * f32) * most
                if q.dtype != torch.float32:
                    tol[t, h] += u * (w @ vv[see].abs()) * 1.01 + u * out[t, h].abs() + 2.0 ** -24
    return out, tol


def rope(x, pos, turns, rot, layout, mscale, w=None, eps=1e-6):
    """One head in 64 bits and the error a 32-bit result may have: the norm sums
    dim squares (2^-24 a step), sine and cosine are off by a few steps, and a
    pair's values mix."""
    x = x.double()
    D = x.numel()
    e = torch.zeros(D, dtype=torch.float64)
    if w is not None:
        x = x / math.sqrt(float((x * x).sum()) / D + eps) * w.double()
        e += (D + 8) * 2.0 ** -24 * x.abs()
    y = x.clone()
    for i in range(rot // 2):
        a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
        t = 2 * math.pi * math.fmod(pos * float(turns[i]), 1.0)
        y[a] = mscale * (x[a] * math.cos(t) - x[b] * math.sin(t))
        y[b] = mscale * (x[a] * math.sin(t) + x[b] * math.cos(t))
        size = mscale * math.hypot(float(x[a]), float(x[b]))
        both = mscale * float(e[a] + e[b]) + 12 * 2.0 ** -24 * size
        e[a] = e[b] = both
    return y, e


def fork(table, lens, parents, refs, page, room):
    """(table, lens, refs, copies, whether pages ran out), lists of ints."""
    width, refs = len(table[0]) if table else 0, list(refs)
    rows, missing, seen = [], [], set()
    for p in parents:
        row = list(table[p]) if p >= 0 else [-1] * width
        n = lens[p] if p >= 0 else 0
        if p in seen:
            row = [x if j < n // page else -1 for j, x in enumerate(row)]
        seen.add(p)
        rows.append(row)
        need = min(width, -(-(n + room) // page))
        missing.append([j for j in range(need) if row[j] < 0])
    for r in table:
        for x in r:
            if x >= 0:
                refs[x] -= 1
    for r in rows:
        for x in r:
            if x >= 0:
                refs[x] += 1
    free = [p for p, n in enumerate(refs) if n == 0][::-1]
    copies, full = [], False
    for c, p in enumerate(parents):
        n = lens[p] if p >= 0 else 0
        pair = [-1, -1]
        for j in missing[c]:
            if not free:
                full = True
                continue
            rows[c][j] = free.pop()
            refs[rows[c][j]] = 1
            if p >= 0 and p in parents[:c] and n % page and j == n // page and table[p][j] >= 0:
                pair = [table[p][j], rows[c][j]]
        copies.append(pair)
    return rows, [lens[p] if p >= 0 else 0 for p in parents], refs, copies, full


def compact(table, refs):
    """(table, refs, moves), lists of ints."""
    refs, used = list(refs), sum(r > 0 for r in refs)
    to = dict(zip([p for p in range(used, len(refs)) if refs[p] > 0], [p for p in range(used) if refs[p] <= 0]))
    for a, b in to.items():
        refs[b], refs[a] = refs[a], 0
    return [[to.get(x, x) for x in r] for r in table], refs, [list(x) for x in to.items()]
