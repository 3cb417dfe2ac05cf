"""The plain form in 64 bits of attention over the paged cache for batches of many
heads and keys: kv_plain.attention's definition and error terms, a sequence and
head at a time, on the tensors' own device.  And how far fp32 rows may be from it
on average, which is far closer than the worst case."""
import math

import torch

import kv_plain


def make(seed, new, lens, heads, kv_heads, dim, act, kv, page=16, width=0, pad=0, device="cpu", before=0):
    """(q, k, v, starts, lens, table): pools whose unfilled slots are NaN, tables of
    `width` entries at least, `before` and `pad` rows of no sequence."""
    g = torch.Generator(device=device).manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + 2
    order = torch.randperm(pages, generator=g, device=device).tolist()
    table, i = [], 0
    for n in counts:
        table.append(order[i:i + n] + [-1] * (max(counts + [1, width]) - n))
        i += n
    k, v = (torch.randn(pages, kv_heads, page, dim, generator=g, device=device).to(kv) for _ in range(2))
    empty = torch.ones(pages, page, dtype=torch.bool, device=device)
    for row, n in zip(table, lens):
        for j, p in enumerate(row[:-(-n // page)]):
            empty[p, :n - j * page] = False
    k.masked_fill_(empty[:, None, :, None], float("nan"))
    v.masked_fill_(empty[:, None, :, None], float("nan"))
    starts = [before]
    for n in new:
        starts.append(starts[-1] + n)
    q = (1.5 * torch.randn(starts[-1] + pad, heads, dim, generator=g, device=device)).to(act)
    return q, k, v, starts, lens, table


def seen_keys(n, m, window, prefix, row, pages, page, device):
    """n x m: whether row i (at position m - n + i) sees key j, whose page is there."""
    p = torch.arange(m - n, m, device=device)[:, None]
    j = torch.arange(m, device=device)
    see = (j <= p) | (j < prefix)
    if window:
        see &= p - j < window
    ids = torch.tensor([row[x // page] for x in range(m)], dtype=torch.long, device=device)
    return see & (ids >= 0) & (ids < pages), ids.clamp(0, pages - 1)


def attention(q, k, v, starts, lens, table, scale=None, cap=0.0, window=0, prefix=None, slopes=None, fill=7.0):
    """(out, allowed error, rms of the scores): rows of no sequence hold `fill`."""
    T, H, D = q.shape
    G, page, dev = H // k.shape[1], k.shape[2], q.device
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, H, D), fill, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(out)
    f32, u = 2.0 ** -23, kv_plain.HALF_STEP[q.dtype]
    squares = count = 0
    for s, m in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        n = b - a
        if n == 0:
            continue
        if m == 0:
            out[a:b] = 0
            continue
        see, ids = seen_keys(n, m, window, prefix[s] if prefix else 0, table[s], k.shape[0], page, dev)
        any_key = see.any(1)
        far = (torch.arange(m - n, m, device=dev)[:, None] - torch.arange(m, device=dev)).abs().double()
        used = see.any(0)
        slot = torch.arange(m, device=dev) % page
        for h in range(H):
            kk, vv = (torch.where(used[:, None], x[ids, h // G, slot].double(), 0.0) for x in (k, v))
            x = q[a:b, h].double()
            z = x @ kk.T.contiguous() * scale
            size = (x.abs() @ kk.abs().T.contiguous()).masked_fill(~see, 0.0).amax(1) * abs(scale)
            e = (D + 8) * f32 * size + 2.0 ** -22 * size
            if cap:
                z = cap * torch.tanh(z / cap)
                e = e + 8 * f32 * cap
            if slopes is not None:
                z = z - float(slopes[h]) * far
                e = e + 4 * f32 * float(slopes[h]) * far.masked_fill(~see, 0.0).amax(1)
            z = z.masked_fill(~see, -math.inf)
            shown = z.masked_fill(~see, 0.0)
            squares, count = squares + float(shown.pow(2).sum()), count + int(see.sum())
            e = e + 8 * f32 * (shown.abs().amax(1) + 1)
            w = torch.softmax(z.masked_fill(~any_key[:, None], 0.0), 1) * any_key[:, None]
            y = w @ vv
            out[a:b, h] = y
            most = torch.where(see, vv.abs().amax(1), 0.0).amax(1)
            t = ((2 * e + (see.sum(1) + 16) * f32) * most)[:, None].expand(n, D)
            if q.dtype != torch.float32:
                t = t + u * (w @ vv.abs()) * 1.01 + u * y.abs() + 2.0 ** -24
            tol[a:b, h] = t * any_key[:, None]
    return out, tol, math.sqrt(squares / max(count, 1))


def l2_bound(dim, keys, parts, spread):
    """How far fp32 rows may be from the 64-bit form in L2, relative to it.

    Rounding errors are independent, so that they add as their squares do, and one of
    up to e has 1/sqrt(3) of it in root mean square; a running sum has half of its
    last square on average.  A weight that is off by e moves the average of values of
    random signs by e of itself.  A score (rms `spread`): q's parts leave up to 2^-22 of
    a product (two of fp16; 2^-24 three of bf16), and each of the dim * parts / 16
    products of a sum is cut by up to 2^-23.  A weight: 2^-23 of its distance to the
    maximum (3 rms of the scores), 2^-23 of the exponential, and what its parts leave.
    The sums over the keys: keys * parts / 16 products cut by up to 2^-23, and `keys`
    additions rounded by 2^-24.  The sorts of error are simply added."""
    left = 2.0 if parts == 2 else 0.5
    score = spread * (left + math.sqrt(dim * parts / 16 / 2))
    sums = math.sqrt(keys * parts / 16 / 2) + math.sqrt(keys / 2) / 2
    return 2.0 ** -23 / math.sqrt(3) * (score + 3 * spread + 1 + left + sums)


def l2(got, want):
    return float((got.double() - want).norm() / want.norm())
