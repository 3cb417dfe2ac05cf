"""fp32 rows keep fp32's accuracy: their L2 distance to the 64-bit form, at every
width, in both kernels.  On the CPU: the bound lies above a plain evaluation in 32
bits and below kernels that would drop parts of q or of the weights."""
import math

import pytest

import kv_dense
import kv_plain

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
WIDTHS = [8, 64, 80, 96, 128, 192, 256]
# (new tokens, tokens, table entries): one token, a few, a chunk in tables too wide for the kernel of few rows
SHAPES = [([1, 1, 1], [700, 300, 40], 0), ([5, 2], [300, 64], 0), ([60, 40], [360, 200], 64)]


def cut(x, kind, parts):
    """x rounded to the sum of `parts` values of `kind`; fp16 rows are scaled to [2^14, 2^15) first."""
    up = torch.ones_like(x[..., :1])
    if kind == F16:
        up = 2.0 ** (15 - torch.frexp(x.abs().amax(-1, keepdim=True))[1].double()).clamp(max=2.0 ** 60)
    rest, y = x * up, 0.0
    for _ in range(parts):
        part = rest.to(kind).to(x.dtype)
        y, rest = y + part, rest - part
    return y / up


def emulated(case, q_parts, p_parts):
    """attention's rows where q and the weights are cut to parts of the cache's type and nothing else is rounded."""
    q, k, v, starts, lens, table = case
    G, kind = q.shape[1] // k.shape[1], k.dtype
    out = torch.zeros(q.shape, dtype=torch.float64)
    for s, m in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        see, ids = kv_dense.seen_keys(b - a, m, 0, 0, table[s], k.shape[0], 16, q.device)
        for h in range(q.shape[1]):
            kk, vv = (x[ids, h // G, torch.arange(m) % 16].double() for x in (k, v))
            z = (cut(q[a:b, h].double(), kind, q_parts) @ kk.T) * q.shape[2] ** -0.5
            p = torch.exp((z - z.masked_fill(~see, -math.inf).amax(1, keepdim=True))).masked_fill(~see, 0.0)
            up = 2.0 ** (14 if kind == F16 else 0)
            rest, w = p * up, 0.0
            for _ in range(p_parts):
                part = rest.to(kind).double()
                w, rest = w + part, rest - part
            out[a:b, h] = (w / up) @ vv / p.sum(1, keepdim=True)
    return out


@pytest.mark.parametrize("kv,parts", [(F16, 2), (BF16, 3)])
@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("new,lens,width", SHAPES)
def test_the_bound_sees_a_part_that_is_dropped(kv, parts, dim, new, lens, width):
    case = kv_dense.make(60 + dim, new, lens, 4, 2, dim, F32, kv, width=width)
    want, _, spread = kv_dense.attention(*case)
    bound = kv_dense.l2_bound(dim, max(lens), parts, spread)
    assert kv_dense.l2(emulated(case, parts, parts), want) < bound / 4
    for q_parts, p_parts in ((1, parts), (parts, 1), (1, 1)) + (((2, 2),) if parts == 3 else ()):
        assert kv_dense.l2(emulated(case, q_parts, p_parts), want) > bound, (q_parts, p_parts)
    # a plain evaluation in 32 bits keeps it
    q, k, v, starts, lens, table = case
    plain = torch.zeros(q.shape)
    for s, m in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        see, ids = kv_dense.seen_keys(b - a, m, 0, 0, table[s], k.shape[0], 16, q.device)
        for h in range(q.shape[1]):
            kk, vv = (x[ids, h // 2, torch.arange(m) % 16].float() for x in (k, v))
            z = (q[a:b, h] @ kk.T * dim ** -0.5).masked_fill(~see, -math.inf)
            p = torch.exp(z - z.amax(1, keepdim=True))
            plain[a:b, h] = p @ vv / p.sum(1, keepdim=True)
    assert kv_dense.l2(plain, want) < bound


@pytest.mark.parametrize("act,kv", [(F32, F16), (F16, F16), (BF16, BF16)])
def test_both_plain_forms_are_one(act, kv):
    """kv_dense's against kv_plain's, masks and all."""
    slopes = [0.5, 0.25, 0.125, 0.0625]
    for seed, (new, lens, kw) in enumerate([([1, 6, 0, 9], [40, 30, 3, 4], {}), ([5, 20], [33, 20], dict(window=7)),
                                            ([5, 20], [33, 20], dict(prefix=[9, 30], cap=3.0)), ([7], [50], dict(slopes=slopes, scale=0.3))]):
        q, k, v, starts, lens, table = kv_dense.make(seed, new, lens, 4, 2, 24, act, kv, pad=2)
        got, tol, _ = kv_dense.attention(q, k, v, starts, lens, table, **kw)
        kw.setdefault("scale", 24 ** -0.5)
        want, tol2 = kv_plain.attention(q, k, v, starts, lens, table, **kw, fill=torch.full(q.shape, 7.0))
        assert float((got - want).abs().max()) < 1e-12
        assert torch.allclose(tol, tol2, rtol=1e-9, atol=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("kv,parts", [(F16, 2), (BF16, 3)])
@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("new,lens,width", SHAPES + [([1], [9000], 0), ([40], [3000], 0)])
def test_fp32_rows(kv, parts, dim, new, lens, width):
    from test_gpu_kv_attn import run
    print("[case]", kv, dim, new, lens, flush=True)
    case = kv_dense.make(70 + dim, new, lens, 4, 2, dim, F32, kv, width=width, device="cuda")
    slopes = [0.02, 0.01, 0.005, 0.0025]
    for kw in ({}, dict(softcap=4.0), dict(slopes=slopes), dict(window=100)):
        got, flags = run(tuple(case), **dict(kw))
        want, _, spread = kv_dense.attention(*case, cap=kw.get("softcap", 0.0), slopes=kw.get("slopes"), window=kw.get("window", 0))
        assert flags == 0
        # (a cap's tanh and a bias add a few steps of their size)
        extra = 2.0 ** -23 * (8 * 4.0 if "softcap" in kw else 4 * 0.02 * max(lens) if "slopes" in kw else 0.0)
        error = kv_dense.l2(got, want.cpu())
        assert error <= kv_dense.l2_bound(dim, max(lens), parts, spread) + extra, (kw, error)
