"""Attention of many rows a sequence over the paged cache, against the plain form
in 64 bits: tables wide enough that no short cache takes the kernel of few rows."""
import pytest

import kv_plain
from test_gpu_kv_attn import BF16, F16, F32, TYPES, build, check, ints, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

WIDTHS = [64, 80, 128, 200, 256]


def wide(case, tokens=1024):
    """The same batch with tables that hold more tokens than any of its sequences."""
    q, k, v, starts, lens, table = case
    n = tokens // k.shape[2]
    return q, k, v, starts, lens, [row + [-1] * (n - len(row)) for row in table]


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_every_head_width_plain_biased_and_capped(act, kv, dim):
    case = wide(build(dim, [50, 0, 3], [120, 7, 90], 4, 1, dim, 16, act, kv, pad=2))
    slopes = [0.5, 0.25, 0.125, 0.0625]
    check(case)
    check(case, slopes=slopes)
    check(case, softcap=2.0)
    check(case, softcap=20.0, slopes=slopes, prefix_lens=[90, 0, 300])


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_keys_split_and_joined(act, kv, dim):
    check(wide(build(dim, [40], [700], 4, 1, dim, 32, act, kv)))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim,window", [(64, 1), (64, 40), (128, 17), (128, 100), (256, 60)])
def test_windows_of_unsplit_tiles(act, kv, dim, window):
    check(wide(build(window, [60], [210], 4, 2, dim, 16, act, kv)), window=window)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("n", [33, 63, 64, 65, 127, 128, 129])
def test_lengths_about_the_tiles(act, kv, n):
    check(wide(build(n, [n], [n], 1, 1, 64, 16, act, kv)))
    check(wide(build(n, [n], [n + 63], 1, 1, 128, 64, act, kv)), window=n)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_rows_that_see_nothing_are_zero(act, kv, dim):
    case = wide(build(9, [40], [4], 4, 2, dim, 16, act, kv))
    check(case, want_flags=16)
    check(case, prefix_lens=[2], want_flags=16)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_hidden_keys_have_no_influence_whatever_they_hold(act, kv, dim, bad):
    for n, m, window in ((70, 90, 0), (64, 200, 40)):
        q, k, v, starts, lens, table = wide(build(10, [n], [m], 4, 1, dim, 16, act, kv))
        clean, _ = run((q, k, v, starts, lens, table), window=window)
        assert bool(torch.isfinite(clean.float()).all())
        # the last token is seen by its own row alone; with a window the first row sees what the next do not
        marks = [m - 1] + ([m - n - window + 1] if window else [])
        for j in marks:
            v[table[0][j // 16], :, j % 16, 5] = bad
        got, _ = run((q, k, v, starts, lens, table), window=window)
        some = 1 if window else 0
        assert torch.equal(got[some:n - 1], clean[some:n - 1])
        for row in [n - 1] + ([0] if window else []):
            seen = got[row].float()
            assert bool((torch.isnan(seen[:, 5]) if bad != bad else seen[:, 5] == bad).all())
            assert bool(torch.isfinite(torch.cat((seen[:, :5], seen[:, 6:]), 1)).all())
        for j in marks:
            k[table[0][j // 16], :, j % 16, ::3] = float("nan")
        got, _ = run((q, k, v, starts, lens, table), window=window)
        assert torch.equal(got[some:n - 1], clean[some:n - 1])
        assert not torch.isfinite(got[n - 1].float()).all()


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_page_ids_outside_the_pool_are_left_out_and_reported(act, kv, dim):
    q, k, v, starts, lens, table = wide(build(12, [40], [100], 4, 2, dim, 16, act, kv))
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = [list(table[0])]
        t[0][2] = bad
        got, flags = run((q, k, v, starts, lens, t))
        assert flags == 8 and bool(torch.isfinite(got.float()).all())
        # as if keys 32 .. 47 were not there, for the last row of head 0
        keep = [j for j in range(100) if not 32 <= j < 48]
        z = kv_plain.gathered(k, table[0], 100, 0)[keep] @ q[-1, 0].double() * dim ** -0.5
        want = torch.softmax(z, 0) @ kv_plain.gathered(v, table[0], 100, 0)[keep]
        # half a step of the weights and of the output, of values under 5; fp32: 100 steps of its sums
        limit = 2 * 5 * kv_plain.HALF_STEP[act] if act != F32 else 5 * 100 * 2.0 ** -23
        assert float((got[-1, 0].double() - want).abs().max()) < limit


def test_extreme_queries_keep_fp32_accuracy():
    for kv in (F16, BF16):
        q, k, v, starts, lens, table = wide(build(11, [40], [90], 4, 2, 128, 16, F32, kv))
        q[:20] *= 1e7
        q[20:] *= 1e-7
        check((q, k, v, starts, lens, table), scale=1e-6)
        check((q * 1e-25, k, v, starts, lens, table), slopes=[0.5, 0.25, 0.125, 0.0625])


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim,heads,tokens", [(64, 130, 150), (128, 260, 150), (256, 260, 150)])
def test_many_tiles_in_one_workgroup_each(act, kv, dim, heads, tokens):
    """260 and 520 tiles and heads, which are not split: halves of a workgroup share the keys of the former."""
    from inferno_hip import device as D
    g = torch.Generator(device="cuda").manual_seed(dim + heads)
    pages = 18
    k, v = (torch.randn(pages, heads, 16, dim, generator=g, device="cuda").to(kv) for _ in range(2))
    q = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(act)
    order = torch.randperm(pages, generator=g, device="cuda").int()
    length = 16 * pages - 5
    table = torch.full((1, 40), -1, dtype=torch.int32, device="cuda")
    table[0, :pages] = order
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = D.attn_paged(q, D.KVCache(k, v), D.KVBatch(ints([0, tokens]), ints([length]), table, tokens), flags=flags)
    # the plain form in 64 bits, head by head
    kk, vv = (x[order.long()].transpose(1, 2).reshape(16 * pages, heads, dim)[:length].double() for x in (k, v))
    at = torch.arange(length, device="cuda")
    hide = at[None, :] > (length - tokens + torch.arange(tokens, device="cuda"))[:, None]
    u, f32 = kv_plain.HALF_STEP[act], 2.0 ** -23
    for h in range(heads):
        z = (q[:, h].double() @ kk[:, h].T.contiguous() * dim ** -0.5).masked_fill(hide, -float("inf"))
        w = torch.softmax(z, 1)
        want = w @ vv[:, h]
        size = float((q[:, h].double().abs() @ kk[:, h].abs().T.contiguous()).max()) * dim ** -0.5
        # (the terms of kv_plain.attention)
        e = (dim + 8) * f32 * size + 2.0 ** -22 * size + 8 * f32 * (size + 1)
        tol = (2 * e + (length + 16) * f32) * float(vv[:, h].abs().max()) * torch.ones_like(want)
        if act != F32:
            tol += u * (w @ vv[:, h].abs()) * 1.01 + u * want.abs() + 2.0 ** -24
        assert bool(((got[:, h].double() - want).abs() <= tol).all()), h
    assert int(flags.item()) == 0
