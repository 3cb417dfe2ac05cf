"""Every variant of the paged attention's launches (kv_variants.py, whose plans the
CPU tests check) against the plain form in 64 bits: two halves of a workgroup,
tiles in one part and in many, windows over several parts, with every sort of
mask, missing pages, rows that see nothing and values that must stay hidden."""
import pytest

import kv_dense
import kv_variants
from test_gpu_kv_attn import BF16, F16, F32, TYPES, ints

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def params(variants):
    return [pytest.param(v, d, id=f"{v.ids()}-{d}") for v in variants for d in v.dims]


def batch_of(v, dim, act, kv, seed=0):
    print("[case]", v.ids(), v.new, v.lens, dim, act, kv, flush=True)
    return kv_dense.make(seed + dim, v.new, v.lens, v.heads, v.kv_heads, dim, act, kv, width=v.width, pad=2, device="cuda")


def run(case, scale=None, prefix=None, slopes=None, cap=0.0, window=0):
    from inferno_hip import device as D
    q, k, v, starts, lens, table = case
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    D.attn_paged(q, D.KVCache(k, v), D.KVBatch(ints(starts), ints(lens), ints(table), q.shape[0]), scale=scale, softcap=cap,
                 window=window, prefix_lens=ints(prefix) if prefix else None,
                 slopes=torch.tensor(slopes, device="cuda") if slopes else None, out=out, flags=flags)
    return out, int(flags.item())


def check(case, want_flags=0, **kw):
    got, flags = run(case, **kw)
    want, tol, spread = kv_dense.attention(*case, **kw)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (kw, float((err - tol).max()), float(err.max()))
    assert flags == want_flags
    return got, want, spread


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("v,dim", params(kv_variants.ALL))
def test_plain(act, kv, v, dim):
    got, want, spread = check(batch_of(v, dim, act, kv), window=v.window)
    if act == F32:
        live = sum(v.new)
        bound = kv_dense.l2_bound(dim, max(v.lens), 2 if kv == F16 else 3, spread)
        assert kv_dense.l2(got[:live], want[:live]) <= bound


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("v,dim", params(kv_variants.HALVES + kv_variants.WHOLE + kv_variants.PARTS + kv_variants.FEW))
def test_biases_caps_windows_and_prefixes(act, kv, v, dim):
    case = batch_of(v, dim, act, kv, 1)
    slopes = [2.0 ** -(1 + i % 9) for i in range(v.heads)]
    most = max(v.lens)
    prefix = [most // 3 if i % 2 else most + 9 for i in range(len(v.lens))]
    check(case, slopes=slopes)
    check(case, cap=3.0)
    check(case, prefix=prefix)
    check(case, cap=20.0, slopes=slopes, prefix=prefix, window=70)
    check(case, window=33)  # (hides whole steps of half a workgroup from the other half's rows)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("v,dim", params(kv_variants.HALVES + kv_variants.WHOLE[:2] + kv_variants.PARTS[::2] + kv_variants.FEW[1:3]))
def test_missing_pages_and_rows_before_the_first_token(act, kv, v, dim):
    q, k, w, starts, lens, table = batch_of(v, dim, act, kv, 2)
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = [list(row) for row in table]
        # the first page, one in a first half's keys and one in a second's, the last
        for row, m in zip(t, lens):
            for p in {0, 3, 5, 9, (m - 1) // 16}:
                if 0 <= p < -(-m // 16):
                    row[p] = bad
        check((q, k, w, starts, lens, t), want_flags=8)
    short = [min(m, n // 2) for n, m in zip(v.new, lens)]
    check((q, k, w, starts, short, table), want_flags=16 if any(n > m for n, m in zip(v.new, short)) else 0)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("v,dim", params(kv_variants.HALVES + kv_variants.WHOLE[:2] + kv_variants.PARTS + kv_variants.WINDOWS))
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_hidden_values_have_no_influence(act, kv, v, dim, bad):
    """The last key of the first sequence is seen by its last row alone, the first key of a window by the first row."""
    case = batch_of(v, dim, act, kv, 3)
    k, w, table = case[1], case[2], case[5][0]
    n, m = v.new[0], v.lens[0]
    for window in (v.window or 0, 40):
        clean, flags = run(case, window=window)
        assert flags == 0 and bool(torch.isfinite(clean.float()).all())
        marks = [m - 1] + ([m - n - window + 1] if 0 < window <= m - n + 1 else [])
        spoilt = w.clone(), k.clone()
        for j in marks:
            spoilt[0][table[j // 16], :, j % 16, 5] = bad
        got, _ = run((case[0], k, spoilt[0], *case[3:]), window=window)
        first = 1 if len(marks) > 1 else 0
        assert torch.equal(got[first:n - 1], clean[first:n - 1]) and torch.equal(got[n:], clean[n:])
        for row in [n - 1] + [0] * first:
            x = got[row].float()
            assert bool((torch.isnan(x[:, 5]) if bad != bad else x[:, 5] == bad).all())
            assert bool(torch.isfinite(torch.cat((x[:, :5], x[:, 6:]), 1)).all())
        for j in marks:
            spoilt[1][table[j // 16], :, j % 16, ::3] = float("nan")
        got, _ = run((case[0], spoilt[1], spoilt[0], *case[3:]), window=window)
        assert torch.equal(got[first:n - 1], clean[first:n - 1]) and torch.equal(got[n:], clean[n:])
        assert not bool(torch.isfinite(got[n - 1].float()).all())


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("v,dim", params(kv_variants.HALVES + kv_variants.WHOLE[:2] + kv_variants.PARTS[2:] + kv_variants.FEW[1:3]))
def test_equal_keys_of_large_scores(act, kv, v, dim):
    """Every third key, far above the others by more than any weight shows, has an equal share."""
    q, k, w, starts, lens, table = batch_of(v, dim, act, kv, 4)
    q.zero_()
    q[..., 0] = 2.0 ** 15
    for row, m in zip(table, lens):
        for j in range(m):
            k[row[j // 16], :, j % 16] = 0.0
            k[row[j // 16], :, j % 16, 0] = 0.0 if j % 3 else 120.0
    for scale in (16.0, 2.0 ** 70):
        got, flags = run((q, k, w, starts, lens, table), scale=scale)
        want, _, _ = kv_dense.attention(q, k, w, starts, lens, table, scale=scale)
        most = float(torch.nan_to_num(w.float()).abs().max())
        limit = most * (max(lens) + 64) * 2.0 ** -24 + (2 * most * {F16: 2.0 ** -11, BF16: 2.0 ** -8}[act] if act != F32 else 0.0)
        assert flags == 0 and float((got.double() - want).abs().max()) <= limit
