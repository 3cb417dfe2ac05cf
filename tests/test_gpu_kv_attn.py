"""Attention over the paged cache against the plain form in 64 bits."""
import random

import pytest

import kv_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def build(seed, new, lens, heads, kv_heads, dim, page, act, kv, pad=0, spare=2, fill=float("nan")):
    """q, pools (what no token has filled holds `fill`), starts, lens, tables; on the CPU."""
    from inferno_hip import device as D  # noqa: F401
    g = torch.Generator().manual_seed(seed)
    rng = random.Random(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + spare
    order = rng.sample(range(pages), sum(counts))
    width = max(counts + [1])
    table, i = [], 0
    for n in counts:
        table.append(order[i:i + n] + [-1] * (width - n))
        i += n
    k = torch.full((pages, kv_heads, page, dim), fill).to(kv)
    v = k.clone()
    for s, n in enumerate(lens):
        for j in range(n):
            k[table[s][j // page], :, j % page] = torch.randn(kv_heads, dim, generator=g).to(kv)
            v[table[s][j // page], :, j % page] = torch.randn(kv_heads, dim, generator=g).to(kv)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = (1.5 * torch.randn(starts[-1] + pad, heads, dim, generator=g)).to(act)
    return q, k, v, starts, lens, table


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run(case, scale=None, **kw):
    from inferno_hip import device as D
    q, k, v, starts, lens, table = case
    cache = D.KVCache(k.cuda(), v.cuda())
    batch = D.KVBatch(ints(starts), ints(lens), ints(table), q.shape[0])
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    for name in ("prefix_lens", "slopes"):
        if kw.get(name) is not None:
            kw[name] = torch.tensor(kw[name], dtype=torch.int32 if name == "prefix_lens" else F32, device="cuda")
    D.attn_paged(q.cuda(), cache, batch, scale=scale, out=out, flags=flags, **kw)
    torch.cuda.synchronize()
    return out.cpu(), int(flags.item())


def check(case, scale=None, softcap=0.0, window=0, prefix_lens=None, slopes=None, want_flags=0):
    print("[case]", tuple(case[0].shape), case[0].dtype, case[1].dtype, tuple(case[1].shape), case[3], case[4], softcap, window,
          prefix_lens, flush=True)
    q, k, v, starts, lens, table = case
    got, flags = run(case, scale, softcap=softcap, window=window, prefix_lens=prefix_lens, slopes=slopes)
    want, tol = kv_plain.attention(q, k, v, starts, lens, table, q.shape[2] ** -0.5 if scale is None else scale, softcap,
                                   window, prefix_lens, slopes, fill=torch.full(q.shape, 7.0))
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))
    assert flags == want_flags


TYPES = [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 200, 256])
def test_one_token_over_every_head_width(act, kv, dim):
    check(build(dim, [1, 1, 1], [1, 37, 300], 6, 2, dim, 16, act, kv))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (5, 1), (16, 1), (20, 1), (12, 4)])
def test_head_groups(act, kv, heads, kv_heads):
    check(build(heads, [1, 3], [130, 61], heads, kv_heads, 64, 16, act, kv))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("page", [16, 32, 128])
def test_chunks_and_single_tokens_in_one_padded_batch(act, kv, page):
    check(build(page, [1, 70, 0, 33, 5], [200, 70, 0, 95, 129], 8, 2, 128, page, act, kv, pad=9))


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129])
def test_lengths_about_the_tiles(n):
    check(build(n, [n], [n], 3, 1, 64, 16, F32, F16))
    check(build(n, [1], [n], 3, 1, 64, 16, BF16, BF16))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 33, 100])
def test_windows(act, kv, window):
    check(build(window, [1, 40, 3], [150, 90, 3], 4, 2, 64, 16, act, kv), window=window)


@pytest.mark.parametrize("act,kv", TYPES)
def test_prefixes_that_see_themselves_whole(act, kv):
    check(build(1, [60, 20, 5, 1], [60, 90, 5, 40], 4, 2, 128, 16, act, kv), prefix_lens=[33, 95, 0, 1000])
    check(build(2, [60, 20], [60, 90], 4, 2, 64, 16, act, kv), prefix_lens=[33, 95], window=7)


@pytest.mark.parametrize("act,kv", TYPES)
def test_capped_scores_and_distance_biases(act, kv):
    slopes = [2.0 ** -(i + 1) for i in range(6)]
    check(build(3, [1, 40], [200, 77], 6, 3, 64, 32, act, kv), softcap=5.0)
    check(build(4, [1, 40], [200, 77], 6, 3, 64, 32, act, kv), slopes=slopes)
    check(build(5, [3, 40], [200, 77], 6, 3, 128, 32, act, kv), softcap=30.0, slopes=slopes, window=50, prefix_lens=[20, 30],
          scale=0.3)


@pytest.mark.parametrize("act,kv", TYPES)
def test_long_caches_split_over_workgroups(act, kv):
    check(build(6, [1], [3001], 4, 1, 128, 16, act, kv))
    check(build(7, [1, 1, 2], [2500, 3, 700], 4, 2, 64, 64, act, kv))
    check(build(8, [37], [2048], 2, 1, 64, 64, act, kv))


@pytest.mark.parametrize("act,kv", TYPES)
def test_rows_that_see_nothing_are_zero(act, kv):
    """More new tokens than tokens: the first rows lie before position 0 (and the length is reported)."""
    check(build(9, [9], [4], 4, 2, 64, 16, act, kv), want_flags=16)
    check(build(9, [40], [4], 4, 2, 64, 16, act, kv), want_flags=16)
    # a prefix reaches rows before position 0 as well; a window of their own hides it from nobody
    check(build(9, [9], [4], 4, 2, 64, 16, act, kv), prefix_lens=[2], want_flags=16)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_hidden_keys_have_no_influence_whatever_they_hold(act, kv, bad):
    """Non-finite keys and values that some rows of a tile see and others do not."""
    for new, lens, window in (([6], [50], 0), ([70], [90], 0), ([5], [80], 9), ([64], [200], 40)):
        q, k, v, starts, lens, table = build(10, new, lens, 4, 1, 64, 16, act, kv)
        n, m = new[0], lens[0]
        # the last token is seen by its own row alone; with a window the first rows see what the last do not
        marks = [m - 1] + ([m - n - window + 1] if window else [])
        clean, _ = run((q, k, v, starts, lens, table), window=window)
        for j in marks:
            for pool in (k, v):
                pool[table[0][j // 16], :, j % 16, ::3] = bad
        got, _ = run((q, k, v, starts, lens, table), window=window)
        first = n - 1  # rows before the last see no marked last token
        some = 1 if window else 0  # rows from here on do not see the marked first key
        assert torch.equal(got[some:first], clean[some:first])
        assert not torch.isfinite(got[n - 1].float()).all() and bool(torch.isfinite(clean.float()).all())
        # an infinite or missing value alone: seen rows have it in its column, hidden rows stay as they were
        q, k, v, starts, lens, table = build(10, new, lens, 4, 1, 64, 16, act, kv)
        v[table[0][(m - 1) // 16], :, (m - 1) % 16, 5] = bad
        got, _ = run((q, k, v, starts, lens, table), window=window)
        assert torch.equal(got[:n - 1], clean[:n - 1])
        last = got[n - 1].float()
        assert bool((torch.isnan(last[:, 5]) if bad != bad else last[:, 5] == bad).all())
        assert bool(torch.isfinite(torch.cat((last[:, :5], last[:, 6:]), 1)).all())


@pytest.mark.parametrize("dim", [8, 72, 80, 128, 200])
def test_an_infinite_score_stays_in_the_rows_that_see_it(dim):
    """An infinity in a key's last value, beside which a narrower head's kernel has zeros of q: rows that see it
    may be NaN, as the interface says; where they are not, the key has no weight.  No other row changes."""
    for act, kv in TYPES:
        for new, lens in (([1], [70]), ([40], [77])):
            case = build(30, new, lens, 4, 1, dim, 16, act, kv)
            q, k, v, starts, _, table = case
            q[..., -1] = q[..., -1].abs() + 0.5
            clean, _ = run(case)
            k[table[0][2], :, 8, -1] = -float("inf")  # token 40: rows 3 .. 39 of 40 see it, or the only one
            got, _ = run(case)
            before = 3 if len(got) > 1 else 0
            assert torch.equal(got[:before], clean[:before])
            m = lens[0]
            keep = [j for j in range(m) if j != 40]
            z = q[-1, 2].double() @ kv_plain.gathered(k, table[0], m, 0)[keep].T * dim ** -0.5
            want = torch.softmax(z, 0) @ kv_plain.gathered(v, table[0], m, 0)[keep]
            if bool(torch.isfinite(got[-1, 2].float()).all()):
                # half a step of the weights and of the output, of values under 4
                assert float((got[-1, 2].double() - want).abs().max()) < 2 * 4 * kv_plain.HALF_STEP[act]
            else:
                assert bool(torch.isnan(got[-1, 2].float()).all()) and (act == F32 or dim not in (64, 128))


@pytest.mark.parametrize("act,kv", TYPES)
def test_windows_and_scales_at_their_limits(act, kv):
    case = build(31, [1, 30], [50, 64], 4, 2, 64, 16, act, kv)
    plain, _ = run(case)
    assert torch.equal(run(case, window=2 ** 31 - 1)[0], plain)
    check(case, scale=0.0)
    check(case, scale=-0.2)
    check(case, scale=1e-12, slopes=[0.5, 0.25, 0.125, 0.0])
    check(case, softcap=1e-3)
    case = build(31, [30], [9], 4, 2, 64, 16, act, kv)  # rows before position 0
    assert torch.equal(run(case, window=2 ** 31 - 1)[0], run(case)[0])


def test_extreme_queries_keep_fp32_accuracy():
    """fp32 rows whose values fp16 could not hold: far over its largest, far under its smallest."""
    case = list(build(11, [1, 5], [90, 40], 4, 2, 128, 16, F32, F16))
    case[0][0] *= 1e7
    case[0][1:] *= 1e-7
    check(tuple(case), scale=1e-6)
    check(tuple(case), slopes=[0.5, 0.25, 0.125, 0.0625], scale=1e-6)
    case[0] *= 1e-25
    check(tuple(case), slopes=[0.5, 0.25, 0.125, 0.0625])
    case[0].zero_()
    check(tuple(case))


def test_page_ids_outside_the_pool_are_left_out_and_reported():
    q, k, v, starts, lens, table = build(12, [1, 30], [100, 64], 4, 2, 64, 16, F32, F16)
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = [list(r) for r in table]
        t[0][2] = t[1][1] = bad
        got, flags = run((q, k, v, starts, lens, t))
        assert flags == 8
        # as if keys 32 .. 47 of the first sequence were not there
        z = q[0].double() @ kv_plain.gathered(k, table[0], 100, 0).T  # (head 0's KV head)
        keep = [j for j in range(100) if not 32 <= j < 48]
        w = torch.softmax(z[0, keep] * 64 ** -0.5, 0)
        want = w @ kv_plain.gathered(v, table[0], 100, 0)[keep]
        assert float((got[0, 0].double() - want).abs().max()) < 1e-5
        assert bool(torch.isfinite(got).all())


def test_lengths_and_starts_that_do_not_fit_are_cut_and_reported():
    q, k, v, starts, lens, table = build(13, [2, 3], [40, 40], 4, 2, 64, 16, F32, F16, pad=3)
    good, flags = run((q, k, v, starts, lens, table))
    assert flags == 0
    for s, n in (([0, 2, 500], lens), ([-7, 2, 5], lens), ([0, 2, 1], lens), (starts, [1 << 30, 40]), (starts, [-5, 40])):
        got, flags = run((q, k, v, s, n, table))
        assert flags & 16
    got, _ = run((q, k, v, [0, 2, 1], lens, table))
    assert torch.equal(got[:2], good[:2]) and bool((got[2:] == 7).all())


def test_strided_pools_layers_and_streams():
    """K and V as halves of one tensor, a layer of several, a stream that is not the current one."""
    from inferno_hip import device as D
    q, k, v, starts, lens, table = build(14, [3, 1], [70, 33], 4, 2, 64, 16, F16, F16)
    want, _ = run((q, k, v, starts, lens, table))
    both = torch.zeros(2, k.shape[0], 2, *k.shape[1:], dtype=F16, device="cuda")
    both[1, :, 0], both[1, :, 1] = k.cuda(), v.cuda()
    cache = D.KVCache(both[:, :, 0], both[:, :, 1])
    assert cache.layers == 2
    batch = D.KVBatch(ints(starts), ints(lens), ints(table), q.shape[0])
    qd = q.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = D.attn_paged(qd, cache.layer(1), batch, stream=side)
    side.synchronize()
    assert torch.equal(got.cpu(), want)
    for bad in (lambda: D.attn_paged(qd, cache, batch), lambda: D.attn_paged(qd.float().double(), cache.layer(0), batch),
                lambda: D.attn_paged(qd[:2], cache.layer(0), batch), lambda: D.KVCache(k.cuda(), v.cuda()[:-1]),
                lambda: D.KVCache(k.cuda().transpose(1, 2), v.cuda().transpose(1, 2)), lambda: D.KVCache(k, v),
                lambda: D.attn_paged(qd, cache.layer(0), batch, out=torch.empty_like(qd).float()),
                lambda: D.attn_paged(qd, cache.layer(0), batch, slopes=torch.zeros(3, device="cuda"))):
        with pytest.raises(D.IHIPArgumentError):
            bad()


def test_a_captured_call_replays_with_new_contents():
    from inferno_hip import device as D
    q, k, v, starts, lens, table = build(15, [1, 1], [1500, 900], 8, 2, 128, 16, F32, F16)
    cache = D.KVCache(k.cuda().nan_to_num_(0.0), v.cuda().nan_to_num_(0.0))
    ln = ints(lens)
    batch = D.KVBatch(ints(starts), ln, ints(table), 2)
    qd, out = q.cuda(), torch.empty_like(q, device="cuda")
    ws = D.attn_workspace(8, cache, batch)
    D.attn_paged(qd, cache, batch, out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D.attn_paged(qd, cache, batch, out=out, workspace=ws)
    for i in range(4):
        qd.normal_(generator=None)
        ln.copy_(ints([1500 - 301 * i, 900 - 17 * i]))
        want = D.attn_paged(qd, cache, batch).clone()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_the_same_call_twice_gives_the_same_bits():
    case = build(16, [1, 40], [2000, 300], 8, 2, 128, 16, BF16, BF16)
    assert torch.equal(run(case)[0], run(case)[0])


def test_offsets_past_32_bits():
    """Pages beyond 2^32 elements and bytes of the pool."""
    from inferno_hip import device as D
    q, k, v, starts, lens, table = build(17, [1], [60], 4, 2, 128, 16, F32, F16)
    per = 1 << 20
    pages = (1 << 32) // per + 8  # 8.6 GB each
    kk = torch.empty(pages * per, dtype=F16, device="cuda")
    vv = torch.empty(pages * per, dtype=F16, device="cuda")
    shape, strides = (pages, 2, 16, 128), (per, 16 * 128, 128, 1)
    kk, vv = kk.as_strided(shape, strides), vv.as_strided(shape, strides)
    far = [pages - 1 - i for i in range(4)]
    for i, p in enumerate(far):
        kk[p], vv[p] = k[table[0][i]].cuda(), v[table[0][i]].cuda()
    want, _ = run((q, k, v, starts, lens, table))
    got = D.attn_paged(q.cuda(), D.KVCache(kk, vv), D.KVBatch(ints(starts), ints(lens), ints([far]), 1))
    # (another capacity may split the keys otherwise: the same to rounding)
    assert float((got.cpu() - want).abs().max()) < 1e-5


def test_one_workspace_serves_calls_of_all_sizes():
    """The counts in its front are zero again after every call, whatever the next one's sizes."""
    from inferno_hip import device as D
    from inferno_hip import _lib
    cases = [build(20, [1], [3000], 8, 2, 64, 16, F32, F16), build(21, [1] * 9, [900] * 9, 8, 8, 64, 16, F32, F16),
             build(22, [40], [700], 8, 2, 64, 16, F32, F16), build(23, [2], [2000], 4, 1, 64, 16, F32, F16)]
    made = []
    for q, k, v, starts, lens, table in cases:
        cache = D.KVCache(k.cuda(), v.cuda())
        batch = D.KVBatch(ints(starts), ints(lens), ints(table), q.shape[0])
        made.append((q.cuda(), cache, batch, D.attn_paged(q.cuda(), cache, batch)))
    n = max(_lib.lib().ihip_attn_paged_scratch_bytes(_lib.F32, q.shape[1], c.ref, b.ref) for q, c, b, _ in made)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    for i in (0, 1, 2, 3, 1, 0, 3, 2, 0):
        q, cache, batch, want = made[i]
        assert torch.equal(D.attn_paged(q, cache, batch, workspace=ws), want)
        assert not bool(ws[:16384].any())
