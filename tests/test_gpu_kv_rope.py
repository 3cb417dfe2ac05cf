"""Norm, rotary positions and the append to the paged cache against the plain
form in 64 bits."""
import pytest

import kv_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(new, lens, heads, kv_heads, dim, rot, layout, norm, act, kv, page=16, pad=0, far=None, scaling="none", q_only=False,
          seed=1):
    from inferno_hip import device as D
    print("[case]", new, lens, heads, kv_heads, dim, rot, layout, norm, act, kv, page, pad, far, scaling, flush=True)
    g = torch.Generator().manual_seed(seed)
    T = sum(new) + pad
    x = 2 * torch.randn(T, heads + 2 * kv_heads, dim, generator=g)
    qn, kn = (1 + 0.2 * torch.randn(dim, generator=g), 1 + 0.2 * torch.randn(dim, generator=g)) if norm else (None, None)
    counts = [-(-n // page) for n in lens]
    pages, width = sum(counts) + 2, max(counts + [1])
    order = torch.randperm(pages, generator=g).tolist()
    table, i = [], 0
    for n in counts:
        table.append(order[i:i + n] + [-1] * (width - n))
        i += n
    k0 = torch.randn(pages, kv_heads, page, dim, generator=g).to(kv)
    v0 = torch.randn(pages, kv_heads, page, dim, generator=g).to(kv)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    if rot:
        turns, m = D.rope_turns(rot, 1e4, scaling, factor=4.0, original=4096)
    else:
        turns, m = torch.zeros(0, dtype=torch.float64, device="cuda"), 1.0
    pos = None if far is None else [far + 3 * t for t in range(T)]
    xd = x.cuda()
    cache = D.KVCache(k0.cuda(), v0.cuda())
    batch = D.KVBatch(ints(starts), ints(lens), ints(table), T)
    out = torch.full((T, heads, dim), 7.0, dtype=act, device="cuda")
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = (None, None) if q_only else (xd[:, heads:heads + kv_heads], xd[:, heads + kv_heads:])
    D.rope_kv(xd[:, :heads], k, v, turns, cache, batch, layout=layout, mscale=m, q_norm=None if qn is None else qn.cuda(),
              k_norm=None if kn is None else kn.cuda(), positions=None if pos is None else ints(pos), out=out, flags=flags)
    torch.cuda.synchronize()
    assert int(flags.item()) == 0
    tw = turns.cpu()
    got, gk, gv = out.cpu(), cache.k.cpu(), cache.v.cpu()
    want_k, want_v = k0.clone(), v0.clone()
    for s, n in enumerate(new):
        for i in range(n):
            t, at = starts[s] + i, lens[s] - n + i
            p = at if pos is None else pos[t]
            for h in range(heads):
                y, e = kv_plain.rope(x[t, h], p, tw, rot, layout, m, qn)
                e = e + kv_plain.HALF_STEP[act] * y.abs() + 2.0 ** -25 * (act == F16) + 2.0 ** -24 * y.abs()
                assert bool(((got[t, h].double() - y).abs() <= e).all()), (t, h, float((got[t, h].double() - y).abs().max()))
            if q_only:
                continue
            page_id, slot = table[s][at // page], at % page
            for h in range(kv_heads):
                y, e = kv_plain.rope(x[t, heads + h], p, tw, rot, layout, m, kn)
                e = e + kv_plain.HALF_STEP[kv] * y.abs() + 2.0 ** -25 * (kv == F16) + 2.0 ** -24 * y.abs()
                assert bool(((gk[page_id, h, slot].double() - y).abs() <= e).all()), (t, h)
                want_k[page_id, h, slot] = gk[page_id, h, slot]
                want_v[page_id, h, slot] = x[t, heads + kv_heads + h].to(kv)
    # values are only rounded; every other slot is as it was, and so are the padded rows
    assert torch.equal(gv, want_v) and torch.equal(gk, want_k)
    assert bool((got[sum(new):] == 7).all())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(8, 8), (64, 64), (64, 16), (80, 20), (80, 80), (128, 128), (128, 2), (200, 100), (256, 64),
                                     (256, 256), (64, 0)])
def test_head_widths_and_rotated_parts(layout, dim, rot):
    check([3, 1], [20, 1], 5, 2, dim, rot, layout, True, F32, F16)


@pytest.mark.parametrize("act", [F32, F16, BF16])
@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("norm", [False, True])
def test_types_and_norms(act, kv, norm):
    check([1, 0, 6], [40, 0, 6], 6, 3, 64, 64, "half", norm, act, kv, page=32, pad=4)


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn", "bands"])
def test_far_positions_under_every_scaling(scaling):
    check([2], [9], 2, 1, 128, 128, "half", False, F32, F16, far=1_000_003, scaling=scaling)
    check([2], [9], 2, 1, 64, 32, "interleaved", False, F32, BF16, far=2_000_000_000, scaling=scaling)
    check([2], [9], 2, 1, 64, 32, "interleaved", False, F32, BF16, far=-70_000, scaling=scaling)


@pytest.mark.parametrize("heads,kv_heads,new", [(64, 8, [1]), (1, 1, [1, 1, 1]), (40, 40, [2]), (71, 1, [1]), (8, 2, [70])])
def test_head_counts_about_the_workgroups(heads, kv_heads, new):
    check(new, [n + 3 for n in new], heads, kv_heads, 64, 64, "half", True, F16, F16)


def test_q_alone():
    check([3, 2], [30, 2], 4, 2, 64, 64, "half", True, F32, F16, q_only=True)


def test_more_sequences_than_a_wave():
    check([1] * 150, [1 + i % 40 for i in range(150)], 2, 1, 16, 16, "half", False, F32, F16)


def small(**kw):
    from inferno_hip import device as D
    T, H, Hk, dim = 4, 4, 2, 64
    g = torch.Generator().manual_seed(5)
    f = dict(x=torch.randn(T, H + 2 * Hk, dim, generator=g).cuda(), starts=[0, 4], lens=[20], table=[[0, 1]])
    f.update(kw)
    cache = D.KVCache(torch.zeros(3, Hk, 16, dim, dtype=F16, device="cuda"), torch.zeros(3, Hk, 16, dim, dtype=F16, device="cuda"))
    batch = D.KVBatch(ints(f["starts"]), ints(f["lens"]), ints(f["table"]), T)
    turns, _ = D.rope_turns(dim, 1e4)
    return f["x"], turns, cache, batch, torch.zeros(1, dtype=torch.int32, device="cuda")


def test_bad_pages_and_lengths_are_left_out_and_reported():
    from inferno_hip import device as D
    for kw, bit in ((dict(table=[[0, 3]]), 8), (dict(table=[[0, -1]]), 8), (dict(table=[[0, 2 ** 31 - 1]]), 8),
                    (dict(lens=[2]), 16), (dict(lens=[900]), 16), (dict(starts=[0, 9]), 16), (dict(lens=[-3]), 16)):
        x, turns, cache, batch, flags = small(**kw)
        out = D.rope_kv(x[:, :4], x[:, 4:6], x[:, 6:], turns, cache, batch, flags=flags)
        torch.cuda.synchronize()
        assert int(flags.item()) == bit, kw
        assert bool(torch.isfinite(out).all())
        if bit == 8:  # positions 16 .. 19 lie on the page that is not there
            assert not bool(cache.k.any()) and not bool(cache.v.any())
    x, turns, cache, batch, flags = small(lens=[2])  # tokens at -2, -1, 0, 1
    D.rope_kv(x[:, :4], x[:, 4:6], x[:, 6:], turns, cache, batch)
    assert torch.equal(cache.v[0, :, :2].cpu(), x[2:, 6:].to(F16).transpose(0, 1).cpu())
    assert not bool(cache.v[0, :, 2:].any()) and not bool(cache.v[1:].any())


def test_in_place_and_another_stream():
    from inferno_hip import device as D
    x, turns, cache, batch, _ = small()
    q = x[:, :4].contiguous()
    want = D.rope_kv(q, x[:, 4:6], x[:, 6:], turns, cache, batch)
    k = cache.k.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = D.rope_kv(q, x[:, 4:6], x[:, 6:], turns, cache, batch, out=q, stream=side)
    side.synchronize()
    assert got is q and torch.equal(q, want) and torch.equal(cache.k, k)


def test_wrapper_refusals():
    from inferno_hip import device as D
    x, turns, cache, batch, _ = small()
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    for bad in (lambda: D.rope_kv(q.half(), k, v, turns, cache, batch), lambda: D.rope_kv(q, k, None, turns, cache, batch),
                lambda: D.rope_kv(q, k[:, :1], v, turns, cache, batch), lambda: D.rope_kv(q, k, v, turns.float(), cache, batch),
                lambda: D.rope_kv(q, k, v, turns, cache, batch, layout="rows"), lambda: D.rope_kv(q[:3], k, v, turns, cache, batch),
                lambda: D.rope_kv(q, k, v, turns, cache, batch, q_norm=torch.ones(63, device="cuda")),
                lambda: D.rope_kv(q, k, v, turns, cache, batch, positions=ints([1, 2, 3])),
                lambda: D.rope_kv(q, k, v, turns, cache, batch, out=torch.empty(4, 4, 64, device="cuda", dtype=torch.float64)),
                lambda: D.rope_kv(q, k, v, torch.cat((turns, turns)), cache, batch), lambda: D.rope_turns(64, 1e4, "other")):
        with pytest.raises(D.IHIPArgumentError):
            bad()
