"""A batch whose first sequence does not start at row 0: the decode rows and the
prompt rows of one buffer called apart, rows before and behind them of no
sequence."""
import pytest

import kv_plain
from test_gpu_kv_attn import TYPES, build, ints, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def behind(case, rows):
    """The same batch with `rows` rows of no sequence before its first one."""
    q, k, v, starts, lens, table = case
    more = torch.randn(rows, *q.shape[1:], generator=torch.Generator().manual_seed(rows)).to(q.dtype)
    return torch.cat((more, q)), k, v, [rows + s for s in starts], lens, table


@pytest.mark.parametrize("rows", [1, 2, 70])
@pytest.mark.parametrize("new,lens,pad", [([3], [10], 0), ([1], [40], 3), ([1, 0, 6, 2], [40, 3, 6, 33], 4), ([1] * 70, [5] * 70, 2)])
def test_rope_and_append(rows, new, lens, pad):
    """Every row as it is in a batch of its own from row 0; other rows and slots as they were."""
    from inferno_hip import device as D
    print("[case]", rows, new, lens, pad, flush=True)
    H, Hk, dim, page = 3, 2, 64, 16
    g = torch.Generator().manual_seed(rows)
    T, n = rows + sum(new) + pad, sum(new)
    x = torch.randn(T, H + 2 * Hk, dim, generator=g).cuda()
    counts = [-(-m // page) for m in lens]
    order = torch.randperm(sum(counts) + 2, generator=g).tolist()
    table, i = [], 0
    for c in counts:
        table.append(order[i:i + c] + [-1] * (max(counts) - c))
        i += c
    turns, m = D.rope_turns(dim, 1e4)
    far = torch.arange(1000, 1000 + T, dtype=torch.int32, device="cuda")
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    made = []
    for first, y, positions in ((0, x[rows:rows + n], far[rows:rows + n]), (rows, x, far), (0, x[rows:rows + n], None), (rows, x, None)):
        cache = D.KVCache(*(torch.full((len(order), Hk, page, dim), 3.0, dtype=torch.float16, device="cuda") for _ in range(2)))
        batch = D.KVBatch(ints([first + s for s in starts]), ints(lens), ints(table), len(y))
        flags = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full((len(y), H, dim), 7.0, device="cuda")
        D.rope_kv(y[:, :H], y[:, H:H + Hk], y[:, H + Hk:], turns, cache, batch, mscale=m, positions=positions, out=out, flags=flags)
        made.append((out, cache.k, cache.v))
        assert int(flags.item()) == 0
    for a, b in ((made[0], made[1]), (made[2], made[3])):
        assert bool((b[0][:rows] == 7).all()) and bool((b[0][rows + n:] == 7).all())
        assert torch.equal(a[0], b[0][rows:rows + n])
        assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    # and against the formula, the first row of the first sequence
    want, e = kv_plain.rope(x[rows, 0].cpu(), lens[0] - new[0], turns.cpu(), dim, "half", m)
    assert bool(((made[3][0][rows, 0].cpu().double() - want).abs() <= e + 2.0 ** -23).all())


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
def test_attention(act, kv, rows):
    """Few rows, a chunk in tables of any length, one whose keys are split and joined."""
    for new, lens, width, pad in (([1, 3], [90, 40], 0, 2), ([50, 0, 2], [70, 3, 40], 64, 3), ([40], [700], 64, 1)):
        q, k, v, starts, lens, table = build(41, new, lens, 4, 2, 64, 16, act, kv, pad=pad)
        case = q, k, v, starts, lens, [r + [-1] * (width - len(r)) for r in table]
        want, _ = run(case)
        far = behind(case, rows)
        got, flags = run(far)
        n = sum(new)
        assert flags == 0 and bool((got[:rows] == 7).all()) and bool((got[rows + n:] == 7).all())
        # (more rows may split the keys otherwise: against the plain form)
        exact, tol = kv_plain.attention(*far, 64 ** -0.5, fill=torch.full(far[0].shape, 7.0))
        assert bool(((got.double() - exact).abs() <= tol).all())
        assert bool(((want.double() - exact[rows:]).abs() <= tol[rows:]).all())
