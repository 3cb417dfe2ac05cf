"""Scores far from 0, whose differences alone say the weights: products of whole
numbers that every sum holds exactly, so that the weights are those of the plain
form in 64 bits however large the scores are."""
import pytest

import kv_plain
from test_gpu_kv_attn import BF16, F16, F32, TYPES, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# (new tokens, tokens, table entries): decode in one part and in several, few rows,
# chunks in one part and in several (tables wide enough for the kernel of many rows)
SHAPES = [([1], [90], 6), ([1], [1500], 94), ([5, 1], [300, 70], 19), ([60, 40], [210, 64], 40), ([40], [700], 64)]


def pools(seed, lens, width, dim, kv, key):
    """Pools, tables and the keys' first values key(s, j, g): the rest of k is 0, v is random."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // 16) for n in lens]
    order = torch.randperm(sum(counts) + 1, generator=g).tolist()
    k = torch.zeros(sum(counts) + 1, 2, 16, dim)
    v = torch.randn(sum(counts) + 1, 2, 16, dim, generator=g).to(kv)
    table, i = [], 0
    for s, n in enumerate(lens):
        table.append(order[i:i + counts[s]] + [-1] * (width - counts[s]))
        i += counts[s]
        for j in range(n):
            x = key(s, j, g)
            k[table[s][j // 16], :, j % 16, :len(x)] = torch.tensor(x)
    assert torch.equal(k.to(kv).float(), k)
    return k.to(kv), v, table


def agree(q, k, v, new, lens, table, scale, act, weights_off, **kw):
    """Every row against the plain form, whose weights are exact but for `weights_off`."""
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    assert torch.equal(q.to(act).float(), q)
    case = q.to(act), k, v, starts, lens, table
    got, flags = run(case, scale, **dict(kw))
    assert flags == 0 and bool(torch.isfinite(got.float()).all())
    want, _ = kv_plain.attention(*case, scale, kw.get("softcap", 0.0), slopes=kw.get("slopes"))
    # an average of the values: sums over the keys and the parts; 16 bits: the weights' rounding and the output's
    most = float(v.float().abs().max())
    limit = most * ((max(lens) + 64) * 2.0 ** -24 + weights_off)
    if act != F32:
        limit += 2 * most * kv_plain.HALF_STEP[act]
    err = float((got.double() - want).abs().max())
    assert err <= limit, (err, limit)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,lens,width", SHAPES)
def test_small_differences_of_large_scores(act, kv, dim, new, lens, width):
    """Scores of 1.5 * 2^24 (over 2^25 as powers of two) and 0 to 6 more: even numbers, which 32 bits hold there.  The
    rows differ in the key that they like best, so that their maxima rise at different steps.

    A weight is e to a difference that is exact.  As a power of two it is off by 1.5 steps of 2^-24 of its size
    (log2 e, and times the scale) and half a step of an exponent under 16 (2^-21, ln 2 of which is the weight's),
    then the exponential's 2^-23 and the parts' 2^-22: with differences to 6 under 2^-19 in all, to 12 under 2^-18."""
    print("[case]", act, kv, dim, new, lens, flush=True)
    k, v, table = pools(1, lens, width, dim, kv, lambda s, j, g: [128.0] + torch.randint(0, 4, (4,), generator=g).tolist())
    T = sum(new)
    q = torch.zeros(T, 4, dim)
    q[:, :, 0] = 1.5 * (2.0 ** 17 if act == F32 else 2.0 ** 15)  # (16 bits: times a scale of 4)
    unit = 2.0 if act == F32 else 0.5
    q[torch.arange(T)[:, None], torch.arange(4), 1 + (torch.arange(T)[:, None] + torch.arange(4)) % 4] = unit
    agree(q, k, v, new, lens, table, 1.0 if act == F32 else 4.0, act, 2.0 ** -19)
    if act == F32:  # below 0, and twice as far
        q[:, :, 0] *= -1
        agree(q, k, v, new, lens, table, 1.0, act, 2.0 ** -19)
        agree(q, k, v, new, lens, table, 2.0, act, 2.0 ** -18)


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,lens,width", SHAPES)
def test_equal_keys_of_any_score_share_the_weight(act, kv, dim, new, lens, width):
    """Keys 0, 3, 6 .. lie above all others by more than any weight shows, from 1e7 up to 1e30; the rows' own
    sizes differ.  Capped the same."""
    print("[case]", act, kv, dim, new, lens, flush=True)
    k, v, table = pools(2, lens, width, dim, kv, lambda s, j, g: [0.0 if j % 3 else 120.0])
    T = sum(new)
    for scale in (2.0, 256.0, 2.0 ** 80):
        q = torch.zeros(T, 4, dim)
        q[:, :, 0] = (2.0 ** 15 + 1024.0 * (torch.arange(4 * T) % 4).view(T, 4)) if act != BF16 else \
            2.0 ** 15 + 256.0 * (torch.arange(4 * T) % 4).view(T, 4)
        agree(q, k, v, new, lens, table, scale, act, 0.0)
        if scale == 256.0:
            agree(q, k, v, new, lens, table, scale, act, 0.0, softcap=2.0 ** 30)


def test_a_bias_that_dwarfs_every_score():
    """Slopes of 2^20 and up: a row's own key has all of the weight."""
    for act, kv in TYPES:
        for new, lens, width in SHAPES:
            k, v, table = pools(3, lens, width, 64, kv, lambda s, j, g: torch.randn(8, generator=g).to(F16).to(BF16).tolist())
            q = torch.randn(sum(new), 4, 64, generator=torch.Generator().manual_seed(4)).to(act).float()
            agree(q, k, v, new, lens, table, 0.125, act, 0.0, slopes=[2.0 ** 20, 2.0 ** 24, 2.0 ** 27, 2.0 ** 30])
