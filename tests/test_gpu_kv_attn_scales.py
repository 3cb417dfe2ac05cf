"""fp32 rows and scales at the ends of their ranges, whose product is an ordinary
score: a power of two moved from one to the other changes no bit.  Caps, scales
and slopes whose ratios pass 32 bits."""
import pytest

import kv_dense
from test_gpu_kv_attn import BF16, F16, F32, TYPES, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# one token in one part and in several, few rows, chunks in one part and in several, halves
SHAPES = [([1], [90], 4, 2, 6), ([1], [1500], 4, 2, 94), ([5, 1], [300, 70], 4, 2, 19), ([150], [200], 130, 130, 40),
          ([40], [700], 4, 2, 64)]


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,lens,heads,kv_heads,width", SHAPES)
def test_powers_of_two_between_q_and_the_scale(kv, dim, new, lens, heads, kv_heads, width):
    print("[case]", kv, dim, new, lens, flush=True)
    q, *rest = kv_dense.make(dim, new, lens, heads, kv_heads, dim, F32, kv, width=width)
    slopes = [0.5 ** (1 + i % 9) for i in range(heads)]
    for kw in ({}, dict(softcap=4.0), dict(slopes=slopes)):
        want, _ = run((q, *rest), scale=dim ** -0.5, **dict(kw))
        for power in (-110, -70, -40, 20, 33):
            # (q's values are normal numbers still: 2^-126 and up but for a few that leave no trace)
            got, flags = run((q * 2.0 ** power, *rest), scale=dim ** -0.5 * 2.0 ** -power, **dict(kw))
            assert flags == 0 and torch.equal(got, want), (kw, power, float((got - want).abs().max()))


@pytest.mark.parametrize("act,kv", TYPES)
@pytest.mark.parametrize("new,lens,heads,kv_heads,width", SHAPES)
def test_ratios_past_32_bits(act, kv, new, lens, heads, kv_heads, width):
    q, k, v, starts, lens, table = kv_dense.make(7, new, lens, heads, kv_heads, 64, act, kv, width=width)
    most = float(torch.nan_to_num(v.float()).abs().max())
    # sums over the keys; 16 bits: the weights' rounding and the output's
    limit = most * ((max(lens) + 64) * 2.0 ** -23 + (2 * {F16: 2.0 ** -11, BF16: 2.0 ** -8}[act] if act != F32 else 0.0))

    def mean_of(weighted):
        """Every key that a row sees has the same weight, or its own key all of it."""
        z = torch.zeros_like(q)
        return kv_dense.attention(z, k, v, starts, lens, table, slopes=[1e9] * heads if weighted else None)[0]

    rows = slice(0, sum(new))
    # all scores are within a cap of 1e-12, however steep the way there; rows of zeros stay at 0
    for x in (q, torch.zeros_like(q)):
        got, _ = run((x, k, v, starts, lens, table), scale=1e30, softcap=1e-12)
        assert float((got[rows].double() - mean_of(False)[rows]).abs().max()) <= limit
    # a cap near the largest number, scores of 0
    got, _ = run((torch.zeros_like(q), k, v, starts, lens, table), scale=1.0, softcap=3e38)
    assert float((got[rows].double() - mean_of(False)[rows]).abs().max()) <= limit
    # a slope that dwarfs the smallest scale and row: a row's own key has all of the weight
    x = q * 2.0 ** -100 if act == F32 else q
    got, _ = run((x, k, v, starts, lens, table), scale=1e-12, slopes=[1e30] * heads)
    assert float((got[rows].double() - mean_of(True)[rows]).abs().max()) <= limit
