"""The choice of a token against its definition in 64 bits (gd_plain.sample): every
token equal, every logprob to fp32's rounding."""
import math

import numpy as np
import pytest

import gd_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def check(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, **kw):
    """logits: rows x vocab on the CPU; settings: lists or None."""
    from inferno_hip import device as D
    n = logits.shape[0]
    f = lambda v: None if v is None else torch.tensor(v, dtype=F32, device="cuda")
    i = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")
    lp, fl = torch.full((n,), 9.0, device="cuda"), torch.full((n,), 77, dtype=torch.int32, device="cuda")
    got = D.sample(kw.get("on_device", logits.cuda()), f(u), temperature=f(temperature), top_k=i(top_k), top_p=f(top_p),
                   min_p=f(min_p), logprobs=lp, flags=fl).tolist()
    at = lambda v, r: None if v is None else v[r] if isinstance(v[r], int) else float(np.float32(v[r]))
    for r in range(n):
        token, logprob, flags = gd_plain.sample(logits[r].double().numpy(), at(u, r), at(temperature, r), at(top_k, r), at(top_p, r),
                                                at(min_p, r))
        assert int(fl[r]) == flags, (r, int(fl[r]), flags)
        assert got[r] == token, (r, got[r], token)
        x = float(lp[r])
        # sums of 2^-52 a token, then one rounding
        assert (math.isnan(x) and math.isnan(logprob)) or abs(x - logprob) <= 2.0 ** -23 * abs(logprob) + 1e-10, (r, x, logprob)
    return got


def rows(seed, n, vocab, kind=F32, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = spread * torch.randn(n, vocab, generator=g)
    x += 12 * torch.rand(n, vocab, generator=g).pow(2) * (torch.rand(n, vocab, generator=g) < 1e-3)
    return x.to(kind), torch.rand(n, generator=g).tolist()


VOCABS = [1, 2, 3, 5, 100, 1023, 4096, 4097, 8192, 8193, 5003, 32000, 151936]


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("vocab", VOCABS)
def test_settings_and_sizes(vocab, kind):
    print("[case]", vocab, kind, flush=True)
    n = 14
    x, u = rows(vocab, n, vocab, kind)
    t = [0.0, 1.0, 0.7, 0.3, 1.5, 1.0, 0.8, 1.0, 0.1, 5.0, 1.0, 1.0, 0.6, 1.0]
    k = [0, 0, 1, 50, 1000, 0, 20, vocab, vocab - 1, 3, 0, -5, 40, 2]
    p = [0.9, 1.0, 0.9, 1.0, 0.95, 0.5, 0.9, 0.0, 0.999, 1.0, 0.99, 1e-6, 0.95, 1.0]
    m = [0.0, 0.0, 0.0, 0.05, 0.0, 0.2, 0.0, 0.0, 1.0, 0.0, 0.01, 0.0, 0.1, 0.0]
    check(x, u, t, k, p, m)
    check(x, u)
    check(x, u, t)
    check(x, u, None, k)
    check(x, u, t, None, p)
    check(x, u, t, None, None, m)
    check(x, u, t, k, None, m)


def test_many_rows_and_launches():
    """Rows of one launch and of several (256 of them each), whole and in few slices."""
    for n, vocab in ((300, 700), (600, 40)):
        x, u = rows(n, n, vocab)
        check(x, u, [0.8] * n, [5 + i % 30 for i in range(n)], [0.9] * n)
        check(x, u, [1.0] * n)


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan])
def test_the_ends_of_u(u):
    x, _ = rows(3, 4, 9000)
    x[:, :3] = -math.inf
    x[:, -2:] = -math.inf
    for settings in ({}, dict(top_k=[5] * 4), dict(top_p=[0.9] * 4), dict(min_p=[0.05] * 4)):
        check(x, [u] * 4, [1.0] * 4, **settings)


def test_equal_logits():
    """Ties go to the lowest index, also where thousands of them lie at a boundary."""
    for vocab in (10, 5000, 20000):
        x = torch.zeros(6, vocab)
        x[2:, ::3] = 1.0
        u = [0.1, 0.99, 0.3, 0.7, 0.999, 0.0]
        check(x, u, [1.0] * 6, [0, 7, vocab // 2, vocab // 2, 1, vocab - 1])
        check(x, u, [1.0] * 6, None, [0.5, 0.9, 0.3, 0.99, 0.01, 0.7])
        check(x, u, [1.0, 2.0, 0.5, 1.0, 3.0, 1.0], [vocab // 3 + 5] * 6, [0.5, 0.9, 0.3, 0.99, 0.01, 0.7])
        check(x, u, [1.0] * 6, None, None, [1.0, 0.3, 1.0, 0.3, 2.0, 0.5])
        check(x, u, [0.0] * 6)


def test_tokens_that_are_ruled_out():
    for kind in (F32, F16, BF16):
        x, u = rows(4, 6, 6000, kind)
        x[0, 5:] = -math.inf
        x[1, 100:] = torch.finfo(kind).min
        x[2, :-1] = -math.inf
        x[3] = -math.inf
        x[4, ::2] = -math.inf
        x[5] = torch.finfo(kind).min
        check(x, u, [0.8] * 6, [50] * 6, [0.95] * 6, [0.02] * 6)
        check(x, u, [0.8] * 6, [3000] * 6)
        check(x, u, [0.8] * 6)
        check(x, u, [0.0] * 6)


def test_rows_that_are_not_finite():
    x, u = rows(5, 5, 9000)
    x[0, 8999], x[1, 17], x[2, 3], x[2, 8000] = math.nan, math.inf, math.nan, math.inf
    x[3] = -math.inf
    for t in (1.0, 0.0):
        check(x, u, [t] * 5, [40] * 5, [0.9] * 5)
        check(x, u, [t] * 5)
        check(x, u, [t] * 5, None, None, [0.1] * 5)


def test_sizes_of_logits_and_temperatures():
    x, u = rows(6, 8, 5000)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] += 1e6
    x[3] -= 1e6
    x[4] *= 1e4
    for t in (1e-30, 1e-3, 1.0, 1e3, 1e30, math.inf, math.nan, -1.0):
        check(x, u, [t] * 8, [30] * 8, [0.9] * 8)
        check(x, u, [t] * 8)
    check(x, u, [1.0] * 8, None, [math.nan] * 8, [math.nan] * 8)


def test_zeros_of_either_sign_are_equal():
    x = torch.full((2, 50), -1.0)
    x[0, 3], x[0, 7], x[1, 3], x[1, 7] = -0.0, 0.0, 0.0, -0.0
    check(x, [0.2, 0.2], [1.0] * 2, [1] * 2)
    check(x, [0.2, 0.2], [0.0] * 2)


def test_more_tokens_at_a_boundary_than_the_list_holds():
    """30000 logits within one bin, and half of them equal."""
    x = torch.rand(3, 30000, generator=torch.Generator().manual_seed(1)) * 1e-3
    x[1, ::2] = 5e-4
    for settings in (dict(top_k=[9000] * 3), dict(top_p=[0.37] * 3), dict(top_k=[20000] * 3, top_p=[0.6] * 3, min_p=[0.9999] * 3)):
        check(x, [0.3, 0.6, 0.99], [1.0] * 3, **settings)


@pytest.mark.parametrize("kind", [F32, F16, BF16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strides_and_alignment(kind, shift):
    x, u = rows(7, 5, 9001, kind)
    wide = torch.full((5, 9010), math.nan).to(kind).cuda()
    view = wide[:, shift:shift + 9001]
    view.copy_(x)
    check(x, u, [0.9] * 5, [60] * 5, [0.9] * 5, on_device=view)
    check(x, u, on_device=view)


def test_the_chances_are_the_shares():
    """Over evenly spread numbers every token comes as often as its share says."""
    x, _ = rows(8, 1, 300)
    n = 2000
    u = [(i + 0.5) / n for i in range(n)]
    got = check(x.expand(n, -1).contiguous(), u, [1.0] * n, [20] * n)
    w = torch.softmax(x[0].double(), 0)
    top = w.topk(20)
    share = (top.values / top.values.sum()).tolist()
    for token, s in zip(top.indices.tolist(), share):
        assert abs(got.count(token) - s * n) <= 2
    assert sorted(got) == got  # the token does not decrease with u
