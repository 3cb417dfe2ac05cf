"""The gated delta rule row by row against its definition in 64 bits, where tokens of one
chunk, or a state and what is written to it, are of very different sizes: no row may
lose its values beside another one's.

What a row may be off by.  A column of the state is no longer than

  env_t = alpha_t env_(t-1) + beta_t |v_t|

(k has unit length, and a write takes back what k brings back).  Each product that leads
to a row of outputs (k's norms, K S, what is written, Q S) is an fp32 sum of up to 128
terms, whose roundings of 2^-24 a term have no common sign: 2^-20 of what the row can sum,
that is of scale * |q^| * env with |q^| <= 1, holds them with room, for the row's
columns together.  Errors of older tokens fade with what they came from, as env does.  A
value that vanishes beside a larger one is off by all of its row.

A decay is e^g with g = decay * softplus(a + dt_bias) of fp32 values: the sum, the
exponential, the logarithm and the product are a step of 2^-24 off or two each, so g is off by
2^-22 of itself and e^g by |g| 2^-22 of itself.  What passes it is off by as much:

  D_t = alpha_t (D_(t-1) + |g_t| env_(t-1)),   2^-22 D_t beside 2^-20 env_t.

And fp32's own numbers end at 2^-126: a product of decays below that may count as nothing,
which takes 2^-126 of the largest env so far.
"""
import pytest

import gd_plain
from test_gpu_gd_delta import Case

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}


def bounds(c):
    """What rows (tokens x heads x v_dim, before norm and gate) and the last states' columns may be off by."""
    _, _, v = c.parts(c.qkv)
    H, dk = v.shape[1], c.shape[2]
    g = c.decay.double().clamp(max=0) * torch.nn.functional.softplus(c.a.double() + c.dt_bias.double(), threshold=600)
    alpha, beta = torch.exp(g), torch.sigmoid(c.b.double())
    rows, last = torch.zeros(v.shape, dtype=torch.float64), {}
    for n, begin, slot, at in zip(c.new, c.begins, c.slots, c.starts):
        if n == 0:
            continue
        env = torch.zeros(H, v.shape[2], dtype=torch.float64) if begin else c.state[slot].double().norm(dim=1)
        D, most = torch.zeros_like(env), env
        for t in range(at, at + n):
            D = alpha[t][:, None] * (D + g[t].abs()[:, None] * env)
            env = alpha[t][:, None] * env + beta[t][:, None] * v[t].double().abs()
            most = torch.maximum(most, env)
            rows[t] = gd_plain.NEAR * env + 2.0 ** -22 * D + 2.0 ** -126 * most
        last[slot] = rows[at + n - 1]
    return dk ** -0.5 * rows, last


def check(c, **kw):
    out, state, flags = c.run(**kw)
    want, held = c.plain()
    rows, last = bounds(c)
    assert flags == 0
    live = slice(c.starts[0], c.starts[-1])
    tol = rows.norm(dim=-1)
    if c.norm_w is not None or c.gate is not None:
        plain_o = gd_plain.delta(*c.parts(c.qkv), c.a, c.b, c.decay, c.dt_bias, c.state, c.new, c.begins, c.slots, c.starts,
                                 c.out.double())[0]
        by = torch.ones_like(plain_o)
        if c.norm_w is not None:
            # o / rms: a row's own error and, at most as much again, its length's
            by = by * c.norm_w.double() * 2 / (plain_o.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        if c.gate is not None:
            by = by * torch.nn.functional.silu(c.gate.double())
        tol = tol * by.abs().amax(-1)
    # the norm's, the gate's and the type's own roundings
    tol = tol + (16 * 2.0 ** -24 + (0 if out.dtype == F32 else gd_plain.HALF_STEP[out.dtype])) * want.norm(dim=-1)
    tol = tol + gd_plain.LEAST[out.dtype] * want.shape[-1] ** 0.5  # (half a step of subnormal outputs)
    off = (out.double() - want).norm(dim=-1)
    worst = (off / tol.clamp(min=1e-300))[live]
    assert bool((off <= tol)[live].all()), (float(worst.max()), (worst == worst.max()).nonzero()[0].tolist())
    for slot, allowed in last.items():
        err = (state[slot].double() - held[slot]).norm(dim=1)
        assert bool((err <= allowed).all()), (slot, float((err / allowed.clamp(min=1e-300)).max()))


@pytest.mark.parametrize("decay", [-1e-3, -1.0, -20.0])
@pytest.mark.parametrize("kind,loud", [("f32", 1e4), ("f32", 1e7), ("f32", 1e12), ("bf16", 1e5), ("bf16", 1e9), ("f16", 1e4)])
def test_a_loud_token(kind, loud, decay):
    """One token's v many times the others': the ones before it are as exact as without it,
    and those behind it up to what it has left in the state."""
    print("[case]", kind, loud, decay, flush=True)
    for at in (0, 31, 70, 127):
        for norm in (False, True):
            c = Case(int(loud) % 1000 + at, [150], [True], dk=64, dv=32, kind=TYPES[kind], out=F32, gate=norm, norm=norm)
            c.decay[:], c.dt_bias[:] = decay, 0.5
            v = c.qkv[:, 2 * c.K * 64:]
            if kind == "f16":
                v.mul_(2.0 ** -6)
            v[at] *= loud
            check(c)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("b", [-12.0, -25.0, -60.0])
def test_heads_that_hardly_write(kind, b):
    """Write strengths of 1e-5 to 1e-26, into an empty state and into one of such a size."""
    for begin in (True, False):
        for new in ([9], [100]):
            c = Case(3, new, [begin], dk=128, dv=48, kind=TYPES[kind], out=F32, gate=False, norm=False)
            c.b[:] = b
            c.b[::7] = b - 5
            if not begin:
                c.state *= 2.0 ** -30
            check(c)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("fade", [-18.0, -40.0])
def test_a_large_state_that_is_forgotten(kind, fade):
    """A state of 1e7 and loud tokens that one strong decay wipes out; quiet tokens follow, in the same chunk and
    in the next one."""
    for at in (1, 20, 63, 64):
        c = Case(at, [140], [False], dk=64, dv=64, kind=TYPES[kind], out=F32, gate=False, norm=False)
        c.state *= 1e7
        c.decay[:], c.dt_bias[:] = -0.05, 0.0
        c.qkv[:at, 2 * c.K * 64:] *= 100
        c.a[at] = fade / -0.05  # softplus of so large a number is itself
        check(c)


def test_quiet_rows_of_keys_and_queries():
    """Rows of q and k of every size have unit length; the columns within a row differ by 1e6 too."""
    for kind in (F32, BF16):
        c = Case(11, [100], [False], dk=64, dv=32, kind=kind, out=F32, gate=False, norm=False)
        qk = c.qkv[:, :2 * c.K * 64]
        qk *= torch.logspace(-9, 9, 100)[:, None].to(kind)
        qk[:, ::8] *= 1e6
        check(c)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [64, 100])
@pytest.mark.parametrize("total", [-20.0, -50.0, -80.0])
def test_fades(kind, total, new):
    """What is left of a state after far decays, spread over a chunk or in one token of it: as exact as the state was."""
    for at in (None, 3, 40):
        c = Case(21, [new], [False], dk=64, dv=32, kind=TYPES[kind], out=F32, gate=False, norm=False)
        c.qkv[:, 2 * c.K * 64:] = 0
        c.b[:] = -30.0
        c.decay[:], c.dt_bias[:] = -1.0, 0.0
        c.a[:] = -80.0 if at is not None else torch.expm1(torch.tensor(-total / 64)).log()  # softplus: 0, or a 64th
        if at is not None:
            c.a[at] = -total
        check(c)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("new", [[9], [100], [100, 3]])
def test_rows_of_zeros_without_an_eps(kind, new):
    """A row of zeros stays one where l2_eps is 0 too, by steps and in chunks."""
    c = Case(17, new, [False] * len(new), dk=64, dv=32, kind=TYPES[kind], out=F32, gate=False, norm=False)
    K = c.K * 64
    c.qkv[2, :K] = 0
    c.qkv[4, K:2 * K] = 0
    c.qkv[-1, :2 * K] = 0
    # (as the definition's limit: 0 / sqrt(0 + 1e-300), which changes no other row in 64 bits)
    c.check(c.run(l2_eps=0.0), c.plain(l2_eps=1e-300))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("size,eps", [(1e24, 1e-6), (1e33, 1e-6), (1e33, 0.0), (1e-24, 0.0), (1e-33, 1e-38)])
@pytest.mark.parametrize("new,dv", [([6], 64), ([6], 112), ([100], 64), ([100, 3], 112)])
def test_norms_of_rows_of_any_size(kind, size, eps, new, dv):
    """Squares of the outputs pass fp32's range, at either end; the norm is the definition's."""
    c = Case(23, new, [False] * len(new), dk=64, dv=dv, kind=TYPES[kind], out=F32, size=size)
    c.check(c.run(norm_eps=eps), c.plain(eps=eps))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("size", [1e35, 1e-35])
@pytest.mark.parametrize("new", [[6], [150]])
def test_values_near_the_ends_of_the_range(kind, norm, size, new):
    """States and values of 10^35, whose products with keys of any scale do not pass fp32's range on the way, and 10^-35."""
    c = Case(29, new, [False], dk=128, dv=32, kind=TYPES[kind], out=F32, gate=False, norm=norm, size=size)
    check(c)
