"""Batches of the gated delta rule whose ranges do not fit: what is computed is the definition's on
the ranges as they are cut, and nothing beside the output's rows and the pool's slots is
written, by steps and in chunks."""
import pytest

import gd_plain
from test_gpu_gd_delta import Case, ints

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

GUARD = 3


def run(c, starts, lens, most):
    """(out, state, flags) with rows and slots around both that nothing may touch."""
    from inferno_hip import device as D
    T, n = c.qkv.shape[0], c.state.shape[0]
    out = torch.full((T + 2 * GUARD, *c.out.shape[1:]), -7.0, device="cuda")
    state = torch.full((n + 2 * GUARD, *c.state.shape[1:]), 5.0, device="cuda")
    state[GUARD:GUARD + n] = c.state.cuda()
    flags = ints([0])
    batch = D.StateBatch(ints(starts), ints(c.slots), T, kv_lens=None if lens is None else ints(lens), most=most)
    layer = D.DeltaLayer(state[GUARD:GUARD + n], c.K, c.decay.cuda(), c.dt_bias.cuda())
    D.gated_delta(*c.parts(c.qkv.cuda()), c.a.contiguous().cuda(), c.b.contiguous().cuda(), layer, batch, out=out[GUARD:GUARD + T],
                  flags=flags)
    for t, mark in ((out, -7.0), (state, 5.0)):
        assert bool((t[:GUARD] == mark).all()) and bool((t[-GUARD:] == mark).all())
    return out[GUARD:GUARD + T].cpu(), state[GUARD:GUARD + n].cpu(), int(flags.item())


@pytest.mark.parametrize("most", [0, 1])  # (chunks, and a token at a time)
@pytest.mark.parametrize("starts,lens,new,at", [
    ([0, 40, 99], None, [40, 20], [0, 40]),             # an end behind the rows
    ([0, 70, 99], None, [60, 0], [0, 60]),              # a start behind them
    ([-3, 40, 60], None, [40, 20], [0, 40]),            # a start before them
    ([0, 50, 20], None, [50, 0], [0, 50]),              # an end before the start
    ([-2 ** 31, 40, 2 ** 31 - 1], None, [40, 20], [0, 40]),
    ([0, 40, 60], [30, 50], [40, 20], [0, 40]),         # fewer tokens than new ones: the sequence begins
    ([0, 40, 60], [-5, -2 ** 31], [40, 20], [0, 40]),
])
def test_what_is_cut(starts, lens, new, at, most):
    from inferno_hip import _lib
    c = Case(11, [40, 20], [False, False], gate=False, norm=False)
    c.out = torch.full((60, 4, 64), -7.0)
    got, state, flags = run(c, starts, lens, most)
    assert flags == _lib.FLAG_KV_LENGTH
    begins = [lens is not None and m <= n for n, m in zip(new, lens or [0, 0])]
    y, held = gd_plain.delta(*c.parts(c.qkv), c.a, c.b, c.decay, c.dt_bias, c.state, new, begins, c.slots, at, c.out)
    for n, first, slot in zip(new, at, c.slots):
        if n:
            assert gd_plain.off(got[first:first + n], y[first:first + n]) <= gd_plain.NEAR
            assert gd_plain.off(state[slot], held[slot]) <= gd_plain.NEAR
        else:
            assert torch.equal(state[slot], c.state[slot])
    rows = torch.ones(60, dtype=torch.bool)
    for n, first in zip(new, at):
        rows[first:first + n] = False
    assert bool((got[rows] == -7).all())


@pytest.mark.parametrize("most", [0, 1])
def test_starts_that_decrease(most):
    """Sequences whose rows overlap: reported, and inside the buffers."""
    from inferno_hip import _lib
    c = Case(12, [40, 0, 20, 0], [False] * 4, gate=False, norm=False)
    for starts in ([0, 40, 20, 60, 60], [50, 10, 60, 0, 60], [60, 0, 60, 0, 60]):
        _, state, flags = run(c, starts, None, most)
        assert flags == _lib.FLAG_KV_LENGTH
        free = [s for s in range(6) if s not in c.slots]
        assert torch.equal(state[free], c.state[free])
