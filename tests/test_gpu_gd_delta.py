"""The gated delta rule against its definition in 64 bits, a token after the other:
lengths around a chunk, head widths and groups, types, gates, states that begin and go
on, sizes of values, slots that no sequence may touch."""
import pytest

import gd_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts_of(new, first=0):
    s = [first]
    for n in new:
        s.append(s[-1] + n)
    return s


class Case:
    def __init__(self, seed, new, begins, K=2, H=4, dk=64, dv=64, kind=F32, out=None, gate=True, norm=True, first=0, pad=0,
                 size=1.0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.begins, self.K = new, begins, K
        self.starts = starts_of(new, first)
        T, n = self.starts[-1] + pad, len(new)
        x = torch.randn(T, 2 * K * dk + H * dv + 8, generator=g) * spread
        x = x * torch.sigmoid(x)
        x[:, 2 * K * dk:] *= size
        self.qkv = x.to(kind)
        ab = torch.randn(T, 2 * H + 3, generator=g)
        self.a, self.b = ab[:, :H], ab[:, H:2 * H]
        self.decay, self.dt_bias = -torch.rand(H, generator=g) * 4, torch.randn(H, generator=g) - 3
        self.gate = torch.randn(T, H, dv, generator=g) if gate else None
        self.norm_w = 1 + 0.1 * torch.randn(dv, generator=g) if norm else None
        self.slots = torch.randperm(n + 2, generator=g)[:n].tolist()
        self.state = 0.3 * size * torch.randn(n + 2, H, dk, dv, generator=g)
        for s, b in zip(self.slots, begins):
            if b:
                self.state[s] = float("nan")
        self.out = torch.full((T, H, dv), -7.0).to(out or kind)
        self.shape = (K, H, dk, dv)

    def parts(self, x):
        K, H, dk, dv = self.shape
        T = x.shape[0]
        return (x[:, :K * dk].view(T, K, dk) if x.is_contiguous() else x[:, :K * dk].unflatten(1, (K, dk)),
                x[:, K * dk:2 * K * dk].unflatten(1, (K, dk)), x[:, 2 * K * dk:2 * K * dk + H * dv].unflatten(1, (H, dv)))

    def plain(self, slots=None, **kw):
        return gd_plain.delta(*self.parts(self.qkv), self.a, self.b, self.decay, self.dt_bias, self.state, self.new, self.begins,
                              slots or self.slots, self.starts, self.out, norm_w=self.norm_w, gate=self.gate, **kw)

    def run(self, most=0, slots=None, lens=True, **kw):
        from inferno_hip import device as D
        dev = lambda t: None if t is None else t.cuda()
        state, out, flags = self.state.cuda(), self.out.cuda(), ints([0])
        lens = ints([n if b else n + 9 for n, b in zip(self.new, self.begins)]) if lens else None
        batch = D.StateBatch(ints(self.starts), ints(slots or self.slots), self.qkv.shape[0], kv_lens=lens, most=most)
        layer = D.DeltaLayer(state, self.K, dev(self.decay), dev(self.dt_bias), norm_w=dev(self.norm_w), **kw)
        ws = D.delta_workspace(layer, batch, self.qkv.dtype)
        if ws is not None:
            ws.fill_(255)  # NaN, wherever something is read that was not written
        ab = torch.cat((self.a, self.b), 1).cuda()
        H = self.shape[1]
        D.gated_delta(*self.parts(self.qkv.cuda()), ab[:, :H], ab[:, H:], layer, batch, gate=dev(self.gate), out=out,
                      workspace=ws, flags=flags)
        return out.cpu(), state.cpu(), int(flags.item())

    def check(self, got, want, near=gd_plain.NEAR):
        """The rows and states of every head of every sequence; what is no sequence's, bit for bit."""
        out, state, _ = got
        y, held = want
        u = 0.0 if out.dtype == F32 else gd_plain.HALF_STEP[out.dtype]
        for n, at, slot in zip(self.new, self.starts, self.slots):
            for h in range(self.shape[1]):
                if n:
                    # (a rounding of half a step at most, of every value)
                    assert gd_plain.off(out[at:at + n, h], y[at:at + n, h]) <= near + u, (n, h, "out")
                    assert gd_plain.off(state[slot, h], held[slot, h]) <= near, (n, h, "state")
        rows = torch.ones(out.shape[0], dtype=torch.bool)
        rows[self.starts[0]:self.starts[-1]] = False
        assert bool((out[rows] == -7).all())
        free = [s for s in range(state.shape[0]) if s not in [x for x, n in zip(self.slots, self.new) if n]]
        assert torch.equal(state[free].nan_to_num(9.0), self.state[free].nan_to_num(9.0))


@pytest.mark.parametrize("kind,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (128, 64), (64, 128), (16, 16), (80, 112), (48, 96), (112, 32)])
def test_lengths_types_and_widths(dk, dv, kind, out):
    """One token to two chunks in one batch: those of few tokens go a token at a time, the others in chunks."""
    print("[case]", dk, dv, kind, out, flush=True)
    new = [1, 0, 17, 16, 64, 65, 130, 2, 63]
    c = Case(dk + dv, new, [i % 3 == 0 for i in range(len(new))], dk=dk, dv=dv, kind=TYPES[kind], out=TYPES[out], first=3, pad=5)
    got = c.run()
    c.check(got, c.plain())
    assert got[2] == 0


@pytest.mark.parametrize("K,H", [(1, 1), (1, 8), (3, 3), (5, 15), (16, 16)])
@pytest.mark.parametrize("new", [[1, 1, 1], [100, 70]])
def test_head_groups(K, H, new):
    c = Case(K * H, new, [False] * len(new), K=K, H=H, dk=32, dv=48, gate=False, norm=False)
    c.check(c.run(), c.plain())


@pytest.mark.parametrize("gate,norm", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_epilogues(kind, gate, norm):
    for new in ([3, 9], [90, 5]):
        c = Case(7, new, [True, False], kind=TYPES[kind], gate=gate, norm=norm)
        c.check(c.run(), c.plain())


@pytest.mark.parametrize("H", [1, 6, 16])
def test_lengths_beside_the_ones_that_go_a_token_at_a_time(H):
    """Up to 4 or 10 beside longer ones; alone up to 10 to 32, by the numbers of heads and sequences."""
    for new in ([3, 4, 5, 33] * 5, [9, 10, 11, 12, 15, 16, 31, 32, 33, 34], [9, 10, 1], [9, 1, 11], [32, 31, 9, 10, 11, 1, 2, 8], [33, 32]):
        c = Case(H, new, [i % 2 == 0 for i in range(len(new))], K=1, H=H, dk=64, dv=32)
        c.check(c.run(), c.plain())
        c.check(c.run(most=max(new)), c.plain())


@pytest.mark.parametrize("most", [1, 4, 16, 17, 200, 1 << 20])
def test_any_hint_gives_the_same_results(most):
    """`most` chooses kernels; the states of either way are the same to rounding."""
    c = Case(5, [40, 1, 150], [True, False, False])
    c.check(c.run(most=most), c.plain())


@pytest.mark.parametrize("new", [[1], [5], [16], [17], [64], [300]])
def test_one_sequence(new):
    for begin in (False, True):
        c = Case(sum(new), new, [begin], dk=128, dv=128)
        c.check(c.run(), c.plain())
        c.check(c.run(most=sum(new)), c.plain())


def test_every_sequence_goes_on_without_lengths():
    c = Case(4, [20, 3], [False, False])
    c.check(c.run(lens=False), c.plain())


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("size", [1e-4, 3e3])
@pytest.mark.parametrize("new", [[6], [100]])
def test_sizes_of_values(size, kind, new):
    c = Case(2, new, [False], kind=TYPES[kind], size=size, out=F32, norm=False)
    c.check(c.run(), c.plain())


@pytest.mark.parametrize("size", [1e-30, 1e30])
@pytest.mark.parametrize("new", [[6], [100]])
def test_sizes_of_fp32_values(size, new):
    c = Case(2, new, [False], size=size, norm=False, gate=False)
    c.check(c.run(), c.plain())


@pytest.mark.parametrize("new", [[9], [100]])
def test_sizes_of_keys(new):
    """q and k of any size have unit length: as small as eps allows, as large as fp32 does; a row of zeros stays one."""
    c = Case(3, new, [False], dk=64, dv=32)
    for r, f in ((1, 1e30), (2, 1e-12), (3, 0.0), (4, 1e18), (5, 1e-38)):
        c.qkv[r, :2 * c.K * 64] *= f
    c.check(c.run(), c.plain())


@pytest.mark.parametrize("new", [[9], [100]])
def test_decays_and_strengths_at_their_ends(new):
    c = Case(6, new, [False], norm=False, gate=False)
    for r, (a, b) in enumerate([(60.0, 90.0), (-90.0, -90.0), (3e4, 0.0), (-3e38, 3e38), (1e30, -3e38), (0.0, 0.0)]):
        c.a[r], c.b[r] = a, b
    c.decay[0] = 0.0     # forgets nothing
    c.decay[1] = 5.0     # would grow: counts as 0
    c.decay[2] = -1e9
    c.check(c.run(), c.plain())


def test_keys_that_repeat():
    """The same key in every token (the triangular inverse at its largest), fully written and hardly forgotten."""
    for kind in (F32, BF16):
        c = Case(8, [128], [False], kind=kind, out=F32, norm=False, gate=False)
        c.qkv[:, :4 * 64] = c.qkv[0, :4 * 64]
        c.b[:], c.decay[:] = 20.0, -1e-4
        c.check(c.run(), c.plain())


def test_scale_and_eps():
    c = Case(9, [70, 3], [True, False], norm=True)
    c.check(c.run(scale=0.5, l2_eps=0.5, norm_eps=0.25), c.plain(scale=0.5, l2_eps=0.5, eps=0.25))
    c = Case(9, [70, 3], [True, False], norm=False)
    c.check(c.run(scale=-2.0, l2_eps=0.0), c.plain(scale=-2.0, l2_eps=0.0))


@pytest.mark.parametrize("new", [[4, 4, 4], [40, 40, 40]])
def test_slots_that_are_not_a_sequences_own(new):
    from inferno_hip import _lib
    for slots, left_out in (([0, 1, 0], [2]), ([0, 5, 1], [1]), ([-1, 1, 2], [0]), ([1, 1, 1], [1, 2])):
        c = Case(1, new, [False] * 3)
        out, state, flags = c.run(slots=slots)
        y, held = c.plain(slots=[-1 if i in left_out else s for i, s in enumerate(slots)])
        assert flags == _lib.FLAG_STATE_SLOT
        assert gd_plain.off(out, y) <= gd_plain.NEAR and gd_plain.off(state, held) <= gd_plain.NEAR
        for i in left_out:
            assert bool((out[c.starts[i]:c.starts[i + 1]] == -7).all())
    # a sequence without new tokens holds nothing
    c = Case(1, [0, new[0], new[0]], [False] * 3)
    out, state, flags = c.run(slots=[2, 2, 1])
    y, held = c.plain(slots=[2, 2, 1])
    assert flags == 0 and gd_plain.off(out, y) <= gd_plain.NEAR and gd_plain.off(state, held) <= gd_plain.NEAR


@pytest.mark.parametrize("new", [[5, 6], [90, 200]])
def test_a_nan_stays_in_its_head_and_sequence(new):
    c = Case(10, new, [True, False], gate=False, norm=False)
    y, held = c.plain()
    where = c.starts[1] + new[1] - 1  # the second sequence's last token, first head of v
    c.qkv[where, 2 * c.K * 64 + 3] = float("nan")
    out, state, _ = c.run()
    chunk = c.starts[1] + (new[1] - 1) // 64 * 64  # (the 64 that go together share it)
    assert gd_plain.off(out[:chunk], y[:chunk]) <= gd_plain.NEAR
    assert gd_plain.off(out[:, 1:], y[:, 1:]) <= gd_plain.NEAR
    assert bool(torch.isnan(out[where, 0, 3])) and bool(torch.isnan(state[c.slots[1], 0, :, 3]).all())
    assert gd_plain.off(state[c.slots[0]], held[c.slots[0]]) <= gd_plain.NEAR


def test_ranges_that_do_not_fit_are_cut():
    from inferno_hip import _lib
    for starts in ([0, 40, 99], [-3, 40, 60], [0, 50, 20]):
        c = Case(11, [40, 20], [False, False])
        c.starts = starts
        out, state, flags = c.run()
        assert flags & _lib.FLAG_KV_LENGTH and out.shape[0] == 60
    # more new tokens than tokens: the sequence begins
    c = Case(11, [40, 20], [False, False])
    from inferno_hip import device as D
    flags = ints([0])
    state = c.state.cuda()
    batch = D.StateBatch(ints(c.starts), ints(c.slots), 60, kv_lens=ints([30, 50]))
    layer = D.DeltaLayer(state, c.K, c.decay.cuda(), c.dt_bias.cuda())
    q, k, v = c.parts(c.qkv.cuda())
    D.gated_delta(q, k, v, c.a.contiguous().cuda(), c.b.contiguous().cuda(), layer, batch, flags=flags)
    assert int(flags.item()) & _lib.FLAG_KV_LENGTH


def test_a_long_sequence_in_steps_and_in_one():
    """700 tokens at once, in chunks of odd lengths, and the last ones a token at a time."""
    c = Case(12, [700], [True], dk=128, dv=128, K=1, H=2)
    y, held = c.plain()
    c.check(c.run(), (y, held))
    from inferno_hip import device as D
    state, out = c.state.cuda(), c.out.cuda()
    layer = D.DeltaLayer(state, c.K, c.decay.cuda(), c.dt_bias.cuda(), norm_w=c.norm_w.cuda())
    qkv, a, b, gate = c.qkv.cuda(), c.a.contiguous().cuda(), c.b.contiguous().cuda(), c.gate.cuda()
    at = 0
    for n in [201, 64, 333, 90] + [1] * 12:
        batch = D.StateBatch(ints([0, n]), ints(c.slots), n, kv_lens=ints([at + n]))
        D.gated_delta(*c.parts(qkv[at:at + n]), a[at:at + n], b[at:at + n], layer, batch, gate=gate[at:at + n], out=out[at:at + n])
        at += n
    assert at == 700
    c.check((out.cpu(), state.cpu(), 0), (y, held))
