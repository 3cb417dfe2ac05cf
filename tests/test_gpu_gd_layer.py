"""A recurrent layer and the choice of a token as a serving loop runs them, with the
library's own projections around them: in-projections, short convolution, gated delta
rule with its norm and gate, output projection with the residual, lm_head, sampling; a
batch of prompts and then steps of one token, eagerly, captured in a graph and replayed
with new contents, from four threads, and on streams of their own."""
import threading

import pytest

import gd_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

K, H, DIM, HIDDEN, VOCAB, WIDTH = 2, 4, 64, 512, 3001, 4
CHANNELS = (2 * K + H) * DIM
# From the projections' outputs on: the convolution's roundings (2^-22 of a sum of five
# terms) reach k, q and v, each of which the rule then adds its own to.
NEAR = 4 * gd_plain.NEAR


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Model:
    def __init__(self):
        from inferno_hip import device as D
        from inferno_hip import synth
        rng = synth.rng_for(0x91)
        def weight(outer, inner):
            return D.DeviceWeight(torch.from_numpy(synth.weight(rng, synth.Q4_K, outer, inner)).cuda(), synth.Q4_K, inner, outer)
        g = torch.Generator().manual_seed(2)
        r = lambda *s: torch.randn(s, generator=g)
        self.qkv, self.z, self.wo, self.head = weight(CHANNELS, HIDDEN), weight(H * DIM, HIDDEN), weight(HIDDEN, H * DIM), weight(VOCAB, HIDDEN)
        self.ab, self.norm = (0.05 * r(2 * H, HIDDEN)).cuda(), torch.ones(HIDDEN, device="cuda")
        self.taps = (0.5 * r(CHANNELS, WIDTH)).cuda()
        self.decay, self.dt_bias = -torch.rand(H, generator=g).cuda() * 4, (r(H) - 3).cuda()
        self.norm_w = (1 + 0.1 * r(DIM)).cuda()

    def pools(self, slots):
        return torch.full((slots, WIDTH - 1, CHANNELS), float("nan"), device="cuda"), \
            torch.full((slots, H, DIM, DIM), float("nan"), device="cuda")

    def mix(self, x, ab, z, pools, batch, workspace=None, flags=None, stream=None, kind=torch.float32):
        """Convolution and delta rule of projected rows."""
        from inferno_hip import device as D
        y = D.short_conv(x, self.taps, pools[0], batch, out_dtype=kind, flags=flags, stream=stream)
        layer = D.DeltaLayer(pools[1], K, self.decay, self.dt_bias, norm_w=self.norm_w)
        q, k, v = y[:, :K * DIM], y[:, K * DIM:2 * K * DIM], y[:, 2 * K * DIM:]
        o = D.gated_delta(q.unflatten(1, (K, DIM)), k.unflatten(1, (K, DIM)), v.unflatten(1, (H, DIM)), ab[:, :H], ab[:, H:], layer,
                          batch, gate=z.view(-1, H, DIM), out_dtype=torch.float32, workspace=workspace, flags=flags, stream=stream)
        return y, o


@pytest.fixture(scope="module")
def model():
    return Model()


def plain(m, x, ab, z, n):
    """A whole sequence of one slot in 64 bits, from its projected rows."""
    f = lambda t: t.cpu()
    y, _, _ = gd_plain.conv(f(x), f(m.taps), None, True, torch.zeros(1, WIDTH - 1, CHANNELS), [n], [True], [0], [0],
                            torch.zeros(n, CHANNELS))
    q, k, v = y[:, :K * DIM].view(n, K, DIM), y[:, K * DIM:2 * K * DIM].view(n, K, DIM), y[:, 2 * K * DIM:].view(n, H, DIM)
    out, state = gd_plain.delta(q, k, v, f(ab)[:, :H], f(ab)[:, H:], f(m.decay), f(m.dt_bias), torch.zeros(1, H, DIM, DIM), [n],
                                [True], [0], [0], torch.zeros(n, H, DIM), norm_w=f(m.norm_w), gate=f(z).view(n, H, DIM))
    return out, state[0]


def test_prompts_and_then_tokens(model):
    from inferno_hip import device as D
    m, g = model, torch.Generator().manual_seed(5)
    new, slots = [90, 7, 150], [4, 0, 2]
    T = sum(new)
    X = torch.randn(T, HIDDEN, generator=g).cuda()
    x, z, ab = D.prefill_q4_k_f32(m.qkv, X), D.prefill_q4_k_f32(m.z, X), X @ m.ab.t()
    pools, flags = m.pools(5), ints([0])
    lens = ints(new)
    starts = ints([0, 90, 97, 247])
    _, o = m.mix(x, ab, z, pools, D.StateBatch(starts, ints(slots), T, kv_lens=lens, most=150), flags=flags)
    seqs = []
    for i, n in enumerate(new):
        a = int(starts[i])
        seqs.append([[t[a:a + n]] for t in (x, ab, z)])
        want, state = plain(m, x[a:a + n], ab[a:a + n], z[a:a + n], n)
        assert gd_plain.off(o[a:a + n], want) <= NEAR and gd_plain.off(pools[1][slots[i]], state) <= NEAR
    # one token a sequence at a time, each the embedding of the one that was chosen
    table = torch.randn(VOCAB, HIDDEN, generator=g).cuda()
    tokens = torch.zeros(3, dtype=torch.long, device="cuda")
    starts = ints([0, 1, 2, 3])
    temperature, top_k = torch.tensor([0.8, 0.0, 1.2], device="cuda"), ints([40, 0, 0])
    top_p, min_p = torch.tensor([0.95, 1.0, 0.8], device="cuda"), torch.tensor([0.0, 0.0, 0.05], device="cuda")
    for step in range(6):
        e = table[tokens]
        lens += 1
        x, z = (torch.stack([D.gemv_norm(w, m.norm, 1e-6, e[i].contiguous()) for i in range(3)]) for w in (m.qkv, m.z))
        ab = e @ m.ab.t()
        _, o = m.mix(x, ab, z, pools, D.StateBatch(starts, ints(slots), 3, kv_lens=lens, most=1), flags=flags)
        logits = torch.stack([D.gemv(m.head, D.gemv_add(m.wo, o[i].reshape(-1), e[i].clone())) for i in range(3)])
        u = torch.rand(3, generator=g)
        got = D.sample(logits, u.cuda(), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        for i in range(3):
            for part, t in zip(seqs[i], (x, ab, z)):
                part.append(t[i:i + 1])
            whole = [torch.cat(p) for p in seqs[i]]
            want, state = plain(m, *whole, whole[0].shape[0])
            assert gd_plain.off(o[i], want[-1]) <= NEAR and gd_plain.off(pools[1][slots[i]], state) <= NEAR, (step, i)
            token, _, _ = gd_plain.sample(logits[i].cpu().double().numpy(), float(u[i]), float(temperature[i]), int(top_k[i]),
                                          float(top_p[i]), float(min_p[i]))
            assert int(got[i]) == token
        tokens = got.long()
    assert int(flags.item()) == 0
    assert bool(torch.isnan(pools[1][[1, 3]]).all()) and bool(torch.isnan(pools[0][[1, 3]]).all())


class Step:
    """Buffers of one caller: sequences whose rows, states and settings change from call to call."""

    def __init__(self, m, seed, sequences, tokens, vocab, kind):
        self.m, self.kind, self.n, self.tokens = m, kind, sequences, tokens
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")
        self.x, self.ab, self.z = z(tokens, CHANNELS), z(tokens, 2 * H), z(tokens, H * DIM)
        self.pools0 = z(sequences + 1, WIDTH - 1, CHANNELS), z(sequences + 1, H, DIM, DIM)
        self.pools = tuple(t.clone() for t in self.pools0)
        self.starts, self.slots, self.lens = (z(n, t=torch.int32) for n in (sequences + 1, sequences, sequences))
        self.logits, self.u, self.t, self.p = z(sequences, vocab), z(sequences), z(sequences), z(sequences)
        self.k, self.flags = z(sequences, t=torch.int32), z(1, t=torch.int32)
        from inferno_hip import device as D
        self.batch = D.StateBatch(self.starts, self.slots, tokens, kv_lens=self.lens)
        layer = D.DeltaLayer(self.pools[1], K, m.decay, m.dt_bias)
        self.delta_ws, self.sample_ws = D.delta_workspace(layer, self.batch, kind), D.sample_workspace(sequences, vocab)
        self.contents()

    def contents(self):
        g = self.g
        for t in (self.x, self.ab, self.z, *self.pools0):
            t.normal_(generator=g)
        cuts = torch.randint(0, self.tokens + 1, (self.n - 1,), generator=g, device="cuda").sort()[0].int()
        self.starts[1:self.n], self.starts[self.n] = cuts, self.tokens
        self.slots.copy_(torch.randperm(self.n + 1, generator=g, device="cuda")[:self.n])
        self.lens.copy_(self.starts[1:] - self.starts[:-1] + torch.randint(0, 2, (self.n,), generator=g, device="cuda"))
        self.logits.normal_(std=3.0, generator=g)
        self.u.uniform_(generator=g)
        self.t.uniform_(0.3, 1.5, generator=g)
        self.p.uniform_(0.5, 1.0, generator=g)
        self.k.random_(0, 60, generator=g)
        self.fresh()

    def fresh(self):
        for a, b in zip(self.pools, self.pools0):
            a.copy_(b)
        self.flags.zero_()

    def run(self, stream=None, alone=False):
        from inferno_hip import device as D
        y, o = self.m.mix(self.x, self.ab, self.z, self.pools, self.batch, workspace=None if alone else self.delta_ws, flags=self.flags,
                          stream=stream, kind=self.kind)
        ws = None if alone else self.sample_ws
        one = D.sample(self.logits, self.u, temperature=self.t, top_k=self.k, top_p=self.p, workspace=ws, stream=stream)
        two = D.sample(self.logits, self.u, temperature=self.t, workspace=ws, stream=stream)
        return [y, o, one, two, *self.pools, self.flags]


def same(got, want):
    for i, (a, b) in enumerate(zip(got, want)):
        if a.is_floating_point():
            a, b = a.view(torch.int16 if a.element_size() == 2 else torch.int32), b.view(torch.int16 if b.element_size() == 2 else torch.int32)
        assert torch.equal(a, b), i


# single tokens; a few; chunks; one sequence
SIZES = [(5, 5, 3001, torch.float32), (9, 60, 20000, torch.bfloat16), (3, 400, 9001, torch.float32), (1, 130, 700, torch.float16)]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s[:3])))
def test_a_captured_step_replays_with_new_contents(model, sizes):
    print("[case]", sizes, flush=True)
    s = Step(model, sum(sizes[:3]), *sizes)
    s.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = s.run()
    other = torch.randn(512, 512, device="cuda")
    for _ in range(4):
        s.contents()
        want = [t.clone() for t in s.run()]
        torch.cuda.synchronize()
        s.fresh()
        for t in outs[:4]:
            t.fill_(-77)
        (other @ other).sum().item()  # the program's own work, and a wait, between replays
        graph.replay()
        torch.cuda.synchronize()
        same(outs, want)
        assert int(s.flags.item()) == 0


def test_steps_from_threads_on_their_own_streams(model):
    steps = [Step(model, 50 + i, *sizes) for i, sizes in enumerate(SIZES)]
    want = []
    for s in steps:
        s.fresh()
        want.append([t.clone() for t in s.run()])
    torch.cuda.synchronize()
    kept, errors = [[] for _ in steps], []

    def caller(i):
        try:
            s, side = steps[i], torch.cuda.Stream()
            with torch.cuda.stream(side):
                for r in range(12):
                    s.fresh()
                    kept[i].append([t.clone() for t in s.run(stream=side if r % 2 else None, alone=r % 3 == 2)])
            side.synchronize()
        except BaseException as e:  # reported after the join
            errors.append(e)
    threads = [threading.Thread(target=caller, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    for i in range(len(steps)):
        for got in kept[i]:
            same(got, want[i])


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "-".join(map(str, s[:3])))
def test_another_stream_while_the_current_one_is_behind(model, sizes):
    """What a call on a stream allocates is not what the current stream still has to write."""
    from test_gpu_kv_streams import behind
    s = Step(model, 7, *sizes)
    s.fresh()
    want = [t.clone() for t in s.run()]
    held = [t.numel() * t.element_size() for t in want[:4]] + [t.numel() for t in (s.delta_ws, s.sample_ws) if t is not None]
    side = torch.cuda.Stream()
    for _ in range(2):
        s.fresh()
        torch.cuda.synchronize()
        behind(held)
        got = s.run(stream=side, alone=True)
        torch.cuda.synchronize()
        same(got, want)


def test_wrappers_refuse(model):
    from inferno_hip import device as D
    from inferno_hip._lib import IHIPArgumentError
    s = Step(model, 3, *SIZES[0])
    conv = lambda **kw: D.short_conv(**{**dict(x=s.x, weight=model.taps, state=s.pools[0], batch=s.batch), **kw})
    layer = D.DeltaLayer(s.pools[1], K, model.decay, model.dt_bias)
    q = torch.zeros(5, K, DIM, device="cuda")
    delta = lambda **kw: D.gated_delta(**{**dict(q=q, k=q, v=torch.zeros(5, H, DIM, device="cuda"), a=s.ab[:, :H], b=s.ab[:, H:],
                                                 layer=layer, batch=s.batch), **kw})
    conv(), delta()
    for bad in (dict(x=s.x[:4]), dict(x=s.x.double()), dict(x=s.x.t()), dict(weight=model.taps[:, :3]), dict(weight=model.taps.cpu()),
                dict(state=s.pools[0].half()), dict(state=s.pools[0][:, :2]), dict(state=s.pools[0].cpu()),
                dict(bias=torch.zeros(3, device="cuda")), dict(out=torch.zeros(5, 8, device="cuda")),
                dict(out=torch.zeros(5, CHANNELS, device="cuda"), out_dtype=torch.float16), dict(x=s.x[:, ::2])):
        with pytest.raises(IHIPArgumentError):
            conv(**bad)
    for bad in (dict(q=q.half()), dict(k=q[:, :1]), dict(v=q), dict(a=s.ab), dict(b=s.ab[:, H:].half()), dict(gate=q),
                dict(out_dtype=torch.float16), dict(q=q[:4]), dict(workspace=torch.zeros(4, device="cuda"))):
        with pytest.raises(IHIPArgumentError):
            delta(**bad)
    for bad in (dict(state=s.pools[1][0]), dict(state=s.pools[1].transpose(2, 3)), dict(decay=model.decay[:2]),
                dict(norm_w=torch.zeros(3, device="cuda"))):
        with pytest.raises(IHIPArgumentError):
            D.DeltaLayer(**{**dict(state=s.pools[1], k_heads=K, decay=model.decay, dt_bias=model.dt_bias), **bad})
    with pytest.raises(IHIPArgumentError):
        D.StateBatch(s.starts, s.slots[:3], 5)
    with pytest.raises(IHIPArgumentError):
        D.StateBatch(s.starts.long(), s.slots, 5)
    for bad in (dict(logits=s.logits[0]), dict(logits=s.logits.t()), dict(logits=s.logits.double()), dict(u=s.u[:2]),
                dict(top_k=s.p), dict(temperature=s.t.cpu()), dict(logprobs=torch.zeros(2, device="cuda")),
                dict(workspace=torch.zeros(8, dtype=torch.uint8, device="cuda")), dict(logits=s.logits[:, :0])):
        with pytest.raises(IHIPArgumentError):
            D.sample(**{**dict(logits=s.logits, u=s.u), **bad})
    assert D.sample(s.logits[:0], s.u[:0]).numel() == 0
