"""The paged-cache operators as a decoder layer's attention half uses them, with
the library's own projections around them: norm folded into the grouped
wq/wk/wv GEMV, norms + rotary + append, attention, wo with the residual; a
prompt through the prefill, decode steps one token at a time, forked sequences
and a compacted pool in between."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

H, HK, DIM, HIDDEN, PAGE = 8, 2, 64, 1024, 16
WIDTH = (H + 2 * HK) * DIM
# The plain form rounds keys and values to fp16 after 64 bits, the kernel after 32:
# near a border they fall on neighbours, 2^-10 of the value apart.  With normed
# heads (norms of 1 +- 0.3 each) sum |q k| / sqrt(dim) <= 1.3^2 * 8 = 14, so a score
# is off by at most 14 * 2^-10 and an average by twice that, 2.7 %, if every key of
# a row fell wrong; 2 % of the largest value leaves out the values' own 2^-10.
NEAR = 2e-2


@pytest.fixture(scope="module")
def layer():
    from inferno_hip import device as D
    from inferno_hip import synth
    rng = synth.rng_for(0x71)
    def weight(outer, inner):
        return D.DeviceWeight(torch.from_numpy(synth.weight(rng, synth.Q4_K, outer, inner)).cuda(), synth.Q4_K, inner, outer)
    g = torch.Generator().manual_seed(2)
    f = dict(qkv=weight(WIDTH, HIDDEN), wo=weight(HIDDEN, H * DIM), norm=torch.ones(HIDDEN, device="cuda"),
             qn=(1 + 0.1 * torch.randn(DIM, generator=g)).cuda(), kn=(1 + 0.1 * torch.randn(DIM, generator=g)).cuda())
    f["turns"], f["m"] = D.rope_turns(DIM, 1e6)
    return f


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def attend(f, qkv, cache, batch, ws=None, out=None):
    from inferno_hip import device as D
    x = qkv.view(-1, H + 2 * HK, DIM)
    q = D.rope_kv(x[:, :H], x[:, H:H + HK], x[:, H + HK:], f["turns"], cache, batch, mscale=f["m"], q_norm=f["qn"], k_norm=f["kn"])
    return D.attn_paged(q, cache, batch, workspace=ws, out=out)


def plain(f, qkv, n):
    """The attention of a whole sequence in 64 bits: n x (heads * dim)."""
    x = qkv.double().cpu().view(n, H + 2 * HK, DIM)
    def normed(x, w):
        return x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double().cpu()
    t = torch.arange(n).double()[:, None] * f["turns"].cpu()
    c, s = (2 * torch.pi * t).cos()[:, None], (2 * torch.pi * t).sin()[:, None]
    def turned(x):
        a, b = x.chunk(2, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1)
    q, k, v = turned(normed(x[:, :H], f["qn"])), turned(normed(x[:, H:H + HK], f["kn"])), x[:, H + HK:]
    k, v = k.half().double(), v.half().double()
    out = torch.empty(n, H, DIM, dtype=torch.float64)
    hidden = torch.ones(n, n).triu(1).bool()
    for h in range(H):
        z = (q[:, h] @ k[:, h // (H // HK)].T * DIM ** -0.5).masked_fill(hidden, -torch.inf)
        out[:, h] = z.softmax(1) @ v[:, h // (H // HK)]
    return out.reshape(n, H * DIM)


def test_prompt_decode_fork_and_compaction(layer):
    from inferno_hip import device as D
    f = layer
    g = torch.Generator().manual_seed(3)
    pages = 64
    cache = D.KVCache(torch.full((pages, HK, PAGE, DIM), float("nan"), dtype=torch.float16, device="cuda"),
                      torch.full((pages, HK, PAGE, DIM), float("nan"), dtype=torch.float16, device="cuda"))
    refs, flags = torch.zeros(pages, dtype=torch.int32, device="cuda"), ints([0])
    refs[::2] = 1  # something else holds every other page for now
    steps = 9
    prompt = torch.randn(21, HIDDEN, generator=g).cuda()
    # two sequences out of nothing, room for the prompt
    table, lens, _ = D.kv_fork(torch.full((1, 12), -1, dtype=torch.int32, device="cuda"), ints([0]), ints([-1, -1]), refs, PAGE, room=21,
                               flags=flags)
    chunk = [21, 13]
    X = torch.cat((prompt, prompt[:13]))
    qkv = D.prefill_q4_k_f32(f["qkv"], X.contiguous())
    lens = ints(chunk)
    batch = D.KVBatch(ints([0, 21, 34]), lens, table, 34)
    got = attend(f, qkv, cache, batch)
    seqs = [[qkv[:21]], [qkv[21:]]]
    for s, (a, b) in enumerate(((0, 21), (21, 34))):
        want = plain(f, qkv[a:b], b - a)
        assert float((got[a:b].reshape(b - a, -1).cpu().double() - want).abs().max()) < NEAR * float(want.abs().max())
    # decode: the first sequence goes on three ways, the second once
    parents = [0, 0, 1, 0]
    for step in range(steps):
        table, lens, copies = D.kv_fork(table, lens, ints(parents), refs, PAGE, room=1, flags=flags)
        D.kv_copy(cache, copies, flags=flags)
        if step == 4:  # the other holder lets go, and the pool is compacted
            refs[::2] -= 1
            moves, moved = D.kv_compact(table, refs, flags=flags)
            D.kv_copy(cache, moves, moved, flags=flags)
            used = int((refs > 0).sum())
            assert int(table.max()) < used and int(moved.item()) > 0
        seqs = [list(seqs[p]) for p in parents]
        parents = [0, 1, 2, 3]
        lens = lens + 1
        x = torch.randn(4, HIDDEN, generator=g).cuda()
        rows = torch.stack([D.gemv_norm(f["qkv"], f["norm"], 1e-6, x[i]) for i in range(4)])
        batch = D.KVBatch(ints([0, 1, 2, 3, 4]), lens, table, 4)
        a = attend(f, rows, cache, batch)
        y = [D.gemv_add(f["wo"], a[i].reshape(-1), x[i].clone()) for i in range(4)]
        for i in range(4):
            seqs[i].append(rows[i:i + 1])
            whole = torch.cat(seqs[i])
            want = plain(f, whole, whole.shape[0])[-1]
            got = a[i].reshape(-1).cpu().double()
            assert float((got - want).abs().max()) < NEAR * float(want.abs().max()), (step, i)
            assert bool(torch.isfinite(y[i]).all())
    assert int(flags.item()) == 0
    assert sorted(lens.tolist()) == [13 + steps, 21 + steps, 21 + steps, 21 + steps]


def test_a_captured_decode_step_replays(layer):
    """norm + wq/wk/wv, rope + append, attention and wo of one token as a graph whose length and token change."""
    from inferno_hip import device as D
    f = layer
    n = 40
    def fresh():
        c = D.KVCache(torch.zeros(8, HK, PAGE, DIM, dtype=torch.float16, device="cuda"),
                      torch.zeros(8, HK, PAGE, DIM, dtype=torch.float16, device="cuda"))
        return c, ints([0])
    table = ints([[7, 2, 5, 0, 1, 3, 4, 6]])
    xs = torch.randn(n, HIDDEN, generator=torch.Generator().manual_seed(4)).cuda()

    def step(x, cache, batch, q, rows, a, y, ws):
        D.gemv_norm(f["qkv"], f["norm"], 1e-6, x, out=rows)
        r = rows.view(1, H + 2 * HK, DIM)
        D.rope_kv(r[:, :H], r[:, H:H + HK], r[:, H + HK:], f["turns"], cache, batch, q_norm=f["qn"], k_norm=f["kn"], out=q)
        D.attn_paged(q, cache, batch, out=a, workspace=ws)
        D.gemv_add(f["wo"], a.view(-1), x, out=y)

    def buffers(cache, batch):
        return (torch.empty(1, H, DIM, device="cuda"), torch.empty(WIDTH, device="cuda"), torch.empty(1, H, DIM, device="cuda"),
                torch.empty(HIDDEN, device="cuda"), D.attn_workspace(H, cache, batch))
    eager, lens_e = fresh()
    batch_e = D.KVBatch(ints([0, 1]), lens_e, table, 1)
    be = buffers(eager, batch_e)
    want = []
    for i in range(n):
        lens_e.fill_(i + 1)
        step(xs[i].contiguous(), eager, batch_e, *be)
        want.append(be[3].clone())
    cache, lens = fresh()
    batch = D.KVBatch(ints([0, 1]), lens, table, 1)
    b, x = buffers(cache, batch), xs[0].clone()
    lens.fill_(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(x, cache, batch, *b)
    for i in range(n):
        lens.fill_(i + 1)
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(b[3], want[i]), i
    assert torch.equal(cache.k, eager.k) and torch.equal(cache.v, eager.v)
