"""The paged-cache calls as a step of a serving loop makes them, captured in a graph
and replayed with new contents, and from four threads at once: forks and their page
copies, compaction and its copies, rope with the append, attention.  Every result
equals an eager, serial call's bit for bit."""
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

F16, BF16 = torch.float16, torch.bfloat16
HEADS, KV, DIM, PAGE = 8, 2, 64, 16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Step:
    """Buffers of one caller: `sequences` parents of which `children` go on, each with `new` tokens."""

    def __init__(self, seed, sequences, children, longest, new, kv, layers=2):
        from inferno_hip import device as D
        self.new, self.children, self.sequences = new, children, sequences
        self.width = -(-(longest + new) // PAGE) + 1
        per = self.width * sequences
        self.pages = per + children * (-(-new // PAGE) + 1) + 5
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.longest = g, longest
        self.lens, self.parents = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (sequences, children))
        self.table = torch.zeros(sequences, self.width, dtype=torch.int32, device="cuda")
        self.refs0 = torch.zeros(self.pages, dtype=torch.int32, device="cuda")
        self.k0, self.v0 = (torch.randn(layers, self.pages, KV, PAGE, DIM, generator=g, device="cuda").to(kv) for _ in range(2))
        self.cache = D.KVCache(self.k0.clone(), self.v0.clone())
        self.layer = self.cache.layer(1)
        self.x = torch.zeros(children * new, HEADS + 2 * KV, DIM, device="cuda")
        self.turns, self.mscale = D.rope_turns(DIM, 1e4)
        self.starts = ints([new * i for i in range(children + 1)])
        self.flags = torch.zeros(1, dtype=torch.int32, device="cuda")
        probe = D.KVBatch(self.starts, torch.zeros_like(self.parents), torch.zeros(children, self.width, dtype=torch.int32, device="cuda"),
                          children * new)
        self.workspace = D.attn_workspace(HEADS, self.layer, probe)
        self.refs = self.refs0.clone()

    def contents(self):
        """New lengths, tables, parents and projections; the pools as they were."""
        order = torch.randperm(self.pages, generator=self.g, device="cuda").int()
        self.lens.random_(0, self.longest + 1, generator=self.g)
        self.parents.random_(-1, self.sequences, generator=self.g)
        used = torch.arange(self.width, device="cuda") < ((self.lens + PAGE - 1) // PAGE)[:, None]
        self.table.copy_(torch.where(used, order[:self.width * self.sequences].view(self.sequences, self.width), -1))
        self.refs0.zero_()
        self.refs0[self.table[used].long()] = 1
        self.x.normal_(generator=self.g)
        self.fresh()

    def fresh(self):
        self.cache.k.copy_(self.k0)
        self.cache.v.copy_(self.v0)
        self.flags.zero_()

    def run(self, stream=None, alone=False):
        from inferno_hip import device as D
        self.refs.copy_(self.refs0)
        table, lens, copies = D.kv_fork(self.table, self.lens, self.parents, self.refs, PAGE, room=self.new, flags=self.flags, stream=stream)
        D.kv_copy(self.cache, copies, flags=self.flags, stream=stream)
        moves, moved = D.kv_compact(table, self.refs, flags=self.flags, stream=stream)
        D.kv_copy(self.cache, moves, moved, flags=self.flags, stream=stream)
        batch = D.KVBatch(self.starts, lens + self.new, table, self.children * self.new)
        q = D.rope_kv(self.x[:, :HEADS], self.x[:, HEADS:HEADS + KV], self.x[:, HEADS + KV:], self.turns, self.layer, batch,
                      mscale=self.mscale, flags=self.flags, stream=stream)
        out = D.attn_paged(q, self.layer, batch, workspace=None if alone else self.workspace, flags=self.flags, stream=stream)
        self.kept = batch  # (its tensors live as long as a graph that reads them)
        return [table, lens, copies, moves, moved, self.refs, q, out, self.cache.k, self.cache.v, self.flags]


def same(got, want):
    for i, (a, b) in enumerate(zip(got, want)):
        if a.is_floating_point():
            a, b = a.view(torch.int16 if a.element_size() == 2 else torch.int32), b.view(torch.int16 if b.element_size() == 2 else torch.int32)
        assert torch.equal(a, b), i


# one token and a chunk a child; forks of one launch (up to 64 tables) and of two
SIZES = [(3, 5, 300, 1), (2, 3, 700, 40), (30, 60, 200, 1), (1, 2, 2000, 3)]


@pytest.mark.parametrize("kv", [F16, BF16])
@pytest.mark.parametrize("sizes", SIZES)
def test_a_captured_step_replays_with_new_contents(sizes, kv):
    print("[case]", sizes, kv, flush=True)
    s = Step(sum(sizes), *sizes, kv)
    s.contents()
    s.run()
    torch.cuda.synchronize()
    assert int(s.flags.item()) == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = s.run()
    held = s.kept
    other = torch.randn(512, 512, device="cuda")
    for _ in range(4):
        s.contents()
        want = [t.clone() for t in s.run()]
        torch.cuda.synchronize()
        s.fresh()
        for t in outs[:5] + outs[6:8]:
            t.fill_(-77)
        (other @ other).sum().item()  # the program's own work, and a wait, between replays
        graph.replay()
        torch.cuda.synchronize()
        same(outs, want)
        assert int(s.flags.item()) == 0
    assert held.tokens == sizes[1] * sizes[3]


def test_steps_from_threads_on_their_own_streams():
    steps = [Step(100 + i, *sizes, kv) for i, (sizes, kv) in enumerate(zip(SIZES, (F16, BF16, F16, BF16)))]
    want = []
    for s in steps:
        s.contents()
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
    torch.cuda.synchronize()
    threads = [threading.Thread(target=caller, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    for i in range(len(steps)):
        for got in kept[i]:
            same(got, want[i])
