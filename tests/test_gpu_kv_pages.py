"""Forking, extending, freeing, compacting and copying pages against lists of
ints; every value is exact."""
import random

import pytest

import kv_plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def ints(v, *shape):
    t = torch.tensor(v, dtype=torch.int32, device="cuda")
    return t.reshape(shape) if shape else t


def tables(rng, lens, page, width, pages, spare=0):
    """Disjoint tables with up to `spare` pages more than the lengths need, and their counts."""
    order = rng.sample(range(pages), pages)
    table, refs = [], [0] * pages
    for n in lens:
        k = min(width, -(-n // page) + rng.randint(0, spare))
        row = [order.pop() for _ in range(k)]
        for p in row:
            refs[p] = 1
        table.append(row + [-1] * (width - k))
    return table, refs


def fork(table, lens, parents, refs, page, room):
    from inferno_hip import device as D
    print("[fork]", len(table), len(parents), len(refs), page, room, flush=True)
    width = len(table[0])
    r, flags = ints(refs), ints([0])
    t, n, c = D.kv_fork(ints(table, len(table), width), ints(lens), ints(parents), r, page, room=room, flags=flags)
    torch.cuda.synchronize()
    want = kv_plain.fork(table, lens, parents, refs, page, room)
    assert t.tolist() == want[0]
    assert n.tolist() == want[1]
    assert r.tolist() == want[2]
    assert c.tolist() == want[3]
    assert int(flags.item()) == (32 if want[4] else 0)
    return want


@pytest.mark.parametrize("seed", range(12))
def test_random_forks(seed):
    rng = random.Random(seed)
    page = rng.choice((16, 32))
    n = rng.randint(1, 9)
    lens = [rng.choice((0, 1, page, page + 1, 5 * page - 1, rng.randint(0, 900))) for _ in range(n)]
    width = max(-(-m // page) for m in lens) + 4
    pages = sum(-(-m // page) for m in lens) + 2 * n + rng.randint(0, 60)
    table, refs = tables(rng, lens, page, width, pages, spare=2)
    held = rng.randrange(pages)  # a page that something else holds too
    refs[held] += 1
    parents = [rng.randint(-1, n - 1) for _ in range(rng.randint(1, 20))]
    fork(table, lens, parents, refs, page, rng.choice((0, 1, 17, 40)))


def test_release_extend_reorder_and_growing_generations():
    rng = random.Random(3)
    lens, page, width = [30, 64, 5], 16, 12
    table, refs = tables(rng, lens, page, width, 64)
    t, n, r, _, full = fork(table, lens, [2, 0, 1], refs, page, 0)  # reordered
    assert not full and r == refs
    for room in (1, 16, 33):  # extended in place
        t, n, r, _, full = fork(t, n, [0, 1, 2], r, page, room)
        assert not full
    t, n, r, _, _ = fork(t, n, [1], r, page, 0)  # the others freed
    for _ in range(3):
        t, n, r, c, full = fork(t, n, [i // 2 for i in range(2 * len(t))], r, page, 1)
    assert not full
    assert sum(r) == sum(x >= 0 for row in t for x in row)
    _, _, r, _, _ = fork(t, n, [-1], r, page, 0)
    assert sum(r) == 0


def test_no_children_gives_everything_back():
    from inferno_hip import device as D
    rng = random.Random(4)
    table, refs = tables(rng, [50, 20], 16, 6, 20)
    r = ints(refs)
    t, n, c = D.kv_fork(ints(table), ints([50, 20]), ints([]).int(), r, 16)
    assert t.shape == (0, 6) and not bool(r.any())


def test_pages_run_out():
    rng = random.Random(5)
    for pages in (9, 10, 11, 13):
        table, refs = tables(rng, [70, 66], 16, 9, max(pages, 10))
        fork(table, [70, 66], [0, 0, 1, 1, -1], refs, 16, 20)


def test_wide_pools_and_many_children():
    """Pools of several search steps (4096 counts each), the free pages far apart, more children than waves."""
    rng = random.Random(6)
    pages = 20011
    lens = [rng.randint(0, 600) for _ in range(40)]
    table, refs = tables(rng, lens, 16, 45, pages)
    for p in range(pages):
        if refs[p] == 0 and rng.random() < 0.97:
            refs[p] = 1
    parents = [rng.randint(-1, 39) for _ in range(150)]
    fork(table, lens, parents, refs, 16, 30)


def test_fork_leaves_out_what_does_not_fit():
    from inferno_hip import device as D
    table, lens = [[0, 99, 2, -1]], [60]
    refs, flags = ints([1, 0, 1, 0, 0]), ints([0])
    t, n, c = D.kv_fork(ints(table), ints(lens), ints([0, 5, 0]), refs, 16, flags=flags)
    torch.cuda.synchronize()
    assert int(flags.item()) == 8 | 16 | 32  # a page outside the pool, a parent that is not there, too few pages
    assert n.tolist() == [60, 0, 60] and all(x < 5 for row in t.tolist() for x in row)
    flags.zero_()
    t, n, c = D.kv_fork(ints([[0, 1]]), ints([500]), ints([0]), ints([1, 1, 0]), 16, flags=flags)
    assert n.tolist() == [32] and t.tolist() == [[0, 1]] and int(flags.item()) == 16


@pytest.mark.parametrize("seed", range(10))
def test_random_compactions(seed):
    from inferno_hip import device as D
    rng = random.Random(100 + seed)
    pages = rng.choice((1, 2, 3, 50, 4095, 4096, 4097, 9001))
    refs = [rng.choice((0, 0, 1, 2)) for _ in range(pages)] if seed else [0] * pages
    used = [p for p in range(pages) if refs[p]]
    table = [[rng.choice(used) if used and rng.random() < 0.8 else -1 for _ in range(7)] for _ in range(9)]
    print("[compact]", pages, len(used), flush=True)
    t, r, flags = ints(table), ints(refs), ints([0])
    copies, moved = D.kv_compact(t, r, flags=flags)
    torch.cuda.synchronize()
    want = kv_plain.compact(table, refs)
    assert t.tolist() == want[0] and r.tolist() == want[1]
    n = int(moved.item())
    assert copies.tolist()[:n] == want[2] and n == len(want[2])
    assert all(c == [-1, -1] for c in copies.tolist()[n:]) and int(flags.item()) == 0


@pytest.mark.parametrize("layers,heads,page,dim,dtype", [(1, 1, 16, 8, torch.float16), (3, 2, 16, 64, torch.bfloat16),
                                                         (2, 8, 64, 128, torch.float16), (1, 3, 16, 200, torch.bfloat16)])
def test_copies(layers, heads, page, dim, dtype):
    from inferno_hip import device as D
    pages = 23
    both = torch.randn(layers, pages, 2, heads, page, dim, device="cuda").to(dtype)
    k, v = both[:, :, 0], both[:, :, 1]
    want = both.clone()
    pairs = [[3, 4], [-1, -1], [22, 0], [5, -1], [-1, 6], [7, 7], [3, 9]]
    for a, b in pairs:
        if a >= 0 and b >= 0:
            want[:, b] = both[:, a]
    flags = ints([0])
    D.kv_copy(D.KVCache(k, v), ints(pairs), flags=flags)
    torch.cuda.synchronize()
    assert torch.equal(both, want) and int(flags.item()) == 0
    # the count ends the list; ids outside the pool are left out and reported, as are lists that mix
    before = both.clone()
    for count in (0, -3):
        D.kv_copy(D.KVCache(k, v), ints([[1, 2], [2, 3]]), count=ints([count]), flags=flags)
    D.kv_copy(D.KVCache(k, v), ints([[23, 2], [2, 99]]), count=ints([5]), flags=flags)
    torch.cuda.synchronize()
    assert torch.equal(both, before) and int(flags.item()) == 8
    for mixed in ([[1, 2], [3, 2]], [[1, 2], [2, 3]]):
        flags.zero_()
        D.kv_copy(D.KVCache(k, v), ints(mixed), flags=flags)
        assert int(flags.item()) == 8


def test_copies_of_layers_within_pages():
    """All layers of a page together: the layer stride is the smaller one."""
    from inferno_hip import device as D
    both = torch.randn(9, 3, 2, 2, 16, 64, device="cuda").half()  # pages, layers, k and v
    want = both.clone()
    want[7] = both[2]
    k, v = both[:, :, 0].transpose(0, 1), both[:, :, 1].transpose(0, 1)
    D.kv_copy(D.KVCache(k, v), ints([[2, 7]]))
    torch.cuda.synchronize()
    assert torch.equal(both, want)


def test_wrapper_refusals():
    from inferno_hip import device as D
    t, n, r = ints([[0, 1]]), ints([20]), ints([1, 1, 0])
    cache = D.KVCache(torch.zeros(3, 1, 16, 8, dtype=torch.float16, device="cuda"), torch.zeros(3, 1, 16, 8, dtype=torch.float16, device="cuda"))
    for bad in (lambda: D.kv_fork(t.long(), n, n, r, 16), lambda: D.kv_fork(t, ints([1, 2]), n, r, 16), lambda: D.kv_fork(t, n, n, r, 0),
                lambda: D.kv_fork(t, n, n, r, 16, room=-1), lambda: D.kv_compact(t, r.cpu()), lambda: D.kv_copy(cache, r)):
        with pytest.raises(D.IHIPArgumentError):
            bad()
