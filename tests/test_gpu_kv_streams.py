"""The paged-cache calls on a stream of their own while the current stream is
behind: what a call allocates is neither filled nor still used over there."""
import pytest

from test_gpu_kv_attn import BF16, F16, F32, build, ints

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def behind(sizes):
    """Some 10 ms of work on the current stream, and then writes of ones to blocks of
    these sizes that go back to the allocator at once."""
    a = torch.full((8192, 8192), 0.01, dtype=F16, device="cuda")
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    for _ in range(10):
        torch.mm(a, a, out=b)
    for n in sizes:
        torch.full((n,), 1, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("act,kv,new,lens", [(F32, F16, [1], [3000]), (BF16, BF16, [1, 40], [900, 700])])
def test_attention_and_rope(act, kv, new, lens):
    from inferno_hip import device as D
    q, k, v, starts, lens, table = build(40, new, lens, 8, 2, 128, 16, act, kv)
    cache = D.KVCache(k.cuda().nan_to_num_(0.0), v.cuda().nan_to_num_(0.0))
    batch = D.KVBatch(ints(starts), ints(lens), ints(table), q.shape[0])
    qd, side = q.cuda(), torch.cuda.Stream()
    want = D.attn_paged(qd, cache, batch)
    turns, m = D.rope_turns(128, 10000.0)
    turned = D.rope_kv(qd.float(), None, None, turns, cache, batch, mscale=m)
    sizes = [D.attn_workspace(8, cache, batch).numel(), want.numel() * want.element_size(), turned.numel() * 4]
    torch.cuda.synchronize()
    plain = qd.float()
    for _ in range(2):
        behind(sizes)
        got = D.attn_paged(qd, cache, batch, stream=side)
        again = D.rope_kv(plain, None, None, turns, cache, batch, mscale=m, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, turned)


def test_forks_and_compaction():
    from inferno_hip import device as D
    table = ints([[3, 1, 7, -1], [5, 9, -1, -1]])
    lens, parents, side = ints([40, 20]), ints([0, 0, 1, -1]), torch.cuda.Stream()
    refs = [0, 1, 0, 1, 0, 1, 0, 1, 0, 1, 0, 0, 0, 0, 0, 0]
    torch.cuda.synchronize()
    made = []
    for stream in (None, side):
        r = ints(refs)
        torch.cuda.synchronize()
        if stream is not None:
            behind([64, 80])
        t, n, c = D.kv_fork(table, lens, parents, r, 16, room=1, stream=stream)
        torch.cuda.synchronize()
        if stream is not None:
            behind([64, 132])
        moves, count = D.kv_compact(t, r, stream=stream)
        torch.cuda.synchronize()
        made.append([x.tolist() for x in (t, n, c, r, moves, count)])
    assert made[0] == made[1]
