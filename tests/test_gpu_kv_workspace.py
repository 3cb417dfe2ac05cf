"""What attn_paged clears: the counts in front of its workspace, not the parts
behind them (which every call writes before it reads them)."""
import pytest

from test_gpu_kv_attn import F16, F32, build, ints

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def made(seed, new, lens, width=0):
    from inferno_hip import device as D
    q, k, v, starts, lens, table = build(seed, new, lens, 8, 2, 128, 16, F32, F16)
    table = [r + [-1] * (width - len(r)) for r in table]
    cache = D.KVCache(k.cuda().nan_to_num_(0.0), v.cuda().nan_to_num_(0.0))
    return q.cuda(), cache, D.KVBatch(ints(starts), ints(lens), ints(table), q.shape[0])


def left_behind(n):
    """A freed block of n bytes, the only one of its size, all ones (as floats: NaN)."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    t = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    return t.data_ptr()


def test_only_the_counts_are_cleared():
    from inferno_hip import _lib
    from inferno_hip import device as D
    header = (_lib.PKG.parent / "include" / "inferno_hip.h").read_text()
    assert f"#define IHIP_ATTN_COUNT_BYTES {_lib.ATTN_COUNT_BYTES}\n" in header
    q, cache, batch = made(50, [1] * 9, [900] * 9)
    n = D.attn_workspace(8, cache, batch).numel()
    assert n > 10 * _lib.ATTN_COUNT_BYTES
    at = left_behind(n)
    ws = D.attn_workspace(8, cache, batch)
    assert ws.data_ptr() == at
    assert not bool(ws[:_lib.ATTN_COUNT_BYTES].any()) and bool((ws[_lib.ATTN_COUNT_BYTES:] == 255).all())


@pytest.mark.parametrize("new,lens,width", [([1], [3000], 0), ([1, 3], [900, 40], 0), ([40, 9], [700, 30], 64), ([2], [9], 200)])
def test_what_the_parts_held_has_no_influence(new, lens, width):
    from inferno_hip import device as D
    q, cache, batch = made(51, new, lens, width)
    n = D.attn_workspace(8, cache, batch).numel()
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    want = D.attn_paged(q, cache, batch, workspace=ws)
    out = torch.empty_like(q)
    left_behind(n)
    D.attn_paged(q, cache, batch, out=out)
    torch.cuda.synchronize()
    assert bool(torch.isfinite(want).all()) and torch.equal(out, want)
