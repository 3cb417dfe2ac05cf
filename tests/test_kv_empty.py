"""A step without tokens or without sequences: nothing to do, whatever the
addresses of empty buffers are (an empty tensor has none)."""
import ctypes as C

import pytest

from inferno_hip import _lib
from test_kv_refusals import attn, batch, cache, rope

NONE = [dict(tokens=0), dict(sequences=0, q_starts=None, kv_lens=None, page_table=None), dict(tokens=0, sequences=0)]


@pytest.mark.parametrize("b", NONE)
def test_no_tokens_need_no_buffers(b):
    assert rope(b=batch(**b), q=None, k=None, v=None, out=None) == 0, _lib.lib().ihip_last_error()
    assert rope(b=batch(**b), q=None, out=None, k=None, v=None, qs=0, ks=0, vs=0) == 0
    assert attn(b=batch(**b), q=None, out=None) == 0, _lib.lib().ihip_last_error()
    assert _lib.lib().ihip_attn_paged_scratch_bytes(_lib.F16, 4, C.byref(cache()), C.byref(batch(**b))) == 0


@pytest.mark.parametrize("b", NONE)
def test_types_and_sizes_are_checked_all_the_same(b):
    none = dict(b=batch(**b), q=None, out=None)
    for bad in (dict(heads=0), dict(heads=3), dict(type=8), dict(window=-1), dict(scale=float("nan"))):
        assert attn(**none, **bad) == _lib.IHIP_ERR_INVALID
    for bad in (dict(heads=0), dict(type=2), dict(rot=63), dict(rot=66), dict(layout=2)):
        assert rope(**none, k=None, v=None, **bad) == _lib.IHIP_ERR_INVALID
    assert attn(c=cache(head_dim=60), **none) == rope(c=cache(head_dim=60), **none) == _lib.IHIP_ERR_INVALID


@pytest.mark.gpu
def test_empty_tensors():
    torch = pytest.importorskip("torch")
    from inferno_hip import device as D
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    kv = D.KVCache(*(torch.zeros(4, 2, 16, 64, dtype=torch.float16, device="cuda") for _ in range(2)))
    turns, _ = D.rope_turns(64, 1e4)
    x = torch.randn(5, 8, 64, device="cuda")
    for b in (D.KVBatch(ints(0, 0), ints(7), ints(1).view(1, 1), 0),
              D.KVBatch(ints(0), ints(), torch.empty(0, 1, dtype=torch.int32, device="cuda"), 0)):
        for q, k, v in ((x[:0, :4], x[:0, 4:6], x[:0, 6:]), (x[:0, :4], None, None)):
            assert D.rope_kv(q, k, v, turns, kv, b).shape == (0, 4, 64)
            assert D.rope_kv(q, k, v, turns, kv, b, out_dtype=torch.float16).dtype == torch.float16
        assert D.attn_paged(x[:0, :4].contiguous(), kv, b).shape == (0, 4, 64)
        assert D.attn_paged(torch.empty(0, 4, 64, device="cuda"), kv, b, out=torch.empty(0, 4, 64, device="cuda")).numel() == 0
        assert D.attn_workspace(4, kv, b) is None
    # rows of no sequence stay as they are
    out = torch.full((5, 4, 64), 7.0, device="cuda")
    b = D.KVBatch(ints(0), ints(), torch.empty(0, 1, dtype=torch.int32, device="cuda"), 5)
    D.rope_kv(x[:, :4], x[:, 4:6], x[:, 6:], turns, kv, b, out=out)
    D.attn_paged(x[:, :4].contiguous(), kv, b, out=out)
    torch.cuda.synchronize()
    assert bool((out == 7).all()) and not bool(kv.k.any()) and not bool(kv.v.any())
