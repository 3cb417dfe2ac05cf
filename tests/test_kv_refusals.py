"""The paged-cache entry points refuse what they cannot run, before any device
work (no GPU needed: the pointers are never dereferenced), and the rotary table
against its formulas."""
import ctypes as C
import math

import pytest

from inferno_hip import _lib

BASE = 1 << 24
FAR = [BASE + (i << 32) for i in range(40)]  # addresses that nothing overlaps


def cache(**kw):
    f = dict(k=FAR[0], v=FAR[1], type=_lib.F16, pages=8, page_size=16, kv_heads=2, head_dim=64, page_stride=2 * 16 * 64)
    f.update(kw)
    return _lib.KVCacheStruct(**f)


def batch(**kw):
    f = dict(q_starts=FAR[2], kv_lens=FAR[3], page_table=FAR[4], sequences=2, table_stride=4, tokens=6)
    f.update(kw)
    return _lib.KVBatchStruct(**f)


def rope(c=None, b=None, **kw):
    a = dict(q=FAR[5], qs=4 * 64, k=FAR[6], ks=2 * 64, v=FAR[7], vs=2 * 64, heads=4, qn=None, kn=None, eps=1e-6,
             turns=FAR[8], rot=64, layout=0, m=1.0, pos=None, out=FAR[9], type=_lib.F16)
    a.update(kw)
    return _lib.lib().ihip_rope_kv_dev(*a.values(), C.byref(c or cache()), C.byref(b or batch()), None, None)


def attn(c=None, b=None, ws=0, ws_bytes=0, **kw):
    a = dict(q=FAR[5], type=_lib.F16, out=FAR[9], heads=4, scale=0.1, cap=0.0, window=0, prefix=None, slopes=None)
    a.update(kw)
    return _lib.lib().ihip_attn_paged_dev(*a.values(), C.byref(c or cache()), C.byref(b or batch()), None, ws or None,
                                          ws_bytes, None)


def said():
    return _lib.lib().ihip_last_error()


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(type=_lib.F32), dict(type=12), dict(pages=0), dict(pages=-1), dict(page_size=8),
    dict(page_size=24), dict(page_size=0), dict(page_size=1 << 17), dict(kv_heads=0), dict(head_dim=60),
    dict(head_dim=264, page_stride=1 << 20), dict(head_dim=0), dict(page_stride=2 * 16 * 64 - 8),
    dict(page_stride=2 * 16 * 64 + 4), dict(page_stride=-8), dict(page_stride=1 << 61), dict(k=FAR[0] + 8),
    dict(kv_heads=4096, page_size=65536, page_stride=1 << 40)])
def test_a_cache_that_does_not_hold_together_is_refused(bad):
    assert attn(c=cache(**bad)) == _lib.IHIP_ERR_INVALID, said()
    assert rope(c=cache(**bad)) == _lib.IHIP_ERR_INVALID, said()
    assert _lib.lib().ihip_kv_copy_dev(C.byref(cache(**bad)), 1, 0, FAR[5], 1, None, None, None) == _lib.IHIP_ERR_INVALID
    b = batch()
    assert _lib.lib().ihip_attn_paged_scratch_bytes(_lib.F16, 4, C.byref(cache(**bad)), C.byref(b)) == 0


@pytest.mark.parametrize("bad", [dict(q_starts=None), dict(kv_lens=None), dict(page_table=None), dict(sequences=-1),
                                 dict(tokens=-1), dict(table_stride=-1)])
def test_a_batch_that_does_not_hold_together_is_refused(bad):
    assert attn(b=batch(**bad)) == _lib.IHIP_ERR_INVALID, said()
    assert rope(b=batch(**bad)) == _lib.IHIP_ERR_INVALID, said()


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(out=None), dict(heads=3), dict(heads=0), dict(type=_lib.BF16), dict(type=8), dict(window=-1),
    dict(scale=math.nan), dict(scale=math.inf), dict(cap=-1.0), dict(cap=math.nan), dict(cap=1e-20), dict(scale=1e-30), dict(q=FAR[5] + 2),
    dict(out=FAR[9] + 8), dict(out=FAR[5]), dict(out=FAR[5] + 6 * 4 * 64 * 2 - 16), dict(out=FAR[0] + 16)])
def test_attention_arguments_are_refused(bad):
    assert attn(**bad) == _lib.IHIP_ERR_INVALID, said()


def test_attention_sizes_past_the_index_ranges_are_refused():
    for stride in (1 << 30, (1 << 26) + 1):  # 2^30 + 16 tokens
        assert attn(b=batch(table_stride=stride)) == _lib.IHIP_ERR_INVALID
        assert b"2^30" in said()
    assert attn(b=batch(tokens=1 << 30)) == _lib.IHIP_ERR_INVALID


def test_attention_workspace_is_checked():
    c, b = cache(pages=1000), batch(sequences=1, tokens=1, table_stride=900)
    need = _lib.lib().ihip_attn_paged_scratch_bytes(_lib.F16, 4, C.byref(c), C.byref(b))
    assert need > 0
    for ws, n in ((0, need), (FAR[10], need - 1), (FAR[10] + 8, need), (FAR[5], need), (FAR[9], need), (FAR[1], need)):
        assert attn(c=c, b=b, ws=ws, ws_bytes=n) == _lib.IHIP_ERR_INVALID
        assert b"workspace" in said()
    # and never more for shorter tables or fewer rows than it was sized for
    small = batch(sequences=1, tokens=1, table_stride=100)
    assert _lib.lib().ihip_attn_paged_scratch_bytes(_lib.F16, 4, C.byref(c), C.byref(small)) <= need


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(out=None), dict(k=None), dict(v=None), dict(turns=None), dict(heads=0), dict(type=2), dict(rot=63),
    dict(rot=66), dict(rot=-2), dict(layout=2), dict(layout=-1), dict(qs=4 * 64 - 4), dict(qs=4 * 64 + 2), dict(ks=124),
    dict(vs=130), dict(q=FAR[5] + 4), dict(turns=FAR[8] + 4), dict(qn=FAR[10] + 8), dict(out=FAR[5], type=_lib.F16),
    dict(out=FAR[5], type=_lib.F32, qs=4 * 64 + 4), dict(out=FAR[5] + 16, type=_lib.F32), dict(out=FAR[6]),
    dict(out=FAR[7] + 16), dict(out=FAR[0]), dict(k=FAR[1] + 64), dict(qs=1 << 62)])
def test_rope_arguments_are_refused(bad):
    assert rope(**bad) == _lib.IHIP_ERR_INVALID, said()


def test_nothing_to_do_is_no_error():
    for b in (batch(tokens=0), batch(sequences=0)):
        assert attn(b=b) == 0 and rope(b=b) == 0
    L = _lib.lib()
    assert L.ihip_kv_copy_dev(C.byref(cache()), 1, 0, None, 0, None, None, None) == 0
    assert L.ihip_kv_fork_dev(None, None, 0, None, 0, 1, 4, 16, 8, None, None, None, None, None, None, None) == 0


def fork(**kw):
    a = dict(table=FAR[10], lens=FAR[11], sequences=3, parents=FAR[12], children=5, room=1, stride=4, page=16, pages=32,
             refs=FAR[13], table_out=FAR[14], lens_out=FAR[15], copies=FAR[16], scratch=FAR[17], flags=None, stream=None)
    a.update(kw)
    return _lib.lib().ihip_kv_fork_dev(*a.values())


@pytest.mark.parametrize("bad", [
    dict(sequences=-1), dict(children=-1), dict(room=-1), dict(stride=0), dict(page=0), dict(pages=0), dict(table=None),
    dict(lens=None), dict(parents=None), dict(refs=None), dict(table_out=None), dict(lens_out=None), dict(copies=None),
    dict(scratch=None), dict(table_out=FAR[10] + 16), dict(lens_out=FAR[12]), dict(copies=FAR[14]), dict(refs=FAR[11]),
    dict(scratch=FAR[16] + 8), dict(pages=2 ** 31 - 1), dict(children=1 << 20, stride=1 << 20), dict(stride=1 << 28)])
def test_fork_arguments_are_refused(bad):
    assert fork(**bad) == _lib.IHIP_ERR_INVALID, said()


@pytest.mark.parametrize("bad", [
    dict(entries=-1), dict(pages=0), dict(table=None), dict(refs=None), dict(copies=None), dict(moved=None),
    dict(scratch=None), dict(refs=FAR[10]), dict(scratch=FAR[11] + 4), dict(copies=FAR[10] + 8), dict(moved=FAR[11]),
    dict(pages=2 ** 31 - 1)])
def test_compact_arguments_are_refused(bad):
    a = dict(table=FAR[10], entries=12, refs=FAR[11], pages=32, copies=FAR[12], moved=FAR[13], scratch=FAR[14],
             flags=None, stream=None)
    a.update(bad)
    assert _lib.lib().ihip_kv_compact_dev(*a.values()) == _lib.IHIP_ERR_INVALID, said()


@pytest.mark.parametrize("layers,stride,n,copies", [(0, 0, 1, FAR[5]), (2, 8, 1, FAR[5]), (2, 2 * 16 * 64 + 4, 1, FAR[5]),
                                                    (1, -8, 1, FAR[5]), (1, 0, -1, FAR[5]), (1, 0, 1, None)])
def test_copy_arguments_are_refused(layers, stride, n, copies):
    assert _lib.lib().ihip_kv_copy_dev(C.byref(cache()), layers, stride, copies, n, None, None, None) == _lib.IHIP_ERR_INVALID


def turns(scaling, rot, base=1e6, factor=4.0, original=8192, low=1.0, high=32.0):
    out, m = (C.c_double * max(1, rot // 2))(), C.c_float(0)
    rc = _lib.lib().ihip_rope_turns(_lib.ROPE_SCALING.get(scaling, scaling), rot, base, factor, original, low, high, out,
                                    C.byref(m))
    return rc, list(out), m.value


@pytest.mark.parametrize("rot", [2, 16, 20, 64, 128, 256])
def test_rotary_tables_follow_their_formulas(rot):
    """Turns, frequency / (2 pi); a few roundings of 64 bits (pow among them)."""
    plain = [1e6 ** (-2 * i / rot) / (2 * math.pi) for i in range(rot // 2)]
    near = dict(rel=1e-13)
    assert turns("none", rot, factor=1.0)[1] == pytest.approx(plain, **near)
    rc, t, m = turns("linear", rot)
    assert rc == 0 and m == 1.0 and t == pytest.approx([x / 4 for x in plain], **near)
    if rot > 2:
        b = 1e6 * 4.0 ** (rot / (rot - 2))
        assert turns("ntk", rot)[1] == pytest.approx([b ** (-2 * i / rot) / (2 * math.pi) for i in range(rot // 2)], **near)
    rc, t, m = turns("bands", rot)
    for x, y in zip(plain, t):
        made = 8192 * x  # turns over the original length
        keep = min(max((made - 1) / 31, 0), 1)
        assert y == pytest.approx(x / 4 * (1 - keep) + x * keep, **near)
    rc, t, m = turns("yarn", rot)
    assert m == pytest.approx(0.1 * math.log(4.0) + 1, rel=1e-6)
    # pairs that turn more than `high` times keep their frequency, those below `low` are scaled whole
    pair = [rot * math.log(8192 / (n * 2 * math.pi)) / (2 * math.log(1e6)) for n in (32, 1)]
    lo, hi = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), rot - 1)
    for i, (x, y) in enumerate(zip(plain, t)):
        keep = 1 - min(max((i - lo) / max(hi - lo, 0.001), 0), 1)
        assert y == pytest.approx(x / 4 * (1 - keep) + x * keep, **near)


@pytest.mark.parametrize("bad", [dict(scaling=5), dict(scaling=-1), dict(rot=0), dict(rot=7), dict(rot=258), dict(base=0.0),
                                 dict(base=math.nan), dict(factor=0.0), dict(factor=math.inf), dict(rot=2, scaling="ntk"),
                                 dict(scaling="yarn", original=0), dict(scaling="bands", low=4.0, high=4.0),
                                 dict(scaling="yarn", low=0.0), dict(scaling="yarn", base=1.0)])
def test_rotary_tables_that_make_no_sense_are_refused(bad):
    a = dict(scaling="none", rot=64)
    a.update(bad)
    assert turns(**a)[0] == _lib.IHIP_ERR_INVALID
