"""The entry points of recurrent layers and of sampling refuse what they cannot run,
before any device work (no GPU needed: the pointers are never dereferenced)."""
import ctypes as C
import os
import subprocess
import sys
from pathlib import Path

import pytest

from inferno_hip import _lib

BASE = 1 << 24
FAR = [BASE + (i << 32) for i in range(40)]  # addresses that nothing overlaps


def batch(**kw):
    f = dict(q_starts=FAR[0], kv_lens=FAR[1], slots=FAR[2], sequences=2, tokens=40, most=0)
    f.update(kw)
    return _lib.StateBatchStruct(**f)


def layer(**kw):
    f = dict(state=FAR[3], slot_stride=4 * 64 * 64, slots=3, k_heads=2, v_heads=4, k_dim=64, v_dim=64, decay=FAR[4],
             dt_bias=FAR[5], norm_w=FAR[6], norm_eps=1e-6, l2_eps=1e-6, scale=0.1)
    f.update(kw)
    return _lib.DeltaLayerStruct(**f)


def conv(b=None, **kw):
    a = dict(x=FAR[7], type=_lib.F32, stride=64, w=FAR[8], bias=FAR[9], channels=64, width=4, silu=1, state=FAR[10],
             slot=3 * 64, slots=3, out=FAR[11], out_type=_lib.F32)
    a.update(kw)
    return _lib.lib().ihip_short_conv_dev(*a.values(), C.byref(b or batch()), None, None)


def delta(rows=None, l=None, ws=FAR[20], ws_bytes=1 << 30, **kw):
    a = dict(q=FAR[12], qs=512, k=FAR[13], ks=512, v=FAR[14], vs=512, type=_lib.F16, a=FAR[15], as_=8, b=FAR[16], bs=8,
             gate=FAR[17], gs=256, out=FAR[18], out_type=_lib.F16)
    a.update(kw)
    return _lib.lib().ihip_gated_delta_dev(*a.values(), C.byref(l or layer()), C.byref(rows or batch()), None, ws or None, ws_bytes,
                                           None)


def sample(ws=FAR[29], ws_bytes=1 << 30, **kw):
    a = dict(logits=FAR[21], type=_lib.F32, stride=1000, rows=3, vocab=1000, t=FAR[22], k=FAR[23], p=FAR[24], m=FAR[25], u=FAR[26],
             tokens=FAR[27], logprobs=FAR[28], flags=FAR[30])
    a.update(kw)
    return _lib.lib().ihip_sample_dev(*a.values(), ws or None, ws_bytes, None)


def said():
    return _lib.lib().ihip_last_error()


BATCHES = [dict(sequences=-1), dict(tokens=-1), dict(most=-1), dict(q_starts=None), dict(slots=None),
           dict(sequences=1 << 30, tokens=1 << 30)]


@pytest.mark.parametrize("bad", BATCHES)
def test_batches(bad):
    assert conv(batch(**bad)) == _lib.IHIP_ERR_INVALID and said()
    assert delta(batch(**bad)) == _lib.IHIP_ERR_INVALID and said()
    assert _lib.lib().ihip_gated_delta_scratch_bytes(_lib.F16, C.byref(layer()), C.byref(batch(**bad))) == 0


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(w=None), dict(state=None), dict(out=None), dict(type=12), dict(out_type=-1), dict(channels=0),
    dict(channels=60), dict(channels=1 << 25), dict(width=1), dict(width=9), dict(stride=56), dict(stride=68), dict(stride=1 << 62),
    dict(slot=3 * 64 - 4), dict(slot=3 * 64 + 2), dict(slots=0), dict(slot=1 << 62), dict(x=FAR[7] + 8), dict(w=FAR[8] + 4),
    dict(bias=FAR[9] + 4), dict(state=FAR[10] + 4), dict(out=FAR[11] + 2),
    dict(out=FAR[7] + 64 * 4 * 39), dict(state=FAR[7] + 1024), dict(out=FAR[10] + 2 * 768), dict(w=FAR[11]), dict(bias=FAR[10]),
])
def test_the_convolution(bad):
    assert conv(**bad) == _lib.IHIP_ERR_INVALID and said()


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(k=None), dict(v=None), dict(a=None), dict(b=None), dict(out=None), dict(type=12), dict(out_type=_lib.BF16),
    dict(qs=120), dict(qs=516), dict(ks=64), dict(vs=248), dict(as_=3), dict(bs=3), dict(gs=252), dict(gs=258), dict(vs=1 << 62),
    dict(q=FAR[12] + 8), dict(gate=FAR[17] + 4), dict(out=FAR[18] + 8), dict(a=FAR[15] + 2),
    dict(out=FAR[12] + 2 * (39 * 512 + 64)), dict(out=FAR[17] + 16), dict(out=FAR[3] + 64), dict(q=FAR[3] + 64),
    dict(b=FAR[18] + 4), dict(ws=None), dict(ws_bytes=16), dict(ws=FAR[20] + 8), dict(ws=FAR[18] + 16), dict(ws=FAR[14] + 16),
    dict(ws=FAR[3] + 16),
])
def test_the_delta_rule(bad):
    assert delta(**bad) == _lib.IHIP_ERR_INVALID and said()


@pytest.mark.parametrize("bad", [
    dict(state=None), dict(decay=None), dict(dt_bias=None), dict(k_heads=0), dict(v_heads=0), dict(v_heads=3),
    dict(k_heads=8192, v_heads=8192), dict(k_dim=0), dict(k_dim=72), dict(k_dim=144), dict(v_dim=24), dict(v_dim=256),
    dict(slots=0), dict(slot_stride=4 * 64 * 64 - 4), dict(slot_stride=4 * 64 * 64 + 2), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(l2_eps=-1.0), dict(norm_eps=float("nan")), dict(state=FAR[3] + 4), dict(norm_w=FAR[6] + 4),
    dict(decay=FAR[4] + 2), dict(norm_w=FAR[18]), dict(decay=FAR[3]),
])
def test_layers(bad):
    assert delta(l=layer(**bad)) == _lib.IHIP_ERR_INVALID and said()


@pytest.mark.parametrize("bad", [
    dict(logits=None), dict(u=None), dict(tokens=None), dict(type=12), dict(rows=-1), dict(vocab=-1), dict(vocab=(1 << 22) + 1,
                                                                                                          stride=1 << 23),
    dict(stride=999), dict(stride=1 << 62), dict(logits=FAR[21] + 2), dict(ws=None), dict(ws_bytes=100), dict(ws=FAR[29] + 4),
    dict(tokens=FAR[26]), dict(logprobs=FAR[27] + 4), dict(flags=FAR[28]), dict(tokens=FAR[21] + 8), dict(ws=FAR[21] + 16),
    dict(ws=FAR[27] + 0), dict(logprobs=FAR[22] + 8),
])
def test_sampling(bad):
    assert sample(**bad) == _lib.IHIP_ERR_INVALID and said()


def test_rows_of_no_logits_are_an_error_of_their_own():
    assert sample(vocab=0) == _lib.IHIP_ERR_EMPTY and said()


def test_more_workgroups_than_a_launch_has():
    for b in (batch(sequences=1 << 24), batch(tokens=(1 << 30) - 1), batch(sequences=1 << 29)):
        assert conv(b) == _lib.IHIP_ERR_INVALID and b"too many" in said()
        assert delta(b) == _lib.IHIP_ERR_INVALID and b"too many" in said()
    b = batch(sequences=1 << 19)  # 4 heads, up to 8 workgroups a head
    assert delta(b) == _lib.IHIP_ERR_INVALID and b"too many" in said()


def test_nothing_to_do_needs_no_buffers():
    for b in (batch(tokens=0, q_starts=None, slots=None, kv_lens=None), batch(sequences=0, q_starts=None, slots=None)):
        assert conv(b, x=None, w=None, state=None, out=None) == _lib.IHIP_OK
        assert _lib.lib().ihip_gated_delta_scratch_bytes(_lib.F16, C.byref(layer()), C.byref(b)) == 0
        args = [None, 512, None, 512, None, 512, _lib.F16, None, 8, None, 8, None, 0, None, _lib.F16]
        assert _lib.lib().ihip_gated_delta_dev(*args, C.byref(layer()), C.byref(b), None, None, 0, None) == _lib.IHIP_OK
    assert sample(rows=0, logits=None, u=None, tokens=None, ws=None, ws_bytes=0) == _lib.IHIP_OK
    # but sizes and types are checked
    assert conv(batch(tokens=0), width=9) == _lib.IHIP_ERR_INVALID
    assert delta(batch(tokens=0), l=layer(k_dim=72)) == _lib.IHIP_ERR_INVALID


def test_workspaces_grow_with_their_sizes():
    L = _lib.lib()
    of = lambda t, **kw: L.ihip_gated_delta_scratch_bytes(t, C.byref(layer()), C.byref(batch(**kw)))
    assert of(_lib.F16, most=1) == 0 and of(_lib.F32, tokens=2, sequences=2) == 0
    assert 0 < of(_lib.F16) < of(_lib.F16, tokens=400) and of(12) == 0
    assert of(_lib.F32, most=17) == of(_lib.F32) == of(_lib.F32, most=1000)
    assert L.ihip_sample_scratch_bytes(0, 10) == 0 and L.ihip_sample_scratch_bytes(1, (1 << 22) + 1) == 0
    assert 0 < L.ihip_sample_scratch_bytes(1, 1000) <= L.ihip_sample_scratch_bytes(5, 1000)


def test_the_disabled_library_refuses():
    code = ("import sys; sys.path[:0] = ['inferno.jl_amd', 'tests']; import test_gd_refusals as t; "
            "print([f() for f in (t.conv, t.delta, t.sample)])")
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True,
                       env=dict(os.environ, IHIP_DISABLE="1"))
    assert r.stdout.strip() == str([_lib.IHIP_ERR_DISABLED] * 3), r.stdout + r.stderr
