"""Host side of rotary positions, the paged cache and attention: frequencies, refusals, and the check of a batch (no GPU)."""
import ctypes as C
import math

import numpy as np
import pytest

import ojas_engine_b200 as ob
from ojas_engine_b200 import lib as oblib

E_ARG, E_UNSUPPORTED, E_LIMIT = -1, -3, -6


def call(name, *args):
    err = C.create_string_buffer(256)
    return getattr(oblib.load(), name)(*args, err, 256), err.value.decode()


# ---------------------------------------------------------------------------------------------------------- frequencies
@pytest.mark.parametrize("rot,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (96, 1e6)])
def test_frequencies(rot, base):
    got = ob.rope_frequencies(rot, base)
    want = np.array([base ** (-2 * i / rot) for i in range(rot // 2)])
    assert np.allclose(got, want, rtol=1e-14, atol=0)


def test_scaled_frequencies():
    rot, base, orig = 128, 10000.0, 4096
    plain = ob.rope_frequencies(rot, base)
    assert np.allclose(ob.rope_frequencies(rot, base, factor=4.0), plain / 4, rtol=1e-15)
    factors = np.linspace(1, 8, rot // 2).astype(np.float32)
    assert np.allclose(ob.rope_frequencies(rot, base, freq_factors=factors), plain / factors, rtol=1e-15)
    got = ob.rope_frequencies(rot, base, factor=8.0, orig_len=orig, beta_fast=32.0, beta_slow=1.0)
    turns = orig * plain / (2 * math.pi)
    assert np.allclose(got[turns >= 32], plain[turns >= 32], rtol=1e-15)
    assert np.allclose(got[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    middle = (turns > 1) & (turns < 32)
    keep = (turns[middle] - 1) / 31
    assert np.allclose(got[middle], plain[middle] * keep + plain[middle] / 8 * (1 - keep), rtol=1e-14)


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=2048), dict(base=1.0), dict(base=math.nan), dict(base=math.inf),
                                dict(factor=0.0), dict(factor=-2.0), dict(magnitude=0.0), dict(magnitude=math.inf),
                                dict(orig_len=4096, beta_fast=1.0, beta_slow=2.0), dict(freq_factors=[0.0] * 32), dict(freq_factors=[1.0] * 31)])
def test_frequency_refusals(kw):
    with pytest.raises(ob.OjasB200Error):
        ob.rope_frequencies(**{"rot_dim": 64, **kw})


# ------------------------------------------------------------------------------------------------------------- refusals
ROPE = dict(rot=128, layout=0, xt=ob.F32, x=1024, xs=0, yt=ob.F32, y=4096, ys=0, pos=512, M=4, heads=8, dim=128)


@pytest.mark.parametrize("change,code", [
    ({}, 0), (dict(rot=64), 0), (dict(x=4096), 0), (dict(M=0, x=0, y=0, pos=0), 0), (dict(xt=ob.BF16, x=1026), 0), (dict(dim=130, rot=2), 0),
    (dict(layout=2), E_ARG), (dict(xt=2), E_ARG), (dict(yt=8), E_ARG), (dict(heads=0), E_ARG), (dict(dim=127, rot=2), E_ARG), (dict(rot=130), E_ARG),
    (dict(xs=1023), E_ARG), (dict(ys=1000), E_ARG), (dict(x=0), E_ARG), (dict(y=0), E_ARG), (dict(pos=0), E_ARG), (dict(x=1026), E_ARG), (dict(pos=514), E_ARG),
    (dict(x=4096, xs=2048), E_ARG), (dict(x=4096, yt=ob.F16), E_ARG), (dict(M=1 << 30), E_LIMIT), (dict(xs=1 << 41), E_LIMIT)])
def test_rope_rows_refusals(change, code):
    rc, why = call("ojas_b200_rope_rows_check", *{**ROPE, **change}.values())
    assert rc == code, why
    assert bool(why) == bool(code)


KV = dict(t=ob.F16, k=4096, v=8192, pages=4, page=16, heads=2, dim=128, ps=2 * 16 * 128, hs=16 * 128, ts=128)


@pytest.mark.parametrize("change,code", [
    ({}, 0), (dict(t=ob.BF16), 0), (dict(page=48, hs=48 * 128, ps=2 * 48 * 128), 0), (dict(hs=128, ts=256), 0),                        # heads inside a token
    (dict(pages=1, ps=0), 0), (dict(ps=2 * 2 * 16 * 128), 0),                                                                        # k and v of a page side by side
    (dict(t=ob.F32), E_ARG), (dict(dim=96), E_UNSUPPORTED), (dict(page=8), E_UNSUPPORTED), (dict(page=20), E_UNSUPPORTED), (dict(page=0), E_UNSUPPORTED),
    (dict(pages=0), E_ARG), (dict(heads=0), E_ARG), (dict(k=0), E_ARG), (dict(v=8200), E_ARG), (dict(ts=132), E_ARG), (dict(ts=64), E_ARG),
    (dict(ps=2 * 16 * 128 - 8), E_ARG), (dict(hs=128, ts=128), E_ARG), (dict(ts=256), E_ARG), (dict(heads=70000), E_LIMIT), (dict(ps=1 << 40), E_LIMIT)])
def test_cache_refusals(change, code):
    rc, why = call("ojas_b200_kv_check", *{**KV, **change}.values())
    assert rc == code, why


def seqs(**change):
    f = {**dict(cu=256, len=512, table=1024, n_seqs=3, table_stride=8, max_rows=4, max_len=100), **change}
    return C.byref(oblib.SeqsStruct(*f.values()))


APPEND = dict(heads=2, dim=128, rot=128, layout=0, xt=ob.F32, q=1024, qs=0, k=2048, ks=0, v=4096, vs=0, qt=ob.F32, qo=8192, qos=0, hq=8, pos=0, seqs=None, M=12)


@pytest.mark.parametrize("change,code", [
    ({}, 0), (dict(hq=0, q=0, qo=0), 0), (dict(rot=0, layout=7), 0), (dict(pos=128), 0), (dict(qo=1024), 0), (dict(M=0, k=0, v=0, q=0, qo=0), 0),
    (dict(ks=1 << 12, vs=1 << 12, qs=1 << 12), 0), (dict(seqs=seqs(n_seqs=0, cu=0, len=0, table=0)), 0),
    (dict(layout=5), E_ARG), (dict(rot=256), E_ARG), (dict(xt=1000), E_ARG), (dict(qt=7), E_ARG), (dict(k=0), E_ARG), (dict(v=0), E_ARG), (dict(q=0), E_ARG),
    (dict(qo=0), E_ARG), (dict(ks=255), E_ARG), (dict(qs=1023), E_ARG), (dict(qos=8), E_ARG), (dict(k=2050), E_ARG), (dict(pos=126), E_ARG),
    (dict(qo=1024, qt=ob.F16), E_ARG), (dict(hq=1 << 20), E_LIMIT), (dict(M=1 << 30), E_LIMIT),
    (dict(seqs=seqs(cu=0)), E_ARG), (dict(seqs=seqs(table_stride=0)), E_ARG), (dict(seqs=seqs(max_rows=0)), E_ARG), (dict(seqs=seqs(len=514)), E_ARG),
    (dict(seqs=seqs(max_len=1 << 31)), E_LIMIT), (dict(seqs=seqs(n_seqs=1 << 31)), E_LIMIT)])
def test_append_refusals(change, code):
    rc, why = call("ojas_b200_kv_append_check", *{**APPEND, "seqs": seqs(), **change}.values())
    assert rc == code, why


ATTN = dict(ct=ob.F16, page=16, heads=2, dim=128, at=ob.F32, hq=8, q=1024, qs=0, out=4096, os=0, scale=0.1, causal=1, window=0, seqs=None, M=12)


@pytest.mark.parametrize("change,code", [
    ({}, 0), (dict(at=ob.F16), 0), (dict(ct=ob.BF16), 0), (dict(hq=14), 0), (dict(window=1), 0), (dict(causal=0), 0), (dict(scale=-1.0), 0), (dict(qs=1024 + 256), 0),
    (dict(M=0, q=0, out=0), 0), (dict(at=ob.BF16), E_UNSUPPORTED), (dict(dim=80), E_UNSUPPORTED), (dict(page=24), E_UNSUPPORTED), (dict(causal=0, window=5), E_UNSUPPORTED),
    (dict(hq=9), E_ARG), (dict(hq=0), E_ARG), (dict(heads=0), E_ARG), (dict(q=0), E_ARG), (dict(out=0), E_ARG), (dict(q=1032), E_ARG), (dict(out=4100), E_ARG),
    (dict(qs=1000), E_ARG), (dict(qs=1026), E_ARG), (dict(os=1), E_ARG), (dict(scale=math.nan), E_ARG), (dict(scale=math.inf), E_ARG), (dict(window=-1), E_ARG),
    (dict(seqs=seqs(table=0)), E_ARG), (dict(seqs=seqs(max_len=0)), E_ARG), (dict(M=1 << 29), E_LIMIT)])
def test_attention_refusals(change, code):
    rc, why = call("ojas_b200_attention_check", *{**ATTN, "seqs": seqs(), **change}.values())
    assert rc == code, why


def test_calls_without_a_context_are_refused():
    l = oblib.load()
    assert l.ojas_b200_attention(None, None, None, 0, None, 0, 0, 1.0, 1, 0, None, 0, 0, None, 0) == E_ARG
    assert l.ojas_b200_kv_append(None, None, None, None, 0, 0, None, 0, None, 0, None, 0, 0, None, 0, 0, None, 0) == E_ARG
    assert l.ojas_b200_rope_rows(None, None, 0, 0, None, 0, 0, None, 0, None, 0, 0, 0) == E_ARG
    assert l.ojas_b200_attention_workspace_bytes(None, None, None, 0, 1, 1, 0) == 0
    l.ojas_b200_kv_destroy(None)
    l.ojas_b200_rope_destroy(None)


# ---------------------------------------------------------------------------------------------------- a batch's arrays
@pytest.mark.parametrize("change,ok", [
    ({}, True), (dict(cu=[0, 0, 4, 4], max_rows=4), True), (dict(cu=[2, 3, 4, 6], M=8), True), (dict(table=[[0, 1, 2], [3, -1, -1], [5, 6, 1 << 30]]), True),
    (dict(cu=[0, 1, 0, 4]), False), (dict(cu=[-1, 1, 2, 4]), False), (dict(M=3), False), (dict(max_rows=1), False), (dict(lens=[33, 16, 1]), False),
    (dict(lens=[-1, 16, 20]), False), (dict(lens=[49, 16, 20]), False), (dict(max_len=32), False), (dict(table=[[0, 1, 7], [3, 0, 0], [5, 6, 0]]), False),
    (dict(table=[[0, 1, 2], [-1, 0, 0], [5, 6, 0]]), False)])
def test_batch_check(change, ok):
    f = {**dict(cu=[0, 1, 2, 4], lens=[33, 16, 20], table=[[0, 1, 2], [3, 0, 0], [5, 6, 0]], max_rows=2, max_len=64, M=4), **change}
    cu, lens, table = (np.ascontiguousarray(f[n], np.int32) for n in ("cu", "lens", "table"))
    rc, why = call("ojas_b200_seqs_check_host", cu.ctypes.data, lens.ctypes.data, table.ctypes.data, 3, 3, f["max_rows"], f["max_len"], 7, 16, f["M"])
    assert (rc == 0) == ok, why
