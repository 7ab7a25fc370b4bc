"""Refusals of the paged cache, rotary and attention entry points: checked
before any device work, so they hold without a GPU."""
import ctypes as C
import math

import pytest

P = 1 << 20            # any aligned non-null address: a refused call never uses it
FAR = 1 << 40


def cache(flh, **kw):
    a = dict(k=P, v=FAR, dtype=flh.Dtype.F16, n_pages=64, page_size=16, n_kv_head=8, d_k=128, d_v=128,
             k_strides=(16 * 1024, 128, 2048), v_strides=(16 * 1024, 128, 2048))
    a.update(kw)
    return flh.KvCache(**a)


def attn(flh, **kw):
    a = dict(q=P, out=FAR, q_start=P, kv_len=P, table=P, ws=P, ws_bytes=1 << 40, q_tok=4096, q_head=128, o_tok=4096,
             o_head=128, dtype=flh.Dtype.F32, n_head=32, n_seq=2, n_tok=2, max_q=1, table_stride=4, causal=1, window=0,
             scale=0.1)
    a.update(kw)
    return flh.AttnP(**a)


def append(flh, **kw):
    a = dict(q=P, q_out=P, k=P, v=P, pos=P, slot=P, q_tok=6144, q_head=128, qo_tok=6144, qo_head=128, k_tok=6144,
             k_head=128, v_tok=6144, v_head=128, dtype=flh.Dtype.F32, n_tok=3, n_head=32, pos_stride=3)
    a.update(kw)
    return flh.RopeKvP(**a)


def plan(flh, **kw):
    a = dict(held=P, add=P, free_pages=P, taken_in=P, taken=P, table=P, q_start=P, kv_len=P, slot=P, pos=P, info=P, n_seq=2,
             page_size=16, n_free=8, table_stride=4, max_tok=8)
    a.update(kw)
    return flh.KvPlanP(**a)


class S:
    handle = None


def refused(flh, code, word, call, *args):
    with pytest.raises(flh.FlhError) as e:
        call(*args)
    assert e.value.code == code, str(e.value)
    assert word in str(e.value), str(e.value)


CACHES = [("ERR_UNSUPPORTED", "dtype", dict(dtype=0)), ("ERR_UNSUPPORTED", "dtype", dict(dtype=3)),
          ("ERR_ARG", "aligned", dict(k=P + 8)), ("ERR_ARG", "aligned", dict(v=None)),
          ("ERR_UNSUPPORTED", "power of two", dict(page_size=24)), ("ERR_UNSUPPORTED", "power of two", dict(page_size=0)),
          ("ERR_UNSUPPORTED", "power of two", dict(page_size=1 << 17)), ("ERR_ARG", "n_pages", dict(n_pages=0)),
          ("ERR_ARG", "n_pages", dict(n_pages=1 << 28)), ("ERR_ARG", "n_kv_head", dict(n_kv_head=0)),
          ("ERR_UNSUPPORTED", "multiples of 8", dict(d_k=100)), ("ERR_UNSUPPORTED", "multiples of 8", dict(d_v=264)),
          ("ERR_UNSUPPORTED", "multiples of 8", dict(d_v=0)), ("ERR_ARG", "strides", dict(k_strides=(16 * 1024, 100, 2048))),
          ("ERR_ARG", "strides", dict(v_strides=(16 * 1024 + 4, 128, 2048)))]


@pytest.mark.parametrize("code,word,kw", CACHES)
def test_cache_refusals(flh, code, word, kw):
    refused(flh, getattr(flh, code), word, flh.paged_attn, cache(flh, **kw), attn(flh), S)
    refused(flh, getattr(flh, code), word, flh.rope_kv_append, None, cache(flh, **kw), append(flh), S)
    assert flh.paged_attn_ws_bytes(cache(flh, **kw), attn(flh)) == 0


@pytest.mark.parametrize("code,word,kw", [
    ("ERR_ARG", "dtype", dict(dtype=7)), ("ERR_UNSUPPORTED", "cache's dtype", dict(dtype=2)),
    ("ERR_ARG", "multiple of n_kv_head", dict(n_head=12)), ("ERR_ARG", "multiple of n_kv_head", dict(n_head=0)),
    ("ERR_ARG", "scale", dict(scale=-1.0)), ("ERR_ARG", "scale", dict(scale=math.nan)), ("ERR_ARG", "scale", dict(scale=math.inf)),
    ("ERR_ARG", "window", dict(causal=0, window=5)), ("ERR_UNSUPPORTED", "table_stride", dict(table_stride=1 << 28)),
    ("ERR_UNSUPPORTED", "n_tok", dict(n_tok=1 << 30)), ("ERR_ARG", "element aligned", dict(q=None)),
    ("ERR_ARG", "element aligned", dict(out=FAR + 2)), ("ERR_ARG", "q_start", dict(q_start=None)),
    ("ERR_ARG", "q_start", dict(kv_len=P + 2)), ("ERR_ARG", "q_start", dict(table=None)),
    ("ERR_ARG", "overlaps", dict(out=P + 4096))])
def test_attn_refusals(flh, code, word, kw):
    refused(flh, getattr(flh, code), word, flh.paged_attn, cache(flh), attn(flh, **kw), S)


def test_attn_workspace_refusals(flh):
    need = flh.paged_attn_ws_bytes(cache(flh), attn(flh))
    if need == 0:
        pytest.skip("no workspace for this shape")
    for kw in (dict(ws=None), dict(ws=P + 8), dict(ws_bytes=need - 1)):
        refused(flh, flh.ERR_ARG, "ws", flh.paged_attn, cache(flh), attn(flh, **kw), S)


@pytest.mark.parametrize("code,word,kw", [
    ("ERR_ARG", "dtype", dict(dtype=3)), ("ERR_ARG", "k and v", dict(k=None)), ("ERR_ARG", "k and v", dict(v=P + 2)),
    ("ERR_ARG", "slot", dict(slot=None)), ("ERR_ARG", "slot", dict(slot=P + 1)), ("ERR_ARG", "n_head", dict(n_head=70000)),
    ("ERR_ARG", "non-null", dict(q=None)), ("ERR_ARG", "overlaps", dict(q_out=P + 64)), ("ERR_ARG", "overlaps", dict(qo_tok=4096))])
def test_append_refusals(flh, code, word, kw):
    refused(flh, getattr(flh, code), word, flh.rope_kv_append, None, cache(flh), append(flh, **kw), S)


@pytest.mark.parametrize("code,word,kw", [
    ("ERR_UNSUPPORTED", "power of two", dict(page_size=48)), ("ERR_ARG", "null", dict(held=None)),
    ("ERR_ARG", "null", dict(taken=None)), ("ERR_ARG", "null", dict(free_pages=None)), ("ERR_ARG", "null", dict(slot=None)),
    ("ERR_ARG", "null", dict(table_stride=0)), ("ERR_ARG", "aligned", dict(add=P + 2)), ("ERR_ARG", "aligned", dict(info=P + 1)),
    ("ERR_UNSUPPORTED", "table_stride", dict(table_stride=1 << 28))])
def test_plan_refusals(flh, code, word, kw):
    refused(flh, getattr(flh, code), word, flh.kv_plan, plan(flh, **kw), S)


def test_null_structs(flh):
    L = flh.lib()
    assert L.flh_kv_plan(None, None) == flh.ERR_ARG
    assert L.flh_paged_attn(None, C.byref(attn(flh)), None) == flh.ERR_ARG
    assert L.flh_paged_attn(C.byref(cache(flh).c), None, None) == flh.ERR_ARG
    assert L.flh_paged_attn_ws_bytes(C.byref(cache(flh).c), None) == 0
    assert L.flh_rope_kv_append(None, C.byref(cache(flh).c), None, None) == flh.ERR_ARG
    assert L.flh_rope(None, 0, P, 1, 1, P, 1, 1, 1, 1, 64, P, 1, None) == flh.ERR_ARG


@pytest.mark.parametrize("kw", [dict(n_rot=7), dict(n_rot=0), dict(n_rot=2048), dict(n_rot=8, n_axis=0), dict(n_rot=8, n_axis=9),
                                dict(n_rot=8, base=0.0), dict(n_rot=8, base=math.inf), dict(n_rot=8, layout=2),
                                dict(n_rot=8, freq=[1.0, math.nan, 1.0, 1.0]), dict(n_rot=8, axis=[0, 1, 0, 0]),
                                dict(n_rot=8, n_axis=3, axis=[0, 1, 2, 3]), dict(n_rot=8, first=70000)])
def test_rope_table_refusals(flh, kw):
    refused(flh, flh.ERR_ARG, "rope table", lambda: flh.RopeTable(**kw))


def test_rope_table_sizes(flh):
    for kw in (dict(freq=[1.0]), dict(axis=[0, 0, 0])):
        with pytest.raises(ValueError):
            flh.RopeTable(8, **kw)
