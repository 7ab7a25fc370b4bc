"""Refusals of the tree, verification and page entry points: checked before any device
work, so they hold without a GPU."""
import ctypes as C

import pytest

from test_paged_args import FAR, P, S, attn, cache, refused


def tree_plan(flh, **kw):
    a = dict(q_start=P, parent=P, kv_len=P, mask=P, depth=P, pos=P, n_seq=2, n_tok=9, mask_stride=1, window=0)
    a.update(kw)
    return flh.TreePlanP(**a)


def tree(flh, **kw):
    a = dict(mask=P, depth=P, mask_stride=1)
    a.update(kw)
    return flh.TreeP(**a)


def verify(flh, **kw):
    a = dict(target=P, draft=FAR, q_start=P, token=P, parent=P, inv_temp=P, u_accept=P, u_next=P, kv_len=P, n_path=P, path=P,
             next=P, logp=P, len=P, ws=P, ws_bytes=1 << 40, t_row=1000, d_row=1000, dtype=0, n_seq=2, n_tok=9, vocab=1000,
             path_stride=5, max_child=2)
    a.update(kw)
    return flh.VerifyP(**a)


def compact(flh, **kw):
    a = dict(q_start=P, slot=P, n_path=P, path=P, n_seq=2, n_tok=9, path_stride=5)
    a.update(kw)
    return flh.KvCompactP(**a)


PAGES = dict(kv_len=P, table=P, free_pages=P, taken=P, shared=P, copy_src=P, copy_dst=P, copy_n=P, info=P, n_seq=4, n_pages=64,
             page_size=16, n_free=8, table_stride=4)


def fork(flh, **kw):
    return flh.KvForkP(**{**PAGES, "src": P, "dst": P, "len": P, "n_fork": 2, **kw})


def trim(flh, **kw):
    return flh.KvTrimP(**{**PAGES, "keep": P, "held": P, **kw})


@pytest.mark.parametrize("word,kw", [
    ("mask_stride", dict(mask_stride=0)), ("mask_stride", dict(mask_stride=32769)), ("null", dict(q_start=None)),
    ("null", dict(parent=None)), ("null", dict(mask=None)), ("null", dict(depth=None)), ("null", dict(kv_len=None)),
    ("aligned", dict(parent=P + 2)), ("aligned", dict(pos=P + 1))])
def test_tree_plan_refusals(flh, word, kw):
    refused(flh, flh.ERR_ARG, word, flh.tree_plan, tree_plan(flh, **kw), S)


def test_sizes_that_are_too_large(flh):
    refused(flh, flh.ERR_UNSUPPORTED, "n_tok", flh.tree_plan, tree_plan(flh, n_tok=(1 << 30) + 1), S)
    refused(flh, flh.ERR_UNSUPPORTED, "n_fork", flh.kv_fork, fork(flh, n_fork=(1 << 21) + 1), S)
    for kw in (dict(n_tok=1 << 24, vocab=1), dict(n_seq=1 << 24, vocab=1), dict(n_tok=1 << 19, vocab=128256), dict(n_tok=0xFFFFFFFF, vocab=5)):
        refused(flh, flh.ERR_UNSUPPORTED, "rows", flh.spec_verify, verify(flh, **kw), S)


@pytest.mark.parametrize("word,kw,akw", [
    ("mask", dict(mask=None), {}), ("mask", dict(mask=P + 2), {}), ("mask_stride", dict(mask_stride=0), {}),
    ("mask_stride", dict(mask_stride=40000), {}), ("depth", dict(depth=None), dict(window=5)), ("depth", dict(depth=P + 1), {}),
    ("causal", {}, dict(causal=0)), ("scale", {}, dict(scale=-1.0)), ("overlaps", {}, dict(out=P + 4096)),
    ("multiple of n_kv_head", {}, dict(n_head=12)), ("ws", {}, dict(ws=None)), ("ws", {}, dict(ws_bytes=16))])
def test_tree_attn_refusals(flh, word, kw, akw):
    refused(flh, flh.ERR_ARG, word, flh.tree_attn, cache(flh), attn(flh, **akw), tree(flh, **kw), S)


def test_tree_attn_cache_refusals(flh):
    refused(flh, flh.ERR_UNSUPPORTED, "dtype", flh.tree_attn, cache(flh, dtype=0), attn(flh), tree(flh), S)
    assert flh.tree_attn_ws_bytes(cache(flh, dtype=0), attn(flh)) == 0
    for n in (1, 8, 9, 16, 17, 100):
        assert flh.tree_attn_ws_bytes(cache(flh), attn(flh, n_tok=n, max_q=n)) > 0


@pytest.mark.parametrize("code,word,kw", [
    ("ERR_ARG", "dtype", dict(dtype=3)), ("ERR_UNSUPPORTED", "vocab", dict(vocab=0)), ("ERR_UNSUPPORTED", "vocab", dict(vocab=(1 << 22) + 1)),
    ("ERR_ARG", "path_stride", dict(path_stride=0)), ("ERR_ARG", "max_child", dict(max_child=0)),
    ("ERR_ARG", "max_child", dict(max_child=65)), ("ERR_UNSUPPORTED", "rows", dict(n_tok=1 << 31, vocab=9000)),
    ("ERR_UNSUPPORTED", "rows", dict(n_seq=1 << 30, vocab=9000)), ("ERR_ARG", "null", dict(target=None)),
    ("ERR_ARG", "null", dict(q_start=None)), ("ERR_ARG", "null", dict(token=None)), ("ERR_ARG", "null", dict(u_accept=None)),
    ("ERR_ARG", "null", dict(u_next=None)), ("ERR_ARG", "null", dict(n_path=None)), ("ERR_ARG", "null", dict(path=None)),
    ("ERR_ARG", "null", dict(next=None)), ("ERR_ARG", "null", dict(kv_len=None)), ("ERR_ARG", "aligned", dict(token=P + 2)),
    ("ERR_ARG", "aligned", dict(logp=P + 1)), ("ERR_ARG", "element aligned", dict(target=P + 2)),
    ("ERR_ARG", "element aligned", dict(draft=P + 1)), ("ERR_ARG", "ws", dict(ws=None)), ("ERR_ARG", "ws", dict(ws=P + 8)),
    ("ERR_ARG", "ws", dict(ws_bytes=8))])
def test_verify_refusals(flh, code, word, kw):
    refused(flh, getattr(flh, code), word, flh.spec_verify, verify(flh, **kw), S)


def test_verify_workspace(flh):
    a = flh.spec_verify_ws_bytes(verify(flh, draft=None))
    b = flh.spec_verify_ws_bytes(verify(flh))
    assert 0 < a < b
    assert flh.spec_verify_ws_bytes(verify(flh, dtype=9)) == 0
    assert flh.VerifyP().max_child == 1


@pytest.mark.parametrize("kw", [dict(q_start=None), dict(slot=None), dict(n_path=None), dict(path=None), dict(path=P + 2)])
def test_compact_refusals(flh, kw):
    refused(flh, flh.ERR_ARG, "kv compact", flh.kv_compact, flh.KvCaches([cache(flh)]), compact(flh, **kw), S)


def test_caches_have_to_be_alike(flh):
    two = flh.KvCaches([cache(flh), cache(flh, n_pages=63)])
    refused(flh, flh.ERR_ARG, "alike", flh.kv_compact, two, compact(flh), S)
    refused(flh, flh.ERR_ARG, "alike", flh.kv_copy, two, P, P, P, 1, S)
    refused(flh, flh.ERR_ARG, "alike", flh.kv_copy, flh.KvCaches([cache(flh), cache(flh, v_strides=(16 * 1024, 1024, 128))]), P, P, P, 1, S)
    refused(flh, flh.ERR_ARG, "aligned", flh.kv_copy, flh.KvCaches([cache(flh), cache(flh, k=P + 8)]), P, P, P, 1, S)


@pytest.mark.parametrize("args", [(None, P, P), (P, None, P), (P, P, None), (P + 1, P, P)])
def test_copy_refusals(flh, args):
    refused(flh, flh.ERR_ARG, "kv copy", flh.kv_copy, flh.KvCaches([cache(flh)]), *args, 3, S)


@pytest.mark.parametrize("code,word,kw", [
    ("ERR_UNSUPPORTED", "power of two", dict(page_size=24)), ("ERR_ARG", "n_pages", dict(n_pages=1 << 29)),
    ("ERR_ARG", "null", dict(src=None)), ("ERR_ARG", "null", dict(dst=None)), ("ERR_ARG", "null", dict(kv_len=None)),
    ("ERR_ARG", "null", dict(table=None)), ("ERR_ARG", "null", dict(taken=None)), ("ERR_ARG", "null", dict(shared=None)),
    ("ERR_ARG", "null", dict(copy_n=None)), ("ERR_ARG", "null", dict(free_pages=None)), ("ERR_ARG", "null", dict(table_stride=0)),
    ("ERR_ARG", "aligned", dict(len=P + 2)), ("ERR_UNSUPPORTED", "n_fork", dict(n_fork=1 << 31))])
def test_fork_refusals(flh, code, word, kw):
    refused(flh, getattr(flh, code), word, flh.kv_fork, fork(flh, **kw), S)


@pytest.mark.parametrize("code,word,kw", [
    ("ERR_UNSUPPORTED", "power of two", dict(page_size=0)), ("ERR_ARG", "n_pages", dict(n_pages=1 << 29)),
    ("ERR_UNSUPPORTED", "table_stride", dict(n_seq=1 << 20, table_stride=1 << 11)), ("ERR_ARG", "null", dict(kv_len=None)),
    ("ERR_ARG", "null", dict(keep=None)), ("ERR_ARG", "null", dict(held=None)), ("ERR_ARG", "null", dict(table=None)),
    ("ERR_ARG", "null", dict(taken=None)), ("ERR_ARG", "null", dict(copy_dst=None)), ("ERR_ARG", "null", dict(free_pages=None)),
    ("ERR_ARG", "aligned", dict(keep=P + 2)), ("ERR_ARG", "aligned", dict(info=P + 1))])
def test_trim_refusals(flh, code, word, kw):
    refused(flh, getattr(flh, code), word, flh.kv_trim, trim(flh, **kw), S)


def test_null_structs(flh):
    L = flh.lib()
    assert L.flh_tree_plan(None, None) == flh.ERR_ARG
    assert L.flh_tree_attn(None, C.byref(attn(flh)), C.byref(tree(flh)), None) == flh.ERR_ARG
    assert L.flh_tree_attn(C.byref(cache(flh).c), None, C.byref(tree(flh)), None) == flh.ERR_ARG
    assert L.flh_tree_attn(C.byref(cache(flh).c), C.byref(attn(flh)), None, None) == flh.ERR_ARG
    assert L.flh_spec_verify(None, None) == flh.ERR_ARG and L.flh_spec_verify_ws_bytes(None) == 0
    assert L.flh_kv_compact(C.byref(cache(flh).c), 1, None, None) == flh.ERR_ARG
    assert L.flh_kv_copy(None, 1, P, P, P, 1, None) == flh.ERR_ARG
    assert L.flh_kv_fork(None, None) == flh.ERR_ARG and L.flh_kv_trim(None, None) == flh.ERR_ARG
