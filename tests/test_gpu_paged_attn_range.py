"""Attention at the ends of fp32's range: infinite keys, rows all of whose scores
are -infinity, and finite scores that pass the range only when they are turned
into powers of two."""
import math

import numpy as np
import pytest
import torch

from paged_cases import NONE, TORCH, attn_bound, attn_oracle, raw
from test_gpu_paged_attn import Case, TYPES

pytestmark = pytest.mark.gpu
# (heads of 64 and 128; rows a request: single tokens, 17 to 32 rows a kv head, prompts)
SHAPES = [(64, 1), (64, 6), (64, 40), (128, 1), (128, 7), (128, 40)]


def push(c):
    c.cache.push()
    c.b["q"].upload(raw(c.qbuf), c.s)


def heads_of(c, got):
    return got[:, :c.heads * c.dv].unflatten(1, (c.heads, c.dv)).double()


def token(c, s, j):
    return int(c.table[s, j // c.cache.page]), j % c.cache.page


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("d,n", SHAPES)
@pytest.mark.parametrize("finite", [0, 1, 3])
def test_infinite_keys(flh, gpu, act, cdt, d, n, finite):
    """Element 5 of kv head 0's keys of request 0 is infinite but in `finite` of them.  Head 0's
    queries are negative there (scores of -infinity: no weight; not a number where a row sees no
    other key), head 1's positive (not a number where a row sees one), and request 1 is
    untouched."""
    c = Case(flh, gpu, act, cdt, 8, 2, d, d, 16, "head", [(n, 150), (n, n + 20)], 40)
    keep = [10, 77, 149][:finite]
    for j in range(150):
        if j not in keep:
            c.cache.view[0][(*token(c, 0, j), 0, 5)] = math.inf
    c.q[:, 0, 5], c.q[:, 1, 5] = -1.25, 0.75
    push(c)
    c.run()
    got = heads_of(c, c.result())
    scores = c.q[:n].double()
    for i in range(n):
        seen = [j for j in keep if j <= 150 - n + i]
        assert torch.isnan(got[i, 1]).all(), i
        if not seen:
            assert torch.isnan(got[i, 0]).all(), i
            continue
        k = torch.stack([c.cache.view[0][(*token(c, 0, j), 0)] for j in seen]).double()
        v = torch.stack([c.cache.view[1][(*token(c, 0, j), 0)] for j in seen]).double()
        t = k @ scores[i, 0] * c.scale
        w = torch.softmax(t, 0)
        amp = (k.abs() @ scores[i, 0].abs()).max() * c.scale
        lim = attn_bound(w @ v, w @ v.abs(), amp, act, d, 150)
        assert ((got[i, 0] - w @ v).abs() <= lim).all(), i
    # kv head 1 of the request and the other request are as ever
    c.cache.view[0][torch.isinf(c.cache.view[0])] = 0.0
    out, mag, amp = attn_oracle(c.q, c.rows, c.kv_len, c.table, c.cache, c.group, c.scale, True, 0)
    lim = attn_bound(out, mag, amp, act, d, 150)
    ok = (got - out).abs() <= lim
    assert ok[:n, 4:].all() and ok[n:2 * n].all()


def large(act, cdt):
    """(query element, key element, scale) whose product is 2^127, exactly."""
    q, k = {("F32", "F16"): (2.0 ** 112, 2.0 ** 15), ("F32", "BF16"): (2.0 ** 64, 2.0 ** 63), ("F16", "F16"): (2.0 ** 14, 2.0 ** 15),
            ("BF16", "BF16"): (2.0 ** 64, 2.0 ** 63)}[act, cdt]
    return q, k, 2.0 ** 127 / (q * k)


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("d,n", SHAPES)
@pytest.mark.parametrize("keys", [150, 9001])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_near_the_end_of_fp32(flh, gpu, act, cdt, d, n, keys, sign):
    """Scores of up to 1.9 * 2^127 are finite, times log2(e) they are not.  They lie far
    apart, so a row is the value of its largest key, bit for bit; with sign -1 all of
    them are negative.  The rows of request 1 have ordinary scores."""
    c = Case(flh, gpu, act, cdt, 8, 2, d, d, 16, "head", [(n, keys), (n, n + 20)], 41)
    q, k, scale = large(act, cdt)
    c.scale = c.p.scale = scale
    c.q.zero_()
    c.q[:n, :, 3] = q
    c.cache.view[0].zero_()
    rng = np.random.default_rng(42)
    factor = sign * (1.0 + rng.integers(32, 58, keys) / 64.0)      # 1.5 .. 1.9
    best = [keys - n - 3, keys - n // 2 - 1, keys - 1]               # ever larger; the later rows see more of them
    factor[best] = [1.90625, 1.921875, 1.9375] if sign > 0 else [-1.484375, -1.46875, -1.453125]
    for j in range(keys):
        c.cache.view[0][(*token(c, 0, j), slice(None), 3)] = k * factor[j]
    push(c)
    c.run()
    got = heads_of(c, c.result())
    for i in range(n):
        j = max(b for b in best if b <= keys - n + i)
        for h in range(8):
            want = c.cache.view[1][(*token(c, 0, j), h // 4)].to(TORCH[act]).double()
            assert torch.equal(got[i, h], want), (i, h, j)
    # queries of zeros: the mean
    out, mag, _ = attn_oracle(c.q, c.rows, c.kv_len, c.table, c.cache, c.group, 0.0, True, 0)
    lim = attn_bound(out, mag, torch.zeros(out.shape[:2], dtype=torch.float64), act, d, n + 20)
    assert ((got - out).abs() <= lim)[n:2 * n].all()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n", [1, 6, 40])
def test_no_page_is_not_no_weight(flh, gpu, act, cdt, n):
    """Next to a row that is not a number: rows whose keys have no page, long enough to be
    split, and rows in front of the first key are zeros."""
    c = Case(flh, gpu, act, cdt, 8, 2, 64, 64, 16, "head", [(n, 9000), (n, n // 2), (n, 60)], 43)
    c.table[0, :] = NONE
    c.b["table"].upload(c.table.view(np.uint8).reshape(-1), gpu)
    for j in range(60):
        c.cache.view[0][(*token(c, 2, j), 0, 5)] = math.inf
    c.q[:, 0, 5] = -1.25
    push(c)
    c.run()
    got = heads_of(c, c.result())
    assert (got[:n] == 0).all() and (got[n:n + n - n // 2] == 0).all()
    assert torch.isnan(got[2 * n:3 * n, 0]).all()
    assert torch.isfinite(got[2 * n:3 * n, 4:]).all()


@pytest.mark.parametrize("cdt,size", [("F16", 1e37), ("BF16", 1e37), ("F16", 1e-37)])
@pytest.mark.parametrize("n", [2, 6, 40])
@pytest.mark.parametrize("keys", [150, 9001])
def test_rows_done_again_at_any_size(flh, gpu, cdt, size, n, keys):
    """Rows that are done again beside one that is not a number hold what they would hold
    alone, also where q.k passes the range of fp32 and scale q.k does not."""
    c = Case(flh, gpu, "F32", cdt, 4, 2, 64, 64, 16, "head", [(n, keys), (n, n)], 44, scale=0.1 / size)
    c.q *= size
    if size > 1:
        c.cache.view[0].mul_(50.0)                     # q.k of up to about 1e39 and more
        c.scale = c.p.scale = 0.002 / size
    for j in (keys - 1, keys - 2):
        c.cache.view[1][(*token(c, 0, j), 0, 9)] = math.nan
    push(c)
    c.run()
    got = heads_of(c, c.result())[:c.n_tok]
    out, mag, amp = [t[:c.n_tok] for t in attn_oracle(c.q, c.rows, c.kv_len, c.table, c.cache, c.group, c.scale, True, 0)]
    lim = attn_bound(out, mag, amp, "F32", 64, keys)
    nan = torch.isnan(out)
    assert nan.any() and torch.equal(torch.isnan(got), nan)
    assert ((got - out).abs() <= lim)[~nan].all()
