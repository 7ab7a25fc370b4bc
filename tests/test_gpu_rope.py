"""Rotary positions and the cache append against the formula in 64 bits."""
import math

import numpy as np
import pytest
import torch

from paged_cases import Cache, NONE, TORCH, get, half_step, put

pytestmark = pytest.mark.gpu


def turned(x, pos, freq, axis, first, halves):
    """x [token][head][d] float64; freq radians per position; returns the result
    and |a| + |b| of each element's pair (0 where nothing turns)."""
    p = len(freq)
    ang = np.stack([pos[axis[i]].astype(np.float64) * freq[i] for i in range(p)], 1)[:, None, :]
    i = np.arange(p)
    ia, ib = (first + i, first + i + p) if halves else (first + 2 * i, first + 2 * i + 1)
    y, mag = x.copy(), np.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * np.cos(ang) - b * np.sin(ang), a * np.sin(ang) + b * np.cos(ang)
    mag[..., ia] = mag[..., ib] = np.abs(a) + np.abs(b)
    return y, mag


def bound(y, mag, dtype):
    """cos and sin are off by at most 3 * 2^-24 (an angle error of 2 pi 2^-33, its
    float's rounding of at most pi/4 2^-24, and 2 ulp of sincospi below 1); the
    two products and their sum round once each: (|a| + |b|) * 6 * 2^-24.  Then one
    rounding to the result's type."""
    e = mag * 6 * 2.0 ** -24
    u = half_step(dtype) if dtype != "F32" else 0.0
    return e + (np.abs(y) + e) * u + {"F32": 2.0 ** -126, "F16": 2.0 ** -25, "BF16": 2.0 ** -126}[dtype]


def freqs(n_rot, base):
    return np.array([base ** (-2.0 * i / n_rot) for i in range(n_rot // 2)])


ROPE = [
    # dtype, tokens, heads, d, n_rot, first, layout, axes, far, stride pad, base offset (elements)
    ("F32", 1, 32, 128, 128, 0, "HALVES", 1, 8192, 0, 0), ("F32", 1, 1, 64, 64, 0, "PAIRS", 1, 100, 0, 0),
    ("F32", 7, 3, 128, 64, 0, "PAIRS", 1, 1 << 20, 0, 0), ("F32", 5, 16, 192, 64, 128, "PAIRS", 1, 1 << 20, 8, 0),
    ("F16", 33, 5, 128, 128, 0, "HALVES", 3, 4096, 0, 0), ("BF16", 33, 5, 128, 128, 0, "HALVES", 3, 4096, 8, 0),
    ("BF16", 9, 7, 80, 40, 20, "HALVES", 2, 50000, 0, 0), ("F16", 9, 7, 80, 40, 20, "PAIRS", 2, 50000, 4, 4),
    ("F32", 6, 2, 50, 22, 3, "HALVES", 1, 1000, 1, 1), ("BF16", 6, 2, 50, 22, 3, "PAIRS", 1, 1000, 1, 1),
    ("F16", 6, 2, 51, 24, 7, "HALVES", 3, 1000, 3, 0), ("F32", 3, 4, 1200, 1024, 100, "HALVES", 8, 1000, 0, 0),
    ("F32", 300, 9, 96, 96, 0, "HALVES", 1, 2 ** 31 - 1, 0, 0), ("BF16", 700, 40, 256, 256, 0, "HALVES", 1, 2000, 0, 0),
    ("F32", 2, 2, 2, 2, 0, "PAIRS", 1, 100, 0, 0)]


@pytest.mark.parametrize("dtype,n,heads,d,n_rot,first,layout,axes,far,pad,off", ROPE)
@pytest.mark.parametrize("in_place", [False, True])
def test_rope(flh, gpu, dtype, n, heads, d, n_rot, first, layout, axes, far, pad, off, in_place):
    rng = np.random.default_rng(n * 100 + d)
    base = 500000.0
    axis = rng.integers(0, axes, n_rot // 2)
    pos = rng.integers(-far // 3, far, (axes, n + 2)).astype(np.int32)
    row = heads * (d + pad) + pad
    x = torch.full((off + n * row + 16,), float("nan"), dtype=TORCH[dtype])
    view = torch.as_strided(x, (n, heads, d), (row, d + pad, 1), off)
    view.copy_(torch.from_numpy(rng.standard_normal((n, heads, d)) * 2).to(TORCH[dtype]))
    bx, bp = put(flh, gpu, x), put(flh, gpu, torch.from_numpy(pos))
    y0 = torch.full_like(x, 7.0)
    by = bx if in_place else put(flh, gpu, y0)
    t = flh.RopeTable(n_rot, base=base, axis=axis, n_axis=axes, first=first, layout=flh.RopeLayout[layout])
    el = x.element_size()
    flh.rope(t, flh.Dtype[dtype], bx.ptr + off * el, row, d + pad, by.ptr + off * el, row, d + pad, n, heads, d, bp, n + 2, gpu)
    got = get(by, x, gpu)
    want, mag = turned(view.double().numpy(), pos[:, :n], freqs(n_rot, base), axis, first, layout == "HALVES")
    err = np.abs(torch.as_strided(got, (n, heads, d), (row, d + pad, 1), off).double().numpy() - want)
    assert (err <= bound(want, mag, dtype)).all(), err.max()
    # what lies between the heads stays
    rest = torch.ones(len(x), dtype=torch.bool)
    torch.as_strided(rest, (n, heads, d), (row, d + pad, 1), off).fill_(False)
    keep = x if in_place else y0
    assert torch.equal(got[rest].view(torch.uint8), keep[rest].view(torch.uint8))
    t.close()


def test_rope_frequencies_and_inverse(flh, gpu):
    """Frequencies of the caller's own; a turn forward and one back is the identity
    to the roundings of both."""
    rng = np.random.default_rng(3)
    n, d = 20, 64
    freq = rng.uniform(0, 3.5, 32)
    pos = rng.integers(0, 100000, (1, n)).astype(np.int32)
    x = rng.standard_normal((n, 1, d)).astype(np.float32)
    bx, b1, b2 = put(flh, gpu, torch.from_numpy(x)), put(flh, gpu, torch.from_numpy(pos)), put(flh, gpu, torch.from_numpy(-pos))
    t = flh.RopeTable(d, freq=freq)
    flh.rope(t, flh.Dtype.F32, bx, d, d, bx, d, d, n, 1, d, b1, n, gpu)
    y = bx.download(np.float32, n * d, gpu).reshape(n, 1, d)
    want, mag = turned(x.astype(np.float64), pos, freq, [0] * 32, 0, True)
    assert (np.abs(y - want) <= bound(want, mag, "F32")).all()
    flh.rope(t, flh.Dtype.F32, bx, d, d, bx, d, d, n, 1, d, b2, n, gpu)
    z = bx.download(np.float32, n * d, gpu).reshape(n, 1, d)
    back, mag2 = turned(y.astype(np.float64), -pos, freq, [0] * 32, 0, True)
    assert (np.abs(z - back) <= bound(back, mag2, "F32")).all()
    assert (np.abs(z - x) <= 2 * bound(want, mag, "F32") + bound(back, mag2, "F32")).all()


APPEND = [
    # act, cache, tokens, heads, kv heads, dk, dv, n_rot (0: no table), first, layout, axes, page, order, cache pad, column pad
    ("F32", "F16", 1, 32, 8, 128, 128, 128, 0, "PAIRS", 1, 16, "head", 0, 0),
    ("F32", "BF16", 37, 32, 8, 128, 128, 128, 0, "HALVES", 3, 16, "token", 0, 4),
    ("F16", "F16", 37, 14, 2, 64, 64, 64, 0, "HALVES", 1, 1, "head", 8, 0),
    ("BF16", "BF16", 100, 16, 16, 192, 128, 64, 128, "PAIRS", 1, 64, "head", 0, 0),
    ("F16", "BF16", 29, 3, 3, 80, 40, 40, 40, "HALVES", 2, 32, "token", 8, 1),
    ("BF16", "F16", 29, 0, 4, 256, 256, 256, 0, "PAIRS", 1, 128, "head", 0, 2),
    ("F32", "F16", 65, 6, 2, 96, 96, 0, 0, "HALVES", 1, 16, "token", 0, 3),
    ("F32", "F16", 3000, 8, 2, 128, 128, 128, 0, "HALVES", 1, 16, "head", 0, 0),
    ("F32", "F16", 3, 5, 1, 8, 16, 6, 1, "HALVES", 1, 2, "head", 0, 1),
]


@pytest.mark.parametrize("act,cdt,n,heads,hk,dk,dv,n_rot,first,layout,axes,page,order,cpad,xpad", APPEND)
def test_append(flh, gpu, act, cdt, n, heads, hk, dk, dv, n_rot, first, layout, axes, page, order, cpad, xpad):
    rng = np.random.default_rng(n * 10 + dk)
    n_pages = -(-(n + 7) // page) + 2
    cache = Cache(flh, gpu, cdt, n_pages, page, hk, dk, dv, order, cpad)
    row = (heads + hk) * dk + hk * dv + xpad
    x = torch.from_numpy(rng.standard_normal((n, row)) * 3).to(TORCH[act])
    slot = rng.permutation(n_pages * page)[:n].astype(np.uint32)
    slot[rng.random(n) < 0.1] = NONE
    if n > 20:
        slot[3] = n_pages * page                       # just behind the cache
        slot[4] = NONE - 1
    axis = rng.integers(0, axes, max(n_rot, 2) // 2)
    pos = rng.integers(0, 100000, (axes, n)).astype(np.int32)
    bx, bs, bp = put(flh, gpu, x), put(flh, gpu, torch.from_numpy(slot.view(np.int32))), put(flh, gpu, torch.from_numpy(pos))
    el = x.element_size()
    q_out = torch.full((n, max(heads, 1), dk), 5.0, dtype=TORCH[act])
    bq = put(flh, gpu, q_out)
    t = flh.RopeTable(n_rot, base=10000.0, axis=axis, n_axis=axes, first=first, layout=flh.RopeLayout[layout]) if n_rot else None
    p = flh.RopeKvP(q=bx.ptr, q_out=bq.ptr, k=bx.ptr + heads * dk * el, v=bx.ptr + (heads + hk) * dk * el,
                    pos=bp.ptr if n_rot else None, slot=bs.ptr, q_tok=row, q_head=dk, qo_tok=q_out.stride(0), qo_head=dk,
                    k_tok=row, k_head=dk, v_tok=row, v_head=dv, dtype=flh.Dtype[act], n_tok=n, n_head=heads, pos_stride=n)
    flh.rope_kv_append(t, cache.c, p, gpu)
    q = x[:, :heads * dk].reshape(n, heads, dk).double().numpy()
    k = x[:, heads * dk:(heads + hk) * dk].reshape(n, hk, dk).double().numpy()
    v = x[:, (heads + hk) * dk:(heads + hk) * dk + hk * dv].reshape(n, hk, dv)
    f = freqs(n_rot, 10000.0) if n_rot else []
    for src, got, dt in ((q, get(bq, q_out, gpu), act), (k, None, cdt)):
        want, mag = turned(src, pos, f, axis, first, layout == "HALVES") if n_rot else (src, np.zeros_like(src))
        if got is not None:
            if heads:
                assert (np.abs(got.double().numpy() - want) <= bound(want, mag, dt)).all()
            else:
                assert (got == 5.0).all()
            continue
        kc, vc = cache.pull()
        live = slot < n_pages * page
        pg, at = torch.from_numpy((slot[live] // page).astype(np.int64)), torch.from_numpy((slot[live] % page).astype(np.int64))
        err = np.abs(kc[pg, at].double().numpy() - want[live])
        assert (err <= bound(want, mag, dt)[live]).all(), err.max()
        assert torch.equal(vc[pg, at], v[torch.from_numpy(live)].to(TORCH[cdt]))
        # every other slot still holds what it held
        hit = torch.zeros(n_pages, page, dtype=torch.bool)
        hit[pg, at] = True
        assert torch.isnan(kc[~hit]).all() and torch.isnan(vc[~hit]).all()
    # in place: the queries turn where they lie, keys and values beside them stay
    if heads:
        p.q_out, p.qo_tok = p.q, row
        flh.rope_kv_append(t, cache.c, p, gpu)
        again = get(bx, x, gpu)
        assert torch.equal(again[:, :heads * dk].reshape(n, heads, dk), get(bq, q_out, gpu))
        assert torch.equal(again[:, heads * dk:], x[:, heads * dk:])
    if t:
        t.close()


def test_append_nothing(flh, gpu):
    cache = Cache(flh, gpu, "F16", 2, 16, 2, 64, 64)
    flh.rope_kv_append(None, cache.c, flh.RopeKvP(n_tok=0, n_head=4), gpu)
    gpu.sync()


def test_append_values_past_the_range(flh, gpu):
    """What a 16-bit cache cannot hold rounds to infinity, NaN stays NaN."""
    cache = Cache(flh, gpu, "F16", 1, 4, 1, 8, 8)
    x = torch.tensor([[1e6, -1e6, math.inf, math.nan, 65504.0, 65519.0, 65520.0, 1e-9]])
    bx, bs = put(flh, gpu, x), put(flh, gpu, torch.tensor([2], dtype=torch.int32))
    p = flh.RopeKvP(k=bx.ptr, v=bx.ptr, slot=bs.ptr, k_tok=8, k_head=8, v_tok=8, v_head=8, dtype=0, n_tok=1, n_head=0)
    flh.rope_kv_append(None, cache.c, p, gpu)
    for c in cache.pull():
        assert torch.equal(torch.nan_to_num(c[0, 2, 0].float(), nan=9.0), torch.nan_to_num(x[0].half().float(), nan=9.0))


# heads whose unturned part is cut by the turned one at odd multiples of the units
# of 16 bytes, and many heads of few tokens (shared by several workgroups)
UNITS = [("F32", 5, 3, 76, 64, 4, "HALVES", 1, 1000, 0, 0), ("F32", 5, 3, 76, 64, 8, "PAIRS", 2, 1000, 4, 4),
         ("F32", 3, 700, 12, 8, 4, "PAIRS", 1, 1000, 0, 0), ("F16", 4, 3, 88, 64, 8, "HALVES", 1, 1000, 0, 0),
         ("BF16", 4, 3, 104, 64, 24, "PAIRS", 1, 1000, 8, 8), ("BF16", 1, 300, 136, 16, 120, "PAIRS", 3, 1000, 0, 8),
         ("F16", 2, 65, 16, 16, 0, "PAIRS", 1, 1000, 0, 0), ("F32", 513, 33, 132, 128, 0, "HALVES", 1, 1000, 0, 0)]


@pytest.mark.parametrize("case", UNITS)
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_units(flh, gpu, case, in_place):
    test_rope(flh, gpu, *case, in_place)


def test_rope_more_tokens_than_a_launch(flh, gpu):
    """2^24 + 5 tokens of one pair: rows at both ends and around 2^22 and 2^24."""
    n = (1 << 24) + 5
    x = torch.arange(2 * n, dtype=torch.float32).remainder_(251).to(torch.float16)
    pos = (torch.arange(n, dtype=torch.int64) * 7919 % 100003).to(torch.int32)
    bx, bp = put(flh, gpu, x), put(flh, gpu, pos)
    t = flh.RopeTable(2, base=10.0)
    flh.rope(t, flh.Dtype.F16, bx, 2, 2, bx, 2, 2, n, 1, 2, bp, n, gpu)
    got = get(bx, x, gpu)
    rows = np.concatenate([np.arange(c - 5, c + 5) for c in (5, 1 << 22, 1 << 23, 3 << 22, 1 << 24)])
    want, mag = turned(x.reshape(n, 1, 2)[rows].double().numpy(), pos[rows][None].numpy(), np.array([1.0]), [0], 0, True)
    err = np.abs(got.reshape(n, 1, 2)[rows].double().numpy() - want)
    assert (err <= bound(want, mag, "F16")).all(), err.max()
    t.close()
