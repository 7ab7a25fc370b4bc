"""Outputs in the same rows as the inputs: other columns of them, or beside each head, are
apart; what shares a byte is refused (before any device work)."""
import numpy as np
import pytest
import torch

from paged_cases import TORCH, attn_bound, attn_oracle, get, put
from test_paged_args import P, S, attn, cache, refused


# four-byte elements, heads of 128, 32 of them (4096 elements a row of q)
@pytest.mark.parametrize("kw", [
    dict(q_tok=8192, o_tok=8192, out=P + 4 * 4095), dict(q_tok=8191, o_tok=8191, out=P + 4 * 4096),   # the columns run into q's, at either end
    dict(q_tok=8192, o_tok=8200, out=P + 4 * 4096), dict(q_tok=4096, o_tok=4096, out=P + 4 * 4096),   # other rows; the next row of q itself
    dict(q_head=256, q_tok=8192, o_head=256, o_tok=8192, out=P + 4 * 120), dict(q_head=256, q_tok=8192, o_head=256, o_tok=8192, out=P + 4 * 129),
    dict(q_head=256, q_tok=8192, o_head=384, o_tok=12288, out=P + 4 * 128), dict(q_tok=0, o_tok=0, out=P)])
def test_attention_refusals(flh, kw):
    refused(flh, flh.ERR_ARG, "overlaps", flh.paged_attn, cache(flh), attn(flh, **kw), S)


ROWS = ["columns", "columns in front", "beside each head", "one token"]


def layout(how, heads, d, dv, n):
    """(elements of a row, (offset, head stride) of q, of out)."""
    if how == "beside each head":
        return heads * (d + dv), (0, d + dv), (d, d + dv)
    if how == "columns in front":
        return heads * (d + dv) + 24, (heads * dv + 8, d), (0, dv)
    return heads * (d + dv) + 24, (0, d), (heads * d + 8, dv)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ROWS)
@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("BF16", "BF16")])
@pytest.mark.parametrize("n", [1, 30])
def test_attention_in_rows_of_q(flh, gpu, how, act, cdt, n):
    from test_gpu_paged_attn import Case
    heads, d, dv = 6, 64, 40
    c = Case(flh, gpu, act, cdt, heads, 2, d, dv, 16, "head", [(n, 200)] if how == "one token" else [(n, 200), (n, 77)], 70, spare_rows=0)
    row, (q0, qh), (o0, oh) = layout(how, heads, d, dv, n)
    x = torch.full((c.n_tok, row), 3.0, dtype=TORCH[act])
    q, o = [torch.as_strided(x, (c.n_tok, heads, w), (row, h, 1), at) for at, h, w in ((q0, qh, d), (o0, oh, dv))]
    q.copy_(c.q)
    b, el = put(flh, gpu, x), x.element_size()
    c.p.q, c.p.out, c.p.q_tok, c.p.o_tok, c.p.q_head, c.p.o_head = b.ptr + q0 * el, b.ptr + o0 * el, row, row, qh, oh
    c.run()
    got = get(b, x, gpu)
    out, mag, amp = attn_oracle(c.q, c.rows, c.kv_len, c.table, c.cache, c.group, c.scale, True, 0)
    have = torch.as_strided(got, o.shape, o.stride(), o0).double()
    assert ((have - out).abs() <= attn_bound(out, mag, amp, act, d, 200)).all()
    rest = torch.ones(x.shape, dtype=torch.bool)
    torch.as_strided(rest, o.shape, o.stride(), o0).fill_(False)
    assert torch.equal(got[rest], x[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("how", ROWS)
@pytest.mark.parametrize("dtype", ["F32", "BF16"])
def test_rope_in_rows_of_x(flh, gpu, how, dtype):
    from test_gpu_rope import bound, freqs, turned
    heads, d, n = 5, 64, 1 if how == "one token" else 19
    rng = np.random.default_rng(71)
    row, (x0, xh), (y0, yh) = layout(how, heads, d, d, n)
    buf = torch.full((n, row), 3.0, dtype=TORCH[dtype])
    x, y = [torch.as_strided(buf, (n, heads, d), (row, h, 1), at) for at, h in ((x0, xh), (y0, yh))]
    x.copy_(torch.from_numpy(rng.standard_normal((n, heads, d))).to(TORCH[dtype]))
    pos = rng.integers(0, 1000, (1, n)).astype(np.int32)
    b, bp, el = put(flh, gpu, buf), put(flh, gpu, torch.from_numpy(pos)), buf.element_size()
    t = flh.RopeTable(d)
    flh.rope(t, flh.Dtype[dtype], b.ptr + x0 * el, row, xh, b.ptr + y0 * el, row, yh, n, heads, d, bp, n, gpu)
    got = get(b, buf, gpu)
    want, mag = turned(x.double().numpy(), pos, freqs(d, 10000.0), [0] * 32, 0, True)
    err = np.abs(torch.as_strided(got, y.shape, y.stride(), y0).double().numpy() - want)
    assert (err <= bound(want, mag, dtype)).all()
    rest = torch.ones(buf.shape, dtype=torch.bool)
    torch.as_strided(rest, y.shape, y.stride(), y0).fill_(False)
    assert torch.equal(got[rest], buf[rest])
    t.close()
