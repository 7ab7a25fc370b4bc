"""Attention with n_tok inside a request's rows: the rows in front of it stand where
they would without the cut, and those behind it are left as they are."""
import numpy as np
import pytest
import torch

from paged_cases import attn_bound, attn_oracle
from test_gpu_paged_attn import Case, TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 9), (False, 0)])
@pytest.mark.parametrize("lens,n_tok", [([(16, 16)], 10), ([(3, 40), (5, 300), (4, 9)], 5), ([(70, 90), (200, 500), (50, 60)], 133),
                                        ([(40, 5000), (300, 700)], 41), ([(8, 3)], 6)])
def test_rows_behind_the_cut(flh, gpu, act, cdt, causal, window, lens, n_tok):
    c = Case(flh, gpu, act, cdt, 8, 2, 64, 64, 16, "head", lens, 50, causal=causal, window=window)
    c.p.n_tok = n_tok
    c.ws()
    c.run()
    got = c.result()
    out, mag, amp = attn_oracle(c.q, c.rows, c.kv_len, c.table, c.cache, c.group, c.scale, causal, window)
    have = got[:, :8 * 64].unflatten(1, (8, 64)).double()
    lim = attn_bound(out, mag, amp, act, 64, int(c.kv_len.max()))
    assert ((have - out).abs() <= lim)[:n_tok].all()
    assert torch.equal(got[n_tok:], c.out0[n_tok:])


@pytest.mark.parametrize("max_q", [1, 100])
def test_far_ends_of_a_request(flh, gpu, max_q):
    """A q_start far behind n_tok: the rows stand in front of the first key and see nothing."""
    c = Case(flh, gpu, "F32", "F16", 4, 2, 64, 64, 16, "head", [(20, 60)], 51)
    for end in (1 << 30, 0x80000005, 0xFFFFFFFF):
        c.b["start"].upload(np.array([0, end], np.uint32), gpu)
        c.p.max_q = max_q
        c.ws()
        c.run()
        assert (c.result()[:20, :4 * 64] == 0).all()
