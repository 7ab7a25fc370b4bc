"""Attention counts its units of work in 32 bits: calls whose units could pass that are refused, those that cannot are not."""
import pytest

from test_paged_args import S, attn, cache, refused
from test_spec_args import tree


@pytest.mark.parametrize("tree_form", [False, True])
@pytest.mark.parametrize("keys,n_seq,n_tok", [(64, 80_000_000, 80_000_000), (4096, 3_500_000, 7_000_000), (1 << 30, 18, 46)])
def test_units(flh, keys, n_seq, n_tok, tree_form):
    """Strips of 16 rows, one more a request than it has full ones, of tiles of 64 keys; 4 units more a strip."""
    page = 4096 if keys > 4096 else 64
    a = dict(n_seq=n_seq, n_tok=n_tok, max_q=1, table_stride=keys // page, n_head=8)
    c = cache(flh, page_size=page)
    units = 8 * (n_tok / 16 + n_seq) * (keys / 64 + 1 + 4)
    call = (lambda p: flh.tree_attn(c, p, tree(flh), S)) if tree_form else (lambda p: flh.paged_attn(c, p, S))
    assert 2.0e9 < units < 1 << 32
    # refused for its workspace, after the count: there is none
    few = {**a, "n_seq": n_seq // 2 - n_tok // 32, "n_tok": n_tok}
    refused(flh, flh.ERR_ARG, "ws", call, attn(flh, **few, ws_bytes=0, out=1 << 50))
    # more than 32 bits
    more = {**a, "n_seq": 2 * n_seq}
    assert 8 * (n_tok / 16 + 2 * n_seq) * (keys / 64 + 1 + 4) > 4.0e9
    refused(flh, flh.ERR_UNSUPPORTED, "too much work", call, attn(flh, **more, out=1 << 50))
