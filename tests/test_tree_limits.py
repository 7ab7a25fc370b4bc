"""Sizes that could pass what the kernels count, or take too long, are refused; those that cannot are not."""
import pytest

from test_paged_args import S, attn, cache, refused
from test_spec_args import tree, tree_plan


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


@pytest.mark.parametrize("n_tok,stride,ok", [(1 << 22, 1, True), ((1 << 22) + 1, 1, False), (0xFFFFFFFF, 1, False), (1 << 20, 16, True),
                                             (1 << 20, 17, False), (80_000, 2500, True), (100_000, 32768, False), (1 << 14, 32768, True)])
def test_plans_end(flh, n_tok, stride, ok):
    """A plan whose walks, if all rows were one line, would not end for minutes is refused: squares of rows times words."""
    p = tree_plan(flh, n_tok=n_tok, mask_stride=stride, q_start=None)
    if ok:                                                    # (the next check refuses it: nothing is launched)
        refused(flh, flh.ERR_ARG, "null", flh.tree_plan, p, S)
    else:
        refused(flh, flh.ERR_UNSUPPORTED, "n_tok", flh.tree_plan, p, S)
