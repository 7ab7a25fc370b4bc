"""Free lists with entries that are no page: the tokens of those pages have no slot, and
info[1] counts them."""
import numpy as np
import pytest

from test_gpu_kv_plan import NONE, Plan, check, make_table, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [1, 16, 64, 65536])
@pytest.mark.parametrize("rows", [0, -37, 9000])
@pytest.mark.parametrize("taken", [0, 4])
def test_free_entries_that_are_no_page(flh, gpu, page, rows, taken):
    rng = np.random.default_rng(page + taken)
    n = 60
    held, add = rng.integers(0, 300, n).astype(np.uint32), rng.integers(0, 90, n).astype(np.uint32)
    width = -(-400 // page) + 1
    table, free = make_table(held, page, width, rng, 60 * width + 8)
    bad = np.array([NONE, NONE // page + 1 if page > 1 else NONE, 0x80000000 if page > 1 else NONE], np.uint32)
    at = rng.random(len(free)) < 0.3
    free[at] = rng.choice(bad, int(at.sum()))
    free = free[:max(8, len(free) - 40)]
    max_tok = int(add.sum()) + rows
    p = Plan(flh, gpu, held, add, page, free, taken, table, max_tok)
    want = oracle(held, add, page, free, taken, table, max_tok, p.slot0, p.pos0)
    for _ in range(2):
        flh.kv_plan(p.p, gpu)
        check(p.read(), want)


@pytest.mark.parametrize("page", [2, 16])
def test_the_slot_that_is_none(flh, gpu, page):
    """The last token of page 2^32 / page_size - 1 has the number that stands for no slot."""
    last = NONE // page
    held, add = np.array([1, 0, page - 1], np.uint32), np.array([page - 1, 2 * page, 3], np.uint32)
    table = np.full((3, 3), NONE, np.uint32)
    table[0, 0], table[2, 0] = last, last
    free = np.array([last, 3, last, last], np.uint32)
    p = Plan(flh, gpu, held, add, page, free, 0, table, int(add.sum()) + 2)
    want = oracle(held, add, page, free, 0, table, int(add.sum()) + 2, p.slot0, p.pos0)
    assert want["info"][1] >= 3
    flh.kv_plan(p.p, gpu)
    check(p.read(), want)
