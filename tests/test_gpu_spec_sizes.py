"""Sizes and arguments at the ends of what the operators of a speculative step take: more requests than a workgroup
looks at once, large trees and vocabularies, hints that are wrong, one array in two places."""
import numpy as np
import pytest
import torch

from test_gpu_kv_pages import Book
from test_gpu_spec_verify import Verify
from test_gpu_tree_attn import Tree, plan
from tree_cases import plan_oracle, random_parents

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_seq,window,stride", [(2047, 0, 1), (2048, 2, 1), (2049, 0, 3), (5000, 3, 1)])
def test_plans_of_many_requests(flh, gpu, n_seq, window, stride):
    rng = np.random.default_rng(n_seq)
    parents = [random_parents(int(n), rng, 3) for n in rng.integers(0, 8, n_seq)]
    kv = [len(p) + int(rng.integers(0, 900)) for p in parents]
    want = plan_oracle(parents, kv, stride, window)
    for lead in (0, 70):
        got = plan(flh, gpu, parents, kv, stride, window, lead)
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g[lead:lead + len(w)], w)


@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("F32", "BF16"), ("BF16", "BF16")])
@pytest.mark.parametrize("window", [0, 40])
def test_large_trees(flh, gpu, act, cdt, window):
    """Trees of several strips, whose bits are in ten words."""
    c = Tree(flh, gpu, act, cdt, 8, 2, 128, 128, 16, "head", [(300, 300), (7, 50), (290, 1500), (129, 2000)], 81, window=window, back=9)
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("BF16", "BF16")])
@pytest.mark.parametrize("n", [3, 14, 40])
@pytest.mark.parametrize("max_q", [0, 1, 4, 9, 16, 17, 33, 0xFFFFFFFF])
def test_any_max_q(flh, gpu, act, cdt, n, max_q):
    """max_q chooses the kernel; the results hold for any."""
    c = Tree(flh, gpu, act, cdt, 8, 2, 64, 64, 16, "token", [(n, n), (n, 600), (1, 9), (n, 3000)], 82, window=200)
    c.p.max_q = max_q
    c.ws()
    c.run()
    c.check()


@pytest.mark.parametrize("page", [4, 16])
def test_many_forks(flh, gpu, page):
    """More forks than a workgroup has threads, of partly filled pages, and all of them freed again."""
    rng = np.random.default_rng(page)
    b = Book(flh, gpu, page, 4000, 5, 14000, 83)
    for s in range(900):
        b.take(s, int(rng.integers(1, 3 * page)))
    b.fork(rng.integers(0, 900, 3000).tolist(), rng.permutation(np.arange(900, 3900)).tolist(), rng.integers(0, 3 * page, 3000))
    b.sound()
    b.trim(np.where(rng.random(4000) < 0.6, 0, rng.integers(0, 3 * page, 4000)).astype(np.uint32))
    b.sound()
    b.trim(np.zeros(4000, np.uint32))
    b.sound()
    assert b.taken == 0


@pytest.mark.parametrize("n_seq,width", [(1023, 3), (1025, 7), (3000, 5)])
def test_many_requests_trimmed_without_counts(flh, gpu, n_seq, width):
    rng = np.random.default_rng(n_seq)
    b = Book(flh, gpu, 16, n_seq, width, n_seq * width, 84, shared=False)
    for s in range(n_seq):
        b.take(s, int(rng.integers(0, 16 * width + 1)))
    b.trim(np.where(rng.random(n_seq) < 0.5, 0xFFFFFFFF, rng.integers(0, 16 * width, n_seq)).astype(np.uint32), held=True)
    b.trim(np.zeros(n_seq, np.uint32))
    assert b.taken == 0 and len(set(b.free.tolist())) == len(b.free)


@pytest.mark.parametrize("dtype", ["F32", "BF16"])
@pytest.mark.parametrize("draft", [False, True])
def test_the_largest_vocabulary(flh, gpu, draft, dtype):
    v = Verify(flh, gpu, [4, 1], 1 << 22, dtype, draft, 3, seed=85, peak=3.0).push()
    v.run()
    v.check()


def test_many_children(flh, gpu):
    """64 children a row, which nearly all fall."""
    for draft in (False, True):
        v = Verify(flh, gpu, [256, 70, 256], 300, "F32", draft, 64, seed=86, peak=1.0)
        v.u_accept[:] = 0.97 + 0.03 * v.u_accept
        v.push().run()
        v.check()


def test_one_row_of_logits_for_all(flh, gpu):
    """A stride of 0: every row has the same logits."""
    v = Verify(flh, gpu, [9, 4, 13], 5000, "F32", True, 3, seed=87, peak=3.0)
    v.target[:], v.draft[:] = v.target[0].clone(), v.draft[0].clone()
    v.push()
    v.p.t_row = v.p.d_row = 0
    v.run()
    v.check()


def test_len_in_place_of_kv_len(flh, gpu):
    for draft in (False, True):
        v = Verify(flh, gpu, [5, 0, 9, 1, 30], 9001, "F32", draft, 2, seed=88, peak=3.0).push()
        v.p.len = v.p.kv_len
        v.b["len"].close()
        v.b["len"] = v.b["kv"]
        v.run()
        v.check()
