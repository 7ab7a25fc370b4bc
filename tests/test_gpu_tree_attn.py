"""Tree plans against lines walked up one by one, and attention of trees against
softmax(scale q k) v over the keys that each row sees, in 64 bits."""
import math

import numpy as np
import pytest
import torch

from paged_cases import NONE, attn_bound, get, put
from test_gpu_paged_attn import TYPES, Case
from tree_cases import lines, plan_oracle, random_parents, tree_attn_oracle

pytestmark = pytest.mark.gpu


def up(flh, s, a):
    return flh.DeviceBuffer.from_array(a, s, extra=16)


# -------------------------------------------------------------------- plan --
def plan(flh, s, parents, kv, stride, window, lead=0, spare=3, n_tok=None, with_pos=True):
    n = [len(p) for p in parents]
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.uint32) + np.uint32(lead)
    total = int(start[-1]) + spare
    par = np.full(total, 77, np.int32)
    for i, p in enumerate(parents):
        par[start[i]:start[i + 1]] = p
    b = [up(flh, s, x) for x in (start, par, np.array(kv, np.uint32), np.full((total, stride), 0xABABABAB, np.uint32),
                                 np.full(total, 0xABABABAB, np.uint32), np.full(total, -9, np.int32))]
    p = flh.TreePlanP(q_start=b[0].ptr, parent=b[1].ptr, kv_len=b[2].ptr if with_pos else None, mask=b[3].ptr, depth=b[4].ptr,
                      pos=b[5].ptr if with_pos else None, n_seq=len(n), n_tok=total if n_tok is None else n_tok, mask_stride=stride,
                      window=window)
    flh.tree_plan(p, s)
    return (b[3].download(np.uint32, total * stride, s).reshape(total, stride), b[4].download(np.uint32, total, s),
            b[5].download(np.int32, total, s))


@pytest.mark.parametrize("window", [0, 1, 2, 7])
@pytest.mark.parametrize("sizes", [[1], [0, 3, 0, 1, 70, 0], [33, 64, 65, 31, 32], [300, 5], [1, 2] * 600])
def test_plan(flh, gpu, sizes, window):
    rng = np.random.default_rng(len(sizes))
    parents = [random_parents(n, rng, 5) for n in sizes]
    kv = [n + int(rng.integers(0, 5000)) for n in sizes]
    stride = max(1, -(-max(sizes) // 32))
    for lead in (0, 300):
        want = plan_oracle(parents, kv, stride, window)
        got = plan(flh, gpu, parents, kv, stride, window, lead)
        end = lead + sum(sizes)
        for g, w, old in zip(got, want, (0xABABABAB, 0xABABABAB, -9)):
            np.testing.assert_array_equal(g[lead:end], w)
            assert (g[:lead] == old).all() and (g[end:] == old).all()


def test_plan_of_any_parents(flh, gpu):
    """Several roots, parents that are no earlier row, a chain of a few thousand, few words, rows
    cut off, no positions."""
    rng = np.random.default_rng(3)
    odd = np.array([5, -1, 0, 3, 2, -7, 6, 1, 100, 2 ** 31 - 1, 7], np.int32)
    chain = np.arange(5000, dtype=np.int32) - 1
    parents = [odd, chain, random_parents(40, rng)]
    kv = [11, 6000, 40]
    want = plan_oracle(parents, kv, 2, 0)
    got = plan(flh, gpu, parents, kv, 2, 0)
    n = sum(map(len, parents))
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g[:n], w)
    cut = plan(flh, gpu, parents, kv, 2, 0, n_tok=4000)
    for g, w, old in zip(cut, want, (0xABABABAB, 0xABABABAB, -9)):
        np.testing.assert_array_equal(g[:4000], w[:4000])
        assert (g[4000:] == old).all()
    bare = plan(flh, gpu, parents, kv, 2, 0, with_pos=False)
    np.testing.assert_array_equal(bare[0], got[0])
    assert (bare[2] == -9).all()
    flh.tree_plan(flh.TreePlanP(mask_stride=1), gpu)          # nothing to do


# --------------------------------------------------------------- attention --
class Tree(Case):
    """A Case whose requests' rows are trees."""

    def __init__(self, flh, s, act, cdt, heads, hk, dk, dv, page, order, lens, seed, window=0, back=4, stride=None, **kw):
        super().__init__(flh, s, act, cdt, heads, hk, dk, dv, page, order, lens, seed, causal=True, window=window, **kw)
        rng = np.random.default_rng(seed + 1000)
        parents = [random_parents(n, rng, back) for n, _ in lens]
        stride = max(1, -(-max([n for n, _ in lens] + [1]) // 32)) if stride is None else stride
        mask, depth, _ = plan_oracle(parents, self.kv_len, stride, window)
        lead = self.rows[0][0] if self.rows else 0
        total = self.qbuf.shape[0]
        self.mask, self.depth = np.full((total, stride), 0xFFFFFFFF, np.uint32), np.full(total, 0xFFFFFFFF, np.uint32)
        self.mask[lead:lead + len(mask)], self.depth[lead:lead + len(mask)] = mask, depth
        self.cut = None
        self.tree()

    def tree(self):
        self.b["mask"], self.b["depth"] = up(self.flh, self.s, self.mask), up(self.flh, self.s, self.depth)
        self.t = self.flh.TreeP(mask=self.b["mask"].ptr, depth=self.b["depth"].ptr if self.window else None,
                                mask_stride=self.mask.shape[1])

    def ws(self):
        keep, self.flh = self.flh, _Tree(self.flh)
        super().ws()
        self.flh = keep

    def run(self, stream=None):
        self.flh.tree_attn(self.cache.c, self.p, self.t, stream or self.s)

    def oracle(self):
        return tree_attn_oracle(self.q, self.rows, self.kv_len, self.table, self.cache, self.group, self.scale, self.window,
                                self.mask, self.depth, self.cut)

    def check(self, got=None):
        got = self.result() if got is None else got
        out, mag, amp = self.oracle()
        have = got[:, :self.heads * self.dv].unflatten(1, (self.heads, self.dv)).double()
        live = torch.zeros(have.shape[0], dtype=torch.bool)
        for a, b in self.rows:
            live[a:b] = True
        assert torch.equal(got[~live], self.out0[~live]), "rows of no request changed"
        lim = attn_bound(out, mag, amp, self.act, self.dk, int(self.kv_len.max()))
        fin = torch.isfinite(out) & torch.isfinite(lim)
        bad = live[:, None, None] & fin & ~((have - out).abs() <= lim)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist(), float((have - out).abs()[bad].max()))
        odd = live[:, None, None] & ~torch.isfinite(out)
        assert torch.equal(torch.isnan(have[odd]), torch.isnan(out[odd]))
        return got


class _Tree:
    """The library with the tree attention's workspace in the place of the other's."""

    def __init__(self, flh):
        self._flh = flh

    def __getattr__(self, name):
        return getattr(self._flh, "tree_attn_ws_bytes" if name == "paged_attn_ws_bytes" else name)


# by rows a kv head: up to 16, 32, 48, 64 and more
NODES = [1, 4, 8, 12, 16, 17, 40]


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (80, 80), (192, 128), (256, 256), (8, 8), (128, 40)])
@pytest.mark.parametrize("n", NODES)
def test_forms(flh, gpu, act, cdt, dk, dv, n):
    """Every width, type and number of rows; trees alone, behind contexts around the tiles,
    and behind one that many workgroups share; the same bits when run again."""
    lens = [(n, n), (n, n + 31), (1, 200), (max(1, n - 1), 64 + n), (n, 5000), (0, 9), (2, 129), (n, 777)]
    c = Tree(flh, gpu, act, cdt, 8, 2, dk, dv, 16, "token", lens, 90)
    c.run()
    first = c.check().clone()
    c.run()
    assert torch.equal(c.result(), first)


@pytest.mark.parametrize("act,cdt", [("F32", "BF16"), ("F16", "F16")])
@pytest.mark.parametrize("heads,hk", [(4, 4), (5, 1), (32, 8), (64, 2)])
@pytest.mark.parametrize("page,order", [(1, "head"), (16, "head"), (64, "token"), (256, "head")])
def test_head_layouts_and_pages(flh, gpu, heads, hk, page, order, act, cdt):
    lens = [(9, 300), (13, 13), (1, 77), (5, 1023)]
    c = Tree(flh, gpu, act, cdt, heads, hk, 64, 64, page, order, lens, 91, q_pad=24, cache_pad=8, lead=5)
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("BF16", "BF16")])
@pytest.mark.parametrize("n", [5, 14, 60])
@pytest.mark.parametrize("window", [1, 2, 5, 33, 64, 500])
def test_windows(flh, gpu, window, n, act, cdt):
    """Windows shorter than the tree's lines, of a few tiles, and that reach past the begin;
    deep trees (chains of two)."""
    lens = [(n, n), (n, n + 40), (n, 1000), (n, 3001)]
    for back in (1, 2, 6):
        c = Tree(flh, gpu, act, cdt, 8, 2, 128, 128, 16, "head", lens, 92, window=window, back=back)
        c.run()
        c.check()


@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("BF16", "BF16")])
@pytest.mark.parametrize("n", [5, 12, 70])
def test_any_masks(flh, gpu, act, cdt, n):
    """Bits of any rows, behind a row too, and of none; more words than rows, fewer words than rows,
    bits behind the request's last row; a request that has nothing cached, whose rows without bits give 0; depths too large."""
    rng = np.random.default_rng(5)
    lens = [(n, n), (n, n + 3), (n, 400), (n, 3000)]
    for stride, window in ((4, 0), (1, 0), (3, 20)):
        c = Tree(flh, gpu, act, cdt, 8, 2, 128, 128, 16, "head", lens, 93, stride=stride, window=window)
        c.mask = rng.integers(0, 1 << 32, c.mask.shape, dtype=np.uint64).astype(np.uint32)
        c.mask[rng.random(len(c.mask)) < 0.4] = 0
        c.mask[0] = 0
        c.depth = rng.integers(0, 2 * n, c.depth.shape).astype(np.uint32)
        c.depth[1] = 0xFFFFFFFF
        c.tree()
        c.run()
        got = c.check()
        assert (got[0][:8 * 128] == 0).all()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n", [4, 12, 16, 40])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_values_not_seen(flh, gpu, act, cdt, n, value):
    """Keys and values of siblings, and of tokens behind the window, that are no numbers: no
    part of the rows that do not see them."""
    lens = [(n, n + 150), (n, n + 7), (n, 3000)]
    c = Tree(flh, gpu, act, cdt, 8, 2, 128, 128, 16, "head", lens, 94, window=1000, back=3)
    hit = {}
    for s, (r0, r1) in enumerate(c.rows):
        kv = int(c.kv_len[s])
        seen = [sum(int(c.mask[r][b // 32]) >> (b % 32) & 1 for r in range(r0, r1)) for b in range(n)]
        b = n - 1 - int(np.argmin(seen[::-1]))                # a row that fewest see
        hit[s] = b
        for j in [kv - n + b] + ([kv - n - 1500] if kv > 2000 else []):
            pg = int(c.table[s, j // 16])
            c.cache.view[1][pg, j % 16, :, 3] = value
            if math.isnan(value):
                c.cache.view[0][pg, j % 16, :, 5] = value
    c.cache.push()
    c.run()
    out, _, _ = c.oracle()
    c.check()
    assert not torch.isfinite(out).all() and torch.isfinite(out).any()


def test_bad_table_entries_and_short_tables(flh, gpu):
    """Pages of the context and of the tree that are none, and a table that ends inside the tree."""
    for n in (6, 13, 40):
        c = Tree(flh, gpu, "F32", "F16", 8, 2, 64, 64, 16, "token", [(n, 300), (n, 64 + n), (n, 500)], 95, width_extra=0)
        c.table[0, 2], c.table[0, (300 - n) // 16] = NONE, c.cache.n_pages
        c.table[1, :] = NONE
        c.b["table"].upload(c.table, gpu)
        c.run()
        c.check()
        c.table = np.ascontiguousarray(c.table[:, :-1])
        c.b["table"].upload(c.table, gpu)
        c.p.table_stride = c.table.shape[1]
        c.run()
        c.check()


@pytest.mark.parametrize("n", [7, 13, 40])
def test_rows_cut_off(flh, gpu, n):
    """n_tok inside a request: its other rows are not computed, and its keys stay where they are."""
    c = Tree(flh, gpu, "F32", "BF16", 8, 2, 128, 128, 16, "head", [(n, 200), (n, 300)], 96)
    c.p.n_tok = c.n_tok - n // 2
    c.run()
    c.rows = [c.rows[0], (c.rows[1][0], c.rows[1][1] - n // 2)]
    c.cut = [0, n // 2]
    c.check()


@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("BF16", "BF16")])
def test_a_chain_is_causal_attention(flh, gpu, act, cdt):
    """A tree that does not branch, in the same kernel, has the bits of the attention of drafted runs -- where its rows
    are one strip.  The strips of 50 tokens (128 rows: 32 tokens, and 18) are not: causal attention gives the first the 2000 - 50 + 32 keys
    up to its last token, 31 tiles of 64, the tree's may see all 2000, 32 tiles; so the work is cut elsewhere and sums are added in
    another order.  There both are right to their rounding."""
    for n in (1, 4, 8, 17, 50):
        c = Tree(flh, gpu, act, cdt, 8, 2, 128, 128, 16, "head", [(n, n + 100), (n, 2000)], 97, back=1)
        c.run()
        tree = c.check().clone()
        if 32 < 4 * n <= 64:
            continue
        Case.ws(c)
        Case.run(c)
        if 4 * n <= 128:
            assert torch.equal(c.result(), tree), n
        else:
            Case.check(c)


@pytest.mark.parametrize("n", [6, 14, 90])
def test_captured(flh, gpu, n):
    """A captured call, replayed while lengths and trees on the device change."""
    c = Tree(flh, gpu, "F32", "F16", 8, 2, 128, 128, 16, "head", [(n, 900), (n, 333), (n, 64 + n)], 98)
    with flh.Graph.capture(gpu) as g:
        c.run()
    rng = np.random.default_rng(9)
    for step in range(4):
        for i, (r0, r1) in enumerate(c.rows):
            c.kv_len[i] = max(r1 - r0, int(c.kv_len[i]) - 37 * step)
            m, d, _ = plan_oracle([random_parents(r1 - r0, rng)], [c.kv_len[i]], c.mask.shape[1], 0)
            c.mask[r0:r1], c.depth[r0:r1] = m, d
        c.b["kv"].upload(c.kv_len.view(np.uint8), gpu)
        c.b["mask"].upload(c.mask, gpu)
        c.b["out"].upload(np.frombuffer(c.out0.contiguous().view(torch.uint8).numpy().tobytes(), np.uint8), gpu)
        g.launch()
        got = c.check().clone()
        c.run()
        assert torch.equal(c.result(), got)
    g.close()


def test_many_requests_on_another_stream(flh, gpu):
    rng = np.random.default_rng(20)
    lens = [(n, n + int(rng.integers(0, 60))) for n in rng.integers(0, 12, 700).tolist()]
    c = Tree(flh, gpu, "F32", "F16", 4, 1, 64, 64, 16, "head", lens, 99)
    s = flh.Stream()
    gpu.sync()
    c.run(s)
    s.sync()
    c.check()
    s.close()


@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("F32", "BF16"), ("BF16", "BF16")])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
@pytest.mark.parametrize("sizes", [[25, 1, 2, 0, 32, 3, 17, 16, 1, 5], [25, 24, 17, 32, 1, 30], [33, 1, 1, 1, 1, 1, 1, 1]])
def test_few_and_many_rows_on_average(flh, gpu, sizes, dk, dv, act, cdt):
    """Requests of one strip and of several, whichever the strips' length is; the workspace is the same for any rows."""
    rng = np.random.default_rng(len(sizes))
    lens = [(n, n + int(rng.integers(0, 3000))) for n in sizes]
    for window in (0, 300):
        c = Tree(flh, gpu, act, cdt, 8, 2, dk, dv, 16, "head", lens, 91, window=window)
        c.run()
        c.check()
    need = c.p.ws_bytes
    for n_tok in (6, 1000):
        p = type(c.p).from_buffer_copy(c.p)
        p.n_tok = n_tok
        assert flh.tree_attn_ws_bytes(c.cache.c, p) == need
