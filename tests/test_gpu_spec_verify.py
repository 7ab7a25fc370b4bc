"""Verification of drafted tokens against the definition in 64 bits: p is renormalised after
each child that does not stand, and the next token is drawn from what is left."""
import math

import numpy as np
import pytest
import torch

from paged_cases import TORCH, put
from tree_cases import NONE, random_parents, verify_oracle

pytestmark = pytest.mark.gpu


class Verify:
    """Requests with `n` rows each; logits as a language model's: a few likely tokens."""

    def __init__(self, flh, s, n, vocab, dtype="F32", draft=True, kids=1, seed=0, chain=None, path=None, max_child=None, lead=0,
                 pad=0, offset=0, temp=True, peak=6.0):
        rng = np.random.default_rng(seed)
        self.flh, self.s, self.vocab, self.dtype = flh, s, vocab, dtype
        self.start = (np.concatenate([[0], np.cumsum(n)]) + lead).astype(np.uint32)
        self.rows = int(self.start[-1])
        rows = max(self.rows, 1)
        x = rng.standard_normal((rows, vocab)) * 2 + peak * (rng.random((rows, vocab)) < min(1.0, 20 / vocab)) * rng.random((rows, vocab))
        y = x + 0.7 * rng.standard_normal((rows, vocab))
        self.pitch = vocab + pad
        self.target = torch.full((rows, self.pitch), float("nan"), dtype=TORCH[dtype])
        self.draft = torch.full((rows, self.pitch), float("nan"), dtype=TORCH[dtype]) if draft else None
        self.target[:, :vocab] = torch.from_numpy(x).to(TORCH[dtype])
        if draft:
            self.draft[:, :vocab] = torch.from_numpy(y).to(TORCH[dtype])
        self.parent = np.full(rows, -5, np.int32)
        self.token = np.zeros(rows, np.uint32)
        for i in range(len(n)):
            r0 = int(self.start[i])
            for j in range(1, n[i]):
                up = (j - 1) // kids
                self.parent[r0 + j] = up
                z = (y if draft else x)[r0 + up]
                self.token[r0 + j] = int(np.argmax(z + rng.gumbel(size=vocab)))
        self.inv_temp = (rng.random(len(n)) * 1.5 + 0.3).astype(np.float32) if temp else None
        self.u_accept, self.u_next = rng.random(rows).astype(np.float32), rng.random(len(n)).astype(np.float32)
        self.kv_len = (rng.integers(0, 4000, len(n)) + np.array(n, np.int64)).astype(np.uint32)
        self.path = max(list(n) + [1]) if path is None else path
        self.max_child = kids if max_child is None else max_child
        self.chain = kids == 1 if chain is None else chain
        self.n, self.offset = n, offset

    def push(self):
        el = 4 if self.dtype == "F32" else 2
        s, flh = self.s, self.flh
        put_at = lambda t: flh.DeviceBuffer.from_array(                              # noqa: E731
            np.concatenate([np.zeros(self.offset * el, np.uint8), t.contiguous().view(torch.uint8).numpy().reshape(-1)]), s)
        u = lambda a: flh.DeviceBuffer.from_array(a, s, extra=16)                     # noqa: E731
        n_seq = len(self.n)
        b = self.b = dict(target=put_at(self.target), draft=put_at(self.draft) if self.draft is not None else None, start=u(self.start),
                          token=u(self.token), parent=u(self.parent), it=u(self.inv_temp) if self.inv_temp is not None else None,
                          ua=u(self.u_accept), un=u(self.u_next), kv=u(self.kv_len))
        fill = lambda k: u(np.full(max(k, 1), 0xABABABAB, np.uint32))                # noqa: E731
        b.update(n_path=fill(n_seq), path=fill(n_seq * self.path), next=fill(n_seq), logp=fill(n_seq * self.path), len=fill(n_seq))
        ptr = lambda k: b[k].ptr if b[k] is not None else None                       # noqa: E731
        self.p = flh.VerifyP(
            target=b["target"].ptr + self.offset * el, draft=b["draft"].ptr + self.offset * el if b["draft"] is not None else None,
            q_start=ptr("start"), token=ptr("token"), parent=None if self.chain else ptr("parent"), inv_temp=ptr("it"),
            u_accept=ptr("ua"), u_next=ptr("un"), kv_len=ptr("kv"), n_path=ptr("n_path"), path=ptr("path"), next=ptr("next"),
            logp=ptr("logp"), len=ptr("len"), t_row=self.pitch, d_row=self.pitch, dtype=flh.Dtype[self.dtype], n_seq=n_seq,
            n_tok=self.rows, vocab=self.vocab, path_stride=self.path, max_child=self.max_child)
        self.p.ws_bytes = flh.spec_verify_ws_bytes(self.p)
        b["ws"] = flh.DeviceBuffer(max(1, self.p.ws_bytes))
        b["ws"].upload(np.full(self.p.ws_bytes, 0xFF, np.uint8), s)
        self.p.ws = b["ws"].ptr
        return self

    def run(self, stream=None):
        self.flh.spec_verify(self.p, stream or self.s)

    def read(self):
        n = len(self.n)
        d = lambda k, t, c: self.b[k].download(t, c, self.s)                         # noqa: E731
        return (d("n_path", np.uint32, n), d("path", np.uint32, n * self.path).reshape(n, self.path), d("next", np.uint32, n),
                d("logp", np.float32, n * self.path).reshape(n, self.path), d("len", np.uint32, n))

    def check(self):
        x = self.target[:, :self.vocab].double().numpy()
        y = self.draft[:, :self.vocab].double().numpy() if self.draft is not None else None
        n_path, path, nxt, logp, near = verify_oracle(x, y, self.start, self.token, None if self.chain else self.parent, self.inv_temp,
                                                      self.u_accept, self.u_next, self.path, self.max_child, self.vocab)
        got = self.read()
        assert near > 1e-12, near                             # (the inputs decide nothing by less than 64 bits tell)
        np.testing.assert_array_equal(got[0], n_path)
        np.testing.assert_array_equal(got[1], path)
        np.testing.assert_array_equal(got[2], nxt)
        # rounded once to fp32 (half a step), from 64 bits
        assert (np.abs(got[3] - logp) <= np.abs(logp) * 2.0 ** -24 + 1e-12).all(), np.abs(got[3] - logp).max()
        np.testing.assert_array_equal(got[4], self.kv_len - np.array(self.n, np.uint32) + n_path)
        return got


@pytest.mark.parametrize("dtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("vocab", [1, 2, 17, 1000, 4095, 4096, 4097, 50257])
def test_chains(flh, gpu, vocab, draft, dtype):
    v = Verify(flh, gpu, [5, 1, 2, 9, 3, 6], vocab, dtype, draft, seed=vocab).push()
    v.run()
    v.check()


@pytest.mark.parametrize("dtype", ["F32", "BF16"])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("kids", [2, 3, 5])
@pytest.mark.parametrize("vocab", [13, 1003, 9001])
def test_trees(flh, gpu, vocab, kids, draft, dtype):
    for seed in range(3):
        v = Verify(flh, gpu, [1, 30, 7, 13, 0, 21, 2], vocab, dtype, draft, kids, seed=seed, peak=3.0).push()
        v.run()
        v.check()


def test_the_benchmark_vocabulary(flh, gpu):
    for draft in (False, True):
        v = Verify(flh, gpu, [5, 9], 128256, "F32", draft, 2, seed=4).push()
        v.run()
        v.check()


@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (0, 5), (8, 8)])
@pytest.mark.parametrize("dtype", ["F32", "F16"])
def test_strides_and_alignment(flh, gpu, dtype, pad, offset):
    """Rows at any element; what stands between them is no number."""
    v = Verify(flh, gpu, [4, 7, 1, 10], 5003, dtype, True, 3, seed=11, pad=pad, offset=offset, lead=3).push()
    v.run()
    v.check()


@pytest.mark.parametrize("kids", [1, 3])
@pytest.mark.parametrize("draft", [False, True])
def test_temperatures(flh, gpu, draft, kids):
    """Greedy requests among others (ties go to the lowest token), temperatures without end, nonsense."""
    v = Verify(flh, gpu, [8] * 9, 4999, "BF16", draft, kids, seed=12)
    v.inv_temp[:] = [math.inf, 1, math.inf, 0, -2, math.nan, 30, 1e-3, math.inf]
    for s in (0, 2, 8):                                        # drafted as the target would, for a while
        r0 = int(v.start[s])
        v.target[r0:r0 + 8, [77, 4990]] = 40.0
        for j in (1, 2, 5):
            v.token[r0 + j] = 77 if s != 8 else 4990
    v.push().run()
    got = v.check()
    assert got[0][0] > 1 and got[0][8] == 1 and (got[2][[0, 2, 8]] == 77).all() and (got[3][[0, 2, 8]] == 0).all()


@pytest.mark.parametrize("draft", [False, True])
def test_tokens_that_are_not_allowed(flh, gpu, draft):
    """-infinity, not a number and infinity among the logits; rows of which nothing is left; drafted tokens that
    are forbidden, or no tokens; the same token drafted twice."""
    rng = np.random.default_rng(13)
    v = Verify(flh, gpu, [13] * 8, 4500, "F32", draft, 3, seed=13)
    no = torch.from_numpy(rng.random((v.rows, 4500)) < 0.97)
    v.target[:, :4500][no] = -math.inf
    if draft:
        v.draft[:, :4500][no] = -math.inf
    v.target[:, 7] = math.nan
    v.target[int(v.start[2]), 100] = math.inf
    v.target[int(v.start[2]), 4300] = math.inf
    v.target[int(v.start[3])] = -math.inf
    v.target[int(v.start[4])] = math.nan
    if draft:
        v.draft[int(v.start[5])] = -math.inf
        v.draft[int(v.start[6]):int(v.start[7])] = v.target[int(v.start[6]):int(v.start[7])]
    v.token[int(v.start[1]) + 1:int(v.start[1]) + 4] = [4500, 0xFFFFFFFF, 1 << 30]
    v.token[int(v.start[7]) + 2] = v.token[int(v.start[7]) + 1]
    v.inv_temp[3] = 1.0
    v.inv_temp[0] = math.inf
    v.push().run()
    got = v.check()
    assert got[2][3] == NONE and got[2][4] == NONE and got[0][3] == 1
    v.inv_temp[:] = math.inf
    v.push().run()
    got = v.check()
    assert got[2][3] == NONE and got[2][4] == NONE


def test_numbers_at_the_ends(flh, gpu):
    """u = 0 takes every token that may be taken and the first that is likely at all; u just below 1 the last."""
    for u, draft in ((0.0, True), (0.0, False), (1 - 2.0 ** -24, True), (1 - 2.0 ** -24, False)):
        v = Verify(flh, gpu, [6, 1, 3], 9000, "F32", draft, seed=14)
        v.u_accept[:], v.u_next[:] = u, u
        v.push().run()
        v.check()


def test_limits_of_a_path(flh, gpu):
    """Paths cut off at path_stride, children behind max_child, rows behind the 256th."""
    for path in (1, 2, 3):
        v = Verify(flh, gpu, [9, 9, 2, 9], 700, "F32", True, seed=15, path=path)
        v.u_accept[:] = 0
        v.push().run()
        assert (v.check()[0] == min(path, 9)).sum() >= 2
    for most in (1, 2, 3):
        for draft in (False, True):
            v = Verify(flh, gpu, [16, 16, 16], 700, "F32", draft, 5, seed=16, max_child=most, peak=1.0).push()
            v.run()
            v.check()
    v = Verify(flh, gpu, [400, 3], 64, "F32", False, seed=17, path=300)
    v.u_accept[:] = 0
    v.push().run()
    v.check()


def test_any_parents(flh, gpu):
    """Rows that hang on none, or on later ones, are never reached; requests without rows."""
    rng = np.random.default_rng(18)
    for seed in range(4):
        v = Verify(flh, gpu, [0, 20, 12, 0, 9, 0], 900, "F32", seed % 2 == 0, 3, seed=seed, max_child=64, temp=False, peak=2.0)
        for s in (1, 2, 4):
            r0 = int(v.start[s])
            v.parent[r0:r0 + v.n[s]] = random_parents(v.n[s], rng, 6)
            v.parent[r0 + rng.integers(1, v.n[s], 4)] = rng.choice([-1, 77, 2 ** 31 - 1, 19], 4)
        v.push().run()
        v.check()
    v = Verify(flh, gpu, [0, 0], 900).push()
    v.run()
    assert (v.read()[2] == NONE).all() and (v.read()[0] == 0).all() and (v.read()[4] == v.kv_len).all()


@pytest.mark.parametrize("draft", [False, True])
def test_the_tokens_are_distributed_as_the_target(flh, gpu, draft):
    """Over many requests with the same logits the first token that comes out is distributed as p, whatever was
    drafted: 6 standard deviations of a count.  The draft is far from the target, three children a row."""
    n, vocab = 30000, 6
    rng = np.random.default_rng(19)
    v = Verify(flh, gpu, [4] * n, vocab, "F32", draft, 3, seed=19, chain=False, temp=False)
    x, y = np.array([0.0, 1.0, -1.0, 0.5, -3.0, 0.2]), np.array([1.5, -1.0, 0.3, 0.0, 1.0, -0.5])
    v.target[:, :vocab] = torch.from_numpy(x).float()
    p, q = np.exp(x) / np.exp(x).sum(), np.exp(y) / np.exp(y).sum()
    if draft:
        v.draft[:, :vocab] = torch.from_numpy(y).float()
        v.token[:] = rng.choice(vocab, v.rows, p=q)
    else:
        v.token[:] = rng.choice(vocab, v.rows)                # without a distribution: any tokens at all
    v.push().run()
    n_path, path, nxt, _, _ = v.read()
    first = np.where(n_path > 1, v.token[v.start[:-1] + np.where(n_path > 1, path[:, 1], 0)], nxt)
    counts = np.bincount(first, minlength=vocab)
    assert (np.abs(counts - n * p) <= 6 * np.sqrt(n * p * (1 - p))).all(), (counts, n * p)
    assert 0.1 < (n_path > 1).mean() < 1


@pytest.mark.parametrize("kids", [1, 3])
def test_captured(flh, gpu, kids):
    v = Verify(flh, gpu, [7, 4, 13], 9001, "F32", True, kids, seed=20).push()
    with flh.Graph.capture(gpu) as g:
        v.run()
    rng = np.random.default_rng(21)
    for _ in range(4):
        v.u_accept, v.u_next = rng.random(v.rows).astype(np.float32), rng.random(3).astype(np.float32)
        v.b["ua"].upload(v.u_accept, gpu)
        v.b["un"].upload(v.u_next, gpu)
        g.launch()
        got = v.check()
        v.run()
        for a, b in zip(got, v.read()):
            np.testing.assert_array_equal(a, b)
    g.close()


def test_two_streams_and_no_extras(flh, gpu):
    """Two calls at once, each with a workspace of its own; without logp and len."""
    a, b = Verify(flh, gpu, [5] * 20, 9001, "F32", True, 1, seed=22).push(), Verify(flh, gpu, [9] * 11, 5000, "BF16", True, 2, seed=23).push()
    s1, s2 = flh.Stream(), flh.Stream()
    gpu.sync()
    for _ in range(20):
        a.run(s1)
        b.run(s2)
    s1.sync()
    s2.sync()
    want = a.check()
    b.check()
    a.p.logp = a.p.len = a.p.kv_len = None
    a.run()
    for x, y in zip(a.read()[:3], want[:3]):
        np.testing.assert_array_equal(x, y)
    s1.close()
    s2.close()


@pytest.mark.parametrize("draft", [False, True])
def test_logits_of_any_size(flh, gpu, draft):
    """Rows whose largest logit is so large that its neighbour floats are far below it, temperatures that make
    a step of a logit decide, or hardly any; all of them against the same formula."""
    v = Verify(flh, gpu, [6] * 12, 5000, "F32", draft, seed=30, peak=2.0)
    scale = [1e-30, 1e-3, 1.0, 1e3, 1e6, 1e9, 1e15, 1e30, 3e37, 1e3, 1e-3, 1e-30]
    temp = [1e30, 1e3, 1.0, 1e-3, 1e-6, 1e-9, 1e-15, 1e-30, 3e-38, 3.0, 1e-3, 1.0]
    for s in range(12):
        r = slice(int(v.start[s]), int(v.start[s]) + 6)
        v.target[r] = (v.target[r].double() * scale[s] + (scale[s] * 50 if s % 2 else 0)).float()
        if draft:
            v.draft[r] = (v.draft[r].double() * scale[s] + (scale[s] * 50 if s % 2 else 0)).float()
        v.inv_temp[s] = temp[s]
    v.push().run()
    v.check()


@pytest.mark.parametrize("n_seq", [62, 63, 64, 65, 128, 700])
def test_numbers_of_requests(flh, gpu, n_seq):
    """A row's request is found 64 at a time: around that, with requests of no rows among them."""
    rng = np.random.default_rng(n_seq)
    n = rng.integers(0, 7, n_seq).tolist()
    n[0], n[-1] = (0, 3) if n_seq % 2 else (4, 0)
    for draft in (False, True):
        v = Verify(flh, gpu, n, 60, "F32", draft, 2, seed=n_seq, lead=n_seq % 3, peak=2.0).push()
        v.run()
        v.check()
