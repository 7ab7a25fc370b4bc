"""A speculative step as a program runs it, with nothing coming back in between: pages, tree plan, rotary
positions and append, attention of the trees in two layers, verification, the accepted path moved into place,
pages behind it freed -- several steps of several requests, eager and as a replayed graph, against an account
of the tokens that each request holds, in 64 bits."""
import numpy as np
import pytest
import torch

from paged_cases import NONE, TORCH, attn_bound
from test_gpu_rope import bound as rope_bound, freqs, turned
from tree_cases import lines, random_parents, verify_oracle

pytestmark = pytest.mark.gpu
H, HK, D, PAGE, NSEQ, CAP, VOCAB, LAYERS, WIDTH, PAGES, PATH, KIDS = 8, 2, 64, 16, 3, 64, 700, 2, 12, 30, 40, 4
ROW = (H + 2 * HK) * D
STEPS = [(40, 9, 13), (9, 9, 1), (5, 0, 9), (8, 8, 8), (1, 16, 3), (9, 9, 9), (0, 3, 0), (7, 1, 12)]


class Step:
    def __init__(self, flh, s, cdt):
        self.flh, self.s, self.cdt = flh, s, cdt
        rng = np.random.default_rng(51)
        up = lambda a: flh.DeviceBuffer.from_array(a, s, extra=16)             # noqa: E731
        u32 = lambda n, v=0: up(np.full(n, v, np.uint32))                      # noqa: E731
        p = lambda b: b.ptr                                                    # noqa: E731
        self.held, self.add, self.kv, self.len = u32(NSEQ), u32(NSEQ), u32(NSEQ), u32(NSEQ)
        self.free, self.taken = up(rng.permutation(PAGES).astype(np.uint32)), u32(1)
        self.table, self.start, self.slot, self.pos = u32(NSEQ * WIDTH, NONE), u32(NSEQ + 1), u32(CAP), u32(CAP)
        self.info, self.parent, self.token = u32(4), u32(CAP), u32(CAP)
        self.mask, self.depth = u32(CAP * 2), u32(CAP)
        self.path, self.n_path, self.next = u32(NSEQ * PATH), u32(NSEQ), u32(NSEQ)
        self.qkv = [up(np.zeros(CAP * ROW, np.float32)) for _ in range(LAYERS)]
        self.out = [up(np.zeros(CAP * H * D, np.float32)) for _ in range(LAYERS)]
        self.target, self.draft = [up(np.zeros(CAP * VOCAB, np.float32)) for _ in range(2)]
        self.ua, self.un = up(np.zeros(CAP, np.float32)), up(np.zeros(NSEQ, np.float32))
        st = (PAGE * HK * D, HK * D, D)
        nan = np.full(PAGES * PAGE * HK * D, 0x7FFF, np.uint16)
        self.store = [(up(nan), up(nan)) for _ in range(LAYERS)]
        self.caches = [flh.KvCache(k, v, flh.Dtype[cdt], PAGES, PAGE, HK, D, D, st, st) for k, v in self.store]
        self.all = flh.KvCaches(self.caches)
        self.rope = flh.RopeTable(D, base=10000.0, layout=flh.RopeLayout.PAIRS)
        self.plan = flh.KvPlanP(held=p(self.held), add=p(self.add), free_pages=p(self.free), taken_in=p(self.taken), taken=p(self.taken),
                                table=p(self.table), q_start=p(self.start), kv_len=p(self.kv), slot=p(self.slot), info=p(self.info),
                                n_seq=NSEQ, page_size=PAGE, n_free=PAGES, table_stride=WIDTH, max_tok=CAP)
        self.tplan = flh.TreePlanP(q_start=p(self.start), parent=p(self.parent), kv_len=p(self.kv), mask=p(self.mask), depth=p(self.depth),
                                   pos=p(self.pos), n_seq=NSEQ, n_tok=CAP, mask_stride=2)
        self.tree = flh.TreeP(mask=p(self.mask), depth=p(self.depth), mask_stride=2)
        self.app, self.attn = [], []
        for x, o, c in zip(self.qkv, self.out, self.caches):
            q0 = x.ptr
            self.app.append(flh.RopeKvP(q=q0, q_out=q0, k=q0 + H * D * 4, v=q0 + (H + HK) * D * 4, pos=p(self.pos), slot=p(self.slot),
                                        q_tok=ROW, q_head=D, qo_tok=ROW, qo_head=D, k_tok=ROW, k_head=D, v_tok=ROW, v_head=D, dtype=0,
                                        n_tok=CAP, n_head=H, pos_stride=CAP))
            a = flh.AttnP(q=q0, out=o.ptr, q_start=p(self.start), kv_len=p(self.kv), table=p(self.table), q_tok=ROW, q_head=D,
                          o_tok=H * D, o_head=D, dtype=0, n_head=H, n_seq=NSEQ, n_tok=CAP, max_q=16, table_stride=WIDTH,
                          scale=D ** -0.5, causal=1)
            a.ws_bytes = flh.tree_attn_ws_bytes(c, a)
            self.attn.append(a)
        self.ws = flh.DeviceBuffer(max(a.ws_bytes for a in self.attn))
        for a in self.attn:
            a.ws = self.ws.ptr
        v = self.verify = flh.VerifyP(target=p(self.target), draft=p(self.draft), q_start=p(self.start), token=p(self.token),
                                      parent=p(self.parent), u_accept=p(self.ua), u_next=p(self.un), kv_len=p(self.kv),
                                      n_path=p(self.n_path), path=p(self.path), next=p(self.next), len=p(self.len), t_row=VOCAB,
                                      d_row=VOCAB, dtype=0, n_seq=NSEQ, n_tok=CAP, vocab=VOCAB, path_stride=PATH, max_child=KIDS)
        v.ws_bytes = flh.spec_verify_ws_bytes(v)
        self.vws = flh.DeviceBuffer(v.ws_bytes)
        v.ws = self.vws.ptr
        self.compact = flh.KvCompactP(q_start=p(self.start), slot=p(self.slot), n_path=p(self.n_path), path=p(self.path), n_seq=NSEQ,
                                      n_tok=CAP, path_stride=PATH)
        self.trim = flh.KvTrimP(kv_len=p(self.kv), keep=p(self.len), held=p(self.held), table=p(self.table), free_pages=p(self.free),
                                taken=p(self.taken), info=self.info.ptr + 8, n_seq=NSEQ, n_pages=PAGES, page_size=PAGE, n_free=PAGES,
                                table_stride=WIDTH)
        self.hist = [[] for _ in range(NSEQ)]                # of each token held: its rows in the layers

    def issue(self):
        f, s = self.flh, self.s
        f.kv_plan(self.plan, s)
        f.tree_plan(self.tplan, s)
        for app, attn, cache in zip(self.app, self.attn, self.caches):
            f.rope_kv_append(self.rope, cache, app, s)
            f.tree_attn(cache, attn, self.tree, s)
        f.spec_verify(self.verify, s)
        f.kv_compact(self.all, self.compact, s)
        f.kv_trim(self.trim, s)

    def inputs(self, add, rng, first):
        self.n = add
        self.rows = [rng.standard_normal((CAP, ROW)).astype(np.float32) for _ in range(LAYERS)]
        x = rng.standard_normal((CAP, VOCAB)) * 2
        self.x = x.astype(np.float32)
        self.y = (x + 0.4 * rng.standard_normal((CAP, VOCAB))).astype(np.float32)
        self.u, self.w = rng.random(CAP).astype(np.float32) * (0 if first else 0.6), rng.random(NSEQ).astype(np.float32)
        self.par, self.tok, row = np.full(CAP, -1, np.int32), np.zeros(CAP, np.uint32), 0
        for n in add:
            par = np.arange(n, dtype=np.int32) - 1 if first else random_parents(n, rng, 3)
            self.par[row:row + n] = par
            for i in range(1, n):
                self.tok[row + i] = int(np.argmax(self.y[row + par[i]] + rng.gumbel(size=VOCAB)))
            row += n
        for b, a in [(self.add, np.array(add, np.uint32)), (self.parent, self.par), (self.token, self.tok), (self.target, self.x),
                     (self.draft, self.y), (self.ua, self.u), (self.un, self.w), *zip(self.qkv, self.rows)]:
            b.upload(a, self.s)

    def turn(self, layer, row, pos):
        """The row's queries, keys and values, turned, and how far the device's may be off."""
        x = layer[row].astype(np.float64)
        at = np.array([[pos]], np.int64)
        fr = freqs(D, 10000.0)
        (q, qm), (k, km) = [turned(v.reshape(1, -1, D), at, fr, [0] * (D // 2), 0, False) for v in (x[:H * D], x[H * D:(H + HK) * D])]
        return q[0], rope_bound(q, qm, "F32")[0], k[0], rope_bound(k, km, self.cdt)[0], x[(H + HK) * D:].reshape(HK, D)

    def check(self):
        s = self.s
        start = np.concatenate([[0], np.cumsum(self.n)])
        assert self.info.download(np.uint32, 4, s).tolist()[1::2] == [0, 0]
        n_path, path, nxt, _, near = verify_oracle(self.x.astype(np.float64), self.y.astype(np.float64), start, self.tok, self.par, None,
                                                   self.u, self.w, PATH, KIDS, VOCAB)
        assert near > 1e-12
        np.testing.assert_array_equal(self.n_path.download(np.uint32, NSEQ, s), n_path)
        np.testing.assert_array_equal(self.path.download(np.uint32, NSEQ * PATH, s).reshape(NSEQ, PATH), path)
        np.testing.assert_array_equal(self.next.download(np.uint32, NSEQ, s), nxt)
        u = torch.finfo(TORCH[self.cdt]).eps / 2
        for layer in range(LAYERS):
            got = self.out[layer].download(np.float32, CAP * H * D, s).reshape(CAP, H, D)
            for r in range(NSEQ):
                old = len(self.hist[r])
                line_of = lines(self.par[start[r]:start[r + 1]])
                mine = [self.turn(self.rows[layer], start[r] + i, old + len(line_of[i]) - 1) for i in range(self.n[r])]
                for i in range(self.n[r]):
                    seen = [h[layer] for h in self.hist[r]] + [mine[j][2:] for j in sorted(line_of[i])]
                    kk, kb, vv = (np.stack([t[j] for t in seen]) for j in range(3))
                    for h in range(H):
                        g = h // (H // HK)
                        q, qb = mine[i][0][h], mine[i][1][h]
                        t = kk[:, g] @ q * D ** -0.5
                        e = np.exp(t - t.max())
                        w = e / e.sum()
                        want, mag = w @ vv[:, g], w @ np.abs(vv[:, g])
                        amp = (np.abs(kk[:, g]) @ np.abs(q)).max() * D ** -0.5
                        lim = attn_bound(torch.from_numpy(want), torch.from_numpy(mag), torch.tensor(amp), "F32", D, len(kk)).numpy()
                        # queries and keys are off by their rotation's and the cache's rounding, values by the latter
                        off = (kb[:, g] @ np.abs(q) + np.abs(kk[:, g]) @ qb + kb[:, g] @ qb).max() * D ** -0.5
                        lim = lim + mag * (2 * off + u)
                        assert (np.abs(got[start[r] + i, h] - want) <= lim).all(), (layer, r, i, h)
        # the path's tokens stand behind the cached ones
        for r in range(NSEQ):
            for j in range(int(n_path[r])):
                at = start[r] + int(path[r, j])
                self.hist[r].append([self.turn(self.rows[layer], at, len(self.hist[r]))[2:] for layer in range(LAYERS)])
        held = self.held.download(np.uint32, NSEQ, s)
        assert held.tolist() == [len(h) for h in self.hist]
        table = self.table.download(np.uint32, NSEQ * WIDTH, s).reshape(NSEQ, WIDTH)
        used = []
        for r in range(NSEQ):
            pages = -(-len(self.hist[r]) // PAGE)
            used += table[r, :pages].tolist()
            assert (table[r, pages:] == NONE).all()
        free = self.free.download(np.uint32, PAGES, s)[int(self.taken.download(np.uint32, 1, s)[0]):].tolist()
        assert sorted(used + free) == list(range(PAGES))
        for layer, (kb, vb) in enumerate(self.store):
            dt = TORCH[self.cdt]
            k, v = [torch.from_numpy(b.download(np.uint8, PAGES * PAGE * HK * D * 2, s)).view(dt).reshape(PAGES, PAGE, HK, D).double().numpy()
                    for b in (kb, vb)]
            for r in range(NSEQ):
                for j, h in enumerate(self.hist[r]):
                    wk, bound, wv = h[layer]
                    at = (int(table[r, j // PAGE]), j % PAGE)
                    assert (np.abs(k[at] - wk) <= bound).all(), (layer, r, j)
                    np.testing.assert_array_equal(v[at], torch.from_numpy(wv).to(dt).double().numpy())


@pytest.mark.parametrize("cdt", ["F16", "BF16"])
@pytest.mark.parametrize("captured", [False, True])
def test_steps(flh, gpu, cdt, captured):
    rng = np.random.default_rng(52)
    st = Step(flh, gpu, cdt)
    graph = None
    if captured:
        with flh.Graph.capture(gpu) as graph:
            st.issue()
    for i, add in enumerate(STEPS):
        st.inputs(add, rng, i == 0)
        graph.launch() if graph else st.issue()
        st.check()
    assert max(len(h) for h in st.hist) > 48                 # over page borders
    if graph:
        graph.close()
