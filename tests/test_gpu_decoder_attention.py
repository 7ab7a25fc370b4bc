"""The attention half of a decoder layer as a program runs it: QKV dots, plan,
rotary positions and cache append, attention, O dot -- prompts, chunks and
single tokens of several requests, eager and as a replayed graph -- against the
same layer without a cache, in 64 bits, from the device's own QKV rows."""
import numpy as np
import pytest
import torch

from paged_cases import attn_bound
from test_gpu_rope import bound as rope_bound, freqs, turned

pytestmark = pytest.mark.gpu
HID, H, HK, D, PAGE, NSEQ, CAP = 512, 8, 2, 64, 16, 3, 16
ROW = (H + 2 * HK) * D
NONE = 0xFFFFFFFF


class Layer:
    def __init__(self, flh, s, cdt):
        rng = np.random.default_rng(31)
        self.flh, self.s, self.cdt = flh, s, cdt
        up = lambda a, extra=0: flh.DeviceBuffer.from_array(a, s, extra)       # noqa: E731
        q = lambda r, c: flh.quantize_host(flh.Fmt.Q4_K, (rng.standard_normal((r, c)) * 0.05).astype(np.float32))   # noqa: E731
        self.wqkv, self.wo_host = up(q(ROW, HID)), q(HID, H * D)
        self.wo = up(self.wo_host)
        self.xs = (flh.x_alloc_bytes(HID) + 127) // 128 * 32                   # floats between columns
        self.os = (flh.x_alloc_bytes(H * D) + 127) // 128 * 32
        z = lambda n: up(np.zeros(n, np.uint8))                                # noqa: E731
        self.x, self.qkv, self.att, self.y = z(CAP * self.xs * 4), z(CAP * ROW * 4), z(CAP * self.os * 4), z(CAP * HID * 4)
        n_pages = 40
        nan = np.full(n_pages * PAGE * HK * D, 0x7FFF, np.uint16)
        self.k, self.v = up(nan), up(nan)
        st = (PAGE * HK * D, HK * D, D)
        self.cache = flh.KvCache(self.k, self.v, flh.Dtype[cdt], n_pages, PAGE, HK, D, D, st, st)
        self.lens, self.add = up(np.zeros(NSEQ, np.uint32)), up(np.zeros(NSEQ, np.uint32))
        self.free = up(rng.permutation(n_pages).astype(np.uint32))
        self.taken, self.info = up(np.zeros(1, np.uint32)), up(np.zeros(2, np.uint32))
        self.table = up(np.full(NSEQ * 16, NONE, np.uint32))
        self.start, self.slot, self.pos = up(np.zeros(NSEQ + 1, np.uint32)), up(np.zeros(CAP, np.uint32)), up(np.zeros(CAP, np.int32))
        self.rope = flh.RopeTable(D, base=10000.0, layout=flh.RopeLayout.PAIRS)
        p = lambda b: b.ptr                                                    # noqa: E731
        self.plan = flh.KvPlanP(held=p(self.lens), add=p(self.add), free_pages=p(self.free), taken_in=p(self.taken),
                                taken=p(self.taken), table=p(self.table), q_start=p(self.start), kv_len=p(self.lens),
                                slot=p(self.slot), pos=p(self.pos), info=p(self.info), n_seq=NSEQ, page_size=PAGE,
                                n_free=n_pages, table_stride=16, max_tok=CAP)
        q0 = self.qkv.ptr
        self.app = flh.RopeKvP(q=q0, q_out=q0, k=q0 + H * D * 4, v=q0 + (H + HK) * D * 4, pos=p(self.pos), slot=p(self.slot),
                               q_tok=ROW, q_head=D, qo_tok=ROW, qo_head=D, k_tok=ROW, k_head=D, v_tok=ROW, v_head=D,
                               dtype=0, n_tok=CAP, n_head=H, pos_stride=CAP)
        # the attention's rows are the O dot's activation columns
        self.attn = flh.AttnP(q=q0, out=self.att.ptr, q_start=p(self.start), kv_len=p(self.lens), table=p(self.table),
                              q_tok=ROW, q_head=D, o_tok=self.os, o_head=D, dtype=0, n_head=H, n_seq=NSEQ, n_tok=CAP,
                              max_q=CAP, table_stride=16, scale=D ** -0.5, causal=1)
        self.attn.ws_bytes = flh.paged_attn_ws_bytes(self.cache, self.attn)
        self.ws = flh.DeviceBuffer(max(1, self.attn.ws_bytes))
        self.attn.ws = self.ws.ptr
        self.hist = [[] for _ in range(NSEQ)]

    def issue(self):
        flh, s = self.flh, self.s
        self.qkv.zero(s)
        self.y.zero(s)
        flh.kv_plan(self.plan, s)
        flh.act_q8(self.x, HID, s, nx=CAP, xstride=self.xs)
        flh.stream_dot(flh.Fmt.Q4_K, self.wqkv, ROW, HID, self.x, self.qkv, s, nx=CAP, xstride=self.xs, ystride=ROW)
        flh.rope_kv_append(self.rope, self.cache, self.app, s)
        flh.paged_attn(self.cache, self.attn, s)
        flh.act_q8(self.att, H * D, s, nx=CAP, xstride=self.os)
        flh.stream_dot(flh.Fmt.Q4_K, self.wo, HID, H * D, self.att, self.y, s, nx=CAP, xstride=self.os, ystride=HID)

    def inputs(self, add, rng):
        self.add.upload(np.array(add, np.uint32), self.s)
        x = np.zeros((CAP, self.xs), np.float32)
        x[:, :HID] = rng.standard_normal((CAP, HID))
        self.x.upload(x, self.s)
        # the products alone, for the check: the step turns them in place
        self.qkv.zero(self.s)
        self.flh.act_q8(self.x, HID, self.s, nx=CAP, xstride=self.xs)
        self.flh.stream_dot(self.flh.Fmt.Q4_K, self.wqkv, ROW, HID, self.x, self.qkv, self.s, nx=CAP, xstride=self.xs, ystride=ROW)
        self.rows = self.qkv.download(np.float32, CAP * ROW, self.s).reshape(CAP, ROW).astype(np.float64)

    def check(self, add, orc):
        s, row = self.s, 0
        assert self.info.download(np.uint32, 2, s).tolist() == [sum(add), 0]
        att = self.att.download(np.float32, CAP * self.os, s).reshape(CAP, self.os)
        freq = freqs(D, 10000.0)
        for r, n in enumerate(add):
            for i in range(n):
                self.hist[r].append(self.rows[row + i])
            if n == 0:
                continue
            h = np.stack(self.hist[r])
            pos = np.arange(len(h))[None, :].astype(np.int64)
            split = [h[:, :H * D].reshape(-1, H, D), h[:, H * D:(H + HK) * D].reshape(-1, HK, D), h[:, (H + HK) * D:].reshape(-1, HK, D)]
            (q, qm), (k, km) = turned(split[0], pos, freq, [0] * 32, 0, False), turned(split[1], pos, freq, [0] * 32, 0, False)
            dt = {"F16": torch.float16, "BF16": torch.bfloat16}[self.cdt]
            u = torch.finfo(dt).eps / 2
            v = split[2]
            for i in range(len(h) - n, len(h)):
                for head in range(H):
                    kk, vv = k[:i + 1, head // (H // HK)], v[:i + 1, head // (H // HK)]
                    t = kk @ q[i, head] * D ** -0.5
                    e = np.exp(t - t.max())
                    w = e / e.sum()
                    want, mag = w @ vv, w @ np.abs(vv)
                    # keys and values were rounded to the cache's type: a score moves by u sum |q k| scale,
                    # a weight by twice that, a value by u; the rest as for any attention
                    amp = (np.abs(kk) @ np.abs(q[i, head])).max() * D ** -0.5
                    lim = attn_bound(torch.from_numpy(want), torch.from_numpy(mag), torch.tensor(amp), "F32", D, i + 1).numpy()
                    turn = (rope_bound(kk, km[:i + 1, head // (H // HK)], self.cdt).max() * np.abs(q[i, head]).sum() +
                            rope_bound(q[i, head], qm[i, head], "F32").max() * np.abs(kk).sum(1).max()) * D ** -0.5
                    lim = lim + mag * (2 * turn + u)
                    got = att[row + i - (len(h) - n), head * D:(head + 1) * D]
                    assert (np.abs(got - want) <= lim).all(), (r, i, head, np.abs(got - want).max(), lim.min())
            row += n
        # the O dot of the device's own attention rows, bit for bit
        y = self.y.download(np.float32, CAP * HID, s).reshape(CAP, HID)
        want = np.zeros((CAP, HID), np.float32)
        cols = orc.act_q8_cols(att[:row, :H * D].copy(), self.os)
        for c in range(row):
            orc.stream_dot(3, self.wo_host, HID, H * D, cols[c * self.os:(c + 1) * self.os], want[c], xstride=self.os)
        np.testing.assert_array_equal(y[:row].view(np.uint32), want[:row].view(np.uint32))


STEPS = [(5, 0, 11), (1, 7, 1), (1, 1, 1), (9, 1, 0), (1, 1, 1), (0, 1, 1), (1, 14, 1), (1, 1, 1)]


@pytest.mark.parametrize("cdt", ["F16", "BF16"])
@pytest.mark.parametrize("captured", [False, True])
def test_layer(flh, gpu, orc, cdt, captured):
    rng = np.random.default_rng(32)
    layer = Layer(flh, gpu, cdt)
    graph = None
    if captured:
        with flh.Graph.capture(gpu) as graph:
            layer.issue()
    for add in STEPS:
        layer.inputs(add, rng)
        graph.launch() if graph else layer.issue()
        layer.check(add, orc)
    # padded rows of the last steps wrote nothing: the cache holds as many tokens as the requests
    k = layer.k.download(np.uint16, 40 * PAGE * HK * D, gpu).reshape(40 * PAGE, HK * D)
    assert int((~(k == 0x7FFF).all(1)).sum()) == sum(map(sum, STEPS))
    if graph:
        graph.close()
