"""Attention over the paged cache against softmax(scale q k) v in 64 bits."""
import math

import numpy as np
import pytest
import torch

from paged_cases import Cache, NONE, TORCH, attn_bound, attn_oracle, get, put, raw

pytestmark = pytest.mark.gpu


class Case:
    """Requests with (rows, keys) over a cache of shuffled pages; what no
    request has written is NaN."""

    def __init__(self, flh, s, act, cdt, heads, hk, dk, dv, page, order, lens, seed, causal=True, window=0, q_pad=0, cache_pad=0,
                 spare_rows=3, width_extra=1, lead=0, scale=None, amp=1.5, gap=0):
        rng = np.random.default_rng(seed)
        self.flh, self.s, self.act, self.group, self.causal, self.window = flh, s, act, heads // hk, causal, window
        self.scale = dk ** -0.5 if scale is None else scale
        pages = [-(-kv // page) for _, kv in lens]
        n_pages = sum(pages) + 3
        self.cache = Cache(flh, s, cdt, n_pages, page, hk, dk, dv, order, cache_pad)
        perm = rng.permutation(n_pages)
        width = max([*pages, 1]) + width_extra
        self.table = np.full((len(lens), width), NONE, np.uint32)
        at, self.rows, row = 0, [], lead
        for i, ((n, kv), k) in enumerate(zip(lens, pages)):
            self.table[i, :k] = perm[at:at + k]
            at += k
            self.rows.append((row, row + n))
            row += n
            j = np.arange(kv)
            pg = torch.from_numpy(self.table[i][j // page].astype(np.int64))
            for v, d in zip(self.cache.view, (dk, dv)):
                v[pg, torch.from_numpy(j % page)] = torch.from_numpy(rng.standard_normal((kv, hk, d))).to(TORCH[cdt])
        self.cache.push()
        self.n_tok = row
        self.kv_len = np.array([kv for _, kv in lens], np.uint32)
        self.q_start = np.array([r for r, _ in self.rows] + [row], np.uint32)
        total = row + spare_rows
        self.qbuf = torch.full((total, heads * dk + q_pad), float("nan"), dtype=TORCH[act])
        self.q = self.qbuf[:, :heads * dk].unflatten(1, (heads, dk))
        self.q[lead:row] = torch.from_numpy(rng.standard_normal((row - lead, heads, dk)) * amp).to(TORCH[act])
        self.out0 = torch.full((total, heads * dv + q_pad), 3.0, dtype=TORCH[act])
        self.heads, self.dk, self.dv = heads, dk, dv
        self.b = dict(q=put(flh, s, self.qbuf), out=put(flh, s, self.out0), start=put(flh, s, torch.from_numpy(self.q_start.view(np.int32))),
                      kv=put(flh, s, torch.from_numpy(self.kv_len.view(np.int32))),
                      table=put(flh, s, torch.from_numpy(self.table.view(np.int32))))
        b = self.b
        self.p = flh.AttnP(q=b["q"].ptr, out=b["out"].ptr, q_start=b["start"].ptr, kv_len=b["kv"].ptr, table=b["table"].ptr,
                           q_tok=self.qbuf.stride(0), q_head=dk, o_tok=self.out0.stride(0), o_head=dv, dtype=flh.Dtype[act],
                           n_head=heads, n_seq=len(lens), n_tok=self.n_tok, max_q=max([n for n, _ in lens] + [1]),
                           table_stride=width, scale=self.scale, causal=int(causal), window=window)
        self.ws()

    def ws(self):
        self.p.ws_bytes = self.flh.paged_attn_ws_bytes(self.cache.c, self.p)
        if self.p.ws_bytes:
            if self.b.get("ws") is None or self.b["ws"].nbytes < self.p.ws_bytes:
                self.b["ws"] = self.flh.DeviceBuffer(self.p.ws_bytes)
                # whatever a workspace held before is of no account: NaN bits
                self.b["ws"].upload(np.full(min(self.p.ws_bytes, 1 << 26), 0xFF, np.uint8), self.s)
            self.p.ws = self.b["ws"].ptr

    def run(self, stream=None):
        self.flh.paged_attn(self.cache.c, self.p, stream or self.s)

    def result(self):
        return get(self.b["out"], self.out0, self.s)

    def check(self, got=None):
        got = self.result() if got is None else got
        out, mag, amp = attn_oracle(self.q, self.rows, self.kv_len, self.table, self.cache, self.group, self.scale, self.causal,
                                    self.window)
        have = got[:, :self.heads * self.dv].unflatten(1, (self.heads, self.dv)).double()
        live = torch.zeros(have.shape[0], dtype=torch.bool)
        for a, b in self.rows:
            live[a:b] = True
        assert torch.equal(got[~live], self.out0[~live]), "rows of no request changed"
        assert torch.equal(got[:, self.heads * self.dv:], self.out0[:, self.heads * self.dv:]), "between the rows"
        fin = torch.isfinite(out) & torch.isfinite(mag)
        keys = int(self.kv_len.max()) if len(self.kv_len) else 0
        lim = attn_bound(out, mag, amp, self.act, self.dk, keys)
        err = (have - out).abs()
        bad = live[:, None, None] & fin & ~(err <= lim)
        assert not bad.any(), (int(bad.sum()), float(err[bad].max()), float(lim[bad].max()), bad.nonzero()[:3].tolist())
        odd = live[:, None, None] & ~fin
        assert torch.equal(torch.isnan(have[odd]), torch.isnan(out[odd]))
        assert torch.equal(have[odd].nan_to_num(0, 1, -1), out[odd].nan_to_num(0, 1, -1))
        return got


TYPES = [("F32", "F16"), ("F32", "BF16"), ("F16", "F16"), ("BF16", "BF16")]
DIMS = [(128, 128), (64, 64), (80, 80), (96, 96), (192, 128), (256, 256), (8, 8), (128, 40), (24, 200)]


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("dk,dv", DIMS)
def test_one_token(flh, gpu, act, cdt, dk, dv):
    """Decode: a row a request, contexts of every length around the tile sizes."""
    lens = [(1, kv) for kv in (1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 777)]
    c = Case(flh, gpu, act, cdt, 8, 2, dk, dv, 16, "head", lens, 1)
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("dk,dv", DIMS)
def test_chunks(flh, gpu, act, cdt, dk, dv):
    """Ragged prompt chunks behind cached contexts, some whole prompts."""
    lens = [(5, 5), (1, 200), (70, 70), (33, 500), (129, 131), (0, 40), (64, 64), (200, 333)]
    c = Case(flh, gpu, act, cdt, 6, 2, dk, dv, 32, "token", lens, 2)
    c.run()
    c.check()


@pytest.mark.parametrize("heads,hk", [(1, 1), (4, 4), (16, 1), (32, 1), (7, 1), (15, 3), (40, 8), (64, 2), (5, 5)])
@pytest.mark.parametrize("n", [1, 3, 9, 40])
def test_head_layouts(flh, gpu, heads, hk, n):
    lens = [(n, n), (n, n + 100), (1, 77), (n, 260)]
    c = Case(flh, gpu, "F32", "F16", heads, hk, 64, 64, 16, "head", lens, 3)
    c.run()
    c.check()


@pytest.mark.parametrize("window", [1, 2, 16, 31, 64, 100, 1000])
@pytest.mark.parametrize("n,act,cdt", [(1, "F32", "BF16"), (8, "F16", "F16"), (150, "BF16", "BF16"), (150, "F32", "F16")])
def test_windows(flh, gpu, window, n, act, cdt):
    lens = [(n, n), (n, n + 333), (1, 500), (n, 700)]
    c = Case(flh, gpu, act, cdt, 4, 2, 128, 128, 16, "head", lens, 4, window=window)
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n", [1, 7, 100])
def test_not_causal(flh, gpu, act, cdt, n):
    """Cross attention: rows over keys of another length, more rows than keys too."""
    lens = [(n, 3), (n, 150), (2, 77), (n, 0), (n, 129)]
    c = Case(flh, gpu, act, cdt, 4, 4, 64, 64, 64, "token", lens, 5, causal=False)
    c.run()
    c.check()


@pytest.mark.parametrize("page", [1, 2, 8, 64, 128, 4096])
@pytest.mark.parametrize("order,pad", [("head", 0), ("token", 8)])
@pytest.mark.parametrize("n", [1, 50])
def test_pages(flh, gpu, page, order, pad, n):
    lens = [(n, 300), (n, 131), (1, 5), (n, 64)]
    c = Case(flh, gpu, "F32", "F16", 4, 2, 128, 128, page, order, lens, 6, cache_pad=pad)
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n", [1, 20, 100])
def test_rows_that_see_nothing(flh, gpu, act, cdt, n):
    """No keys at all, fewer keys than rows (the first rows stand before the first
    key), no rows: zeros, and nothing else changes."""
    lens = [(n, 0), (n, n // 2), (0, 0), (0, 30), (n, 1), (n, n)]
    c = Case(flh, gpu, act, cdt, 8, 2, 128, 128, 16, "head", lens, 7, window=0)
    c.run()
    got = c.check()
    assert (got[:n, :8 * 128] == 0).all()


@pytest.mark.parametrize("pad,lead", [(1, 0), (3, 2), (8, 1)])
@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("F16", "F16")])
@pytest.mark.parametrize("n", [1, 40])
def test_strides_and_leading_rows(flh, gpu, pad, lead, act, cdt, n):
    """Odd strides (rows aligned to an element only), rows before the first
    request and behind the last one."""
    c = Case(flh, gpu, act, cdt, 6, 3, 80, 80, 16, "head", [(n, 99), (n, n), (n, 250)], 8, q_pad=pad, lead=lead)
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n", [1, 8, 90])
def test_long_contexts_split(flh, gpu, act, cdt, n):
    """Few rows over long contexts: the keys of one request are worked on by
    many workgroups and joined."""
    c = Case(flh, gpu, act, cdt, 4, 1, 128, 128, 64, "head", [(n, 9001), (n, 20000)], 9)
    c.run()
    first = c.check().clone()
    for _ in range(2):                                  # joined in the same order every time
        c.run()
        assert torch.equal(c.result(), first)


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n", [1, 70])
def test_max_q_is_a_hint(flh, gpu, act, cdt, n):
    for hint in (0, 1, 5, 100000):
        c = Case(flh, gpu, act, cdt, 8, 2, 64, 64, 16, "head", [(n, 200), (3, 9), (n, n)], 10)
        c.p.max_q = hint
        c.ws()
        c.run()
        c.check()


@pytest.mark.parametrize("n", [1, 60])
def test_bad_table_entries(flh, gpu, n):
    """Keys whose table entry is no page, or behind the table's row, are not seen."""
    c = Case(flh, gpu, "F32", "F16", 4, 2, 128, 128, 16, "head", [(n, 400), (n, 300), (n, 100)], 11)
    c.table[0, 3], c.table[0, 7], c.table[1, 0], c.table[2, :] = NONE, c.cache.n_pages, 0x80000000, NONE
    c.b["table"].upload(c.table.view(np.uint8).reshape(-1), gpu)
    c.run()
    got = c.check()
    assert (got[2 * n:3 * n, :4 * 128] == 0).all()
    c = Case(flh, gpu, "F32", "F16", 4, 2, 128, 128, 16, "head", [(n, 400), (n, 300)], 12)
    c.table = np.ascontiguousarray(c.table[:, :11])     # 176 tokens wide: the rest of the keys lies behind
    c.b["table"].upload(c.table.view(np.uint8).reshape(-1), gpu)
    c.p.table_stride = 11
    c.ws()
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n,window", [(1, 0), (1, 40), (12, 0), (100, 0), (100, 40)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_values_not_seen(flh, gpu, act, cdt, n, window, value):
    """A key or value that is no number is no part of a row that does not see it,
    also inside a tile that other rows of it see."""
    c = Case(flh, gpu, act, cdt, 4, 2, 64, 64, 16, "head", [(n, 150), (n, n + 7)], 13, window=window)
    kv = 150
    at = [kv - n // 2 - 1, 100, 3]                      # a row's own key, inside, near the begin
    for j in at:
        pg = int(c.table[0, j // 16])
        if math.isinf(value):                           # infinite values reach the rows that see them
            c.cache.view[1][pg, j % 16, 0, 5] = value
        else:
            c.cache.view[0][pg, j % 16, 1, 3] = value
            c.cache.view[1][pg, j % 16, 0, 7] = value
    c.cache.push()
    c.run()
    out, mag, amp = attn_oracle(c.q, c.rows, c.kv_len, c.table, c.cache, c.group, c.scale, c.causal, c.window)
    have = c.result()[:, :4 * 64].unflatten(1, (4, 64)).double()[:c.n_tok]
    out, mag, amp = out[:c.n_tok], mag[:c.n_tok], amp[:c.n_tok]
    # a NaN key makes every element of the rows that see it NaN
    nan = torch.isnan(out)
    assert torch.equal(torch.isnan(have), nan)
    inf = torch.isinf(out)
    assert torch.equal(have[inf], out[inf])
    fin = ~nan & ~inf
    lim = attn_bound(out, mag, amp, c.act, c.dk, 200)
    assert ((have - out).abs()[fin] <= lim[fin]).all()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n", [1, 40])
def test_scales(flh, gpu, act, cdt, n):
    """Scale 0 is the mean; large scores pick single keys and stay finite."""
    for scale, amp in ((0.0, 1.0), (1.0, 4.0), (1e-3, 1.0)):
        c = Case(flh, gpu, act, cdt, 4, 2, 64, 64, 16, "head", [(n, 200), (n, n)], 14, scale=scale, amp=amp)
        c.run()
        c.check()


@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e5, 1e18])
@pytest.mark.parametrize("cdt", ["F16", "BF16"])
@pytest.mark.parametrize("n", [1, 40])
def test_fp32_queries_of_any_size(flh, gpu, size, cdt, n):
    """fp32 queries keep their accuracy at every magnitude, also past a 16-bit
    type's range."""
    c = Case(flh, gpu, "F32", cdt, 4, 2, 64, 64, 16, "head", [(n, 150), (n, n)], 15, amp=size, scale=0.1 / size)
    c.run()
    c.check()


def test_nothing_to_do(flh, gpu):
    c = Case(flh, gpu, "F32", "F16", 4, 2, 64, 64, 16, "head", [(0, 10), (0, 0)], 16)
    c.run()
    c.check()
    c.p.n_seq = 0
    c.p.n_tok = 5
    c.run()
    assert torch.equal(c.result(), c.out0)


@pytest.mark.parametrize("act,cdt", [("F32", "F16"), ("BF16", "BF16")])
@pytest.mark.parametrize("n", [1, 6, 90])
def test_captured(flh, gpu, act, cdt, n):
    """A captured call, replayed while lengths, rows and tables on the device
    change, with eager work of the same program in between; each replay equals the
    eager call."""
    lens = [(n, 900), (n, 333), (n, 64 + n)]
    c = Case(flh, gpu, act, cdt, 8, 2, 128, 128, 16, "head", lens, 17)
    with flh.Graph.capture(gpu) as g:
        c.run()
    for step in range(4):
        for i, (r0, r1) in enumerate(c.rows):
            c.kv_len[i] = max(r1 - r0, int(c.kv_len[i]) - 37 * step)
        c.b["kv"].upload(c.kv_len.view(np.uint8), gpu)
        c.b["out"].upload(np.frombuffer(c.out0.contiguous().view(torch.uint8).numpy().tobytes(), np.uint8), gpu)
        g.launch()
        got = c.check().clone()
        c.run()
        assert torch.equal(c.result(), got)
    g.close()


def test_two_streams_at_once(flh, gpu):
    """Calls on two streams, each with a workspace of its own."""
    a = Case(flh, gpu, "F32", "F16", 8, 2, 128, 128, 16, "head", [(1, 5000), (1, 3000)], 18)
    b = Case(flh, gpu, "BF16", "BF16", 8, 2, 128, 128, 16, "head", [(90, 3000), (40, 1000)], 19)
    s1, s2 = flh.Stream(), flh.Stream()
    gpu.sync()
    for _ in range(10):
        a.run(s1)
        b.run(s2)
    s1.sync()
    s2.sync()
    a.check()
    b.check()
    s1.close()
    s2.close()


def test_many_requests(flh, gpu):
    rng = np.random.default_rng(20)
    lens = [(int(rng.integers(0, 4)), int(rng.integers(4, 60))) for _ in range(700)]
    c = Case(flh, gpu, "F32", "F16", 2, 1, 64, 64, 16, "head", lens, 20)
    c.run()
    c.check()


def test_offsets_past_32_bits(flh, gpu):
    """Pages more than 2^32 elements apart: one allocation of 10 GiB, of which a
    request uses pages at both ends."""
    page, d, hk = 16, 128, 2
    stride = (5 << 30) // 2 // 1024 * 8                 # elements between pages
    n_pages = 250
    buf = flh.DeviceBuffer(n_pages * stride * 2)
    rng = np.random.default_rng(21)
    small = Case(flh, gpu, "F32", "F16", 4, hk, d, d, page, "head", [(3, 100), (1, 60)], 21)
    ids = [0, n_pages - 1, 7, 200, 128, 249 - 3, 100, 5, 244, 31, 60, 190, 222]
    table = small.table.copy()
    host = [t.contiguous() for t in small.cache.store]
    new = {}
    for s in range(2):
        for j in range(table.shape[1]):
            if table[s, j] != NONE:
                old = int(table[s, j])
                table[s, j] = ids[len(new)]
                new[old] = int(table[s, j])
    half = page * hk * d
    for old, pg in new.items():
        for i in range(2):
            buf.upload(host[i][old].reshape(-1).view(torch.uint8).numpy(), gpu, offset=(pg * stride + i * half) * 2)
    cache = flh.KvCache(buf.ptr, buf.ptr + half * 2, flh.Dtype.F16, n_pages, page, hk, d, d, (stride, d, page * d), (stride, d, page * d))
    small.b["table"].upload(table.view(np.uint8).reshape(-1), gpu)
    flh.paged_attn(cache, small.p, gpu)
    small.check()
    del rng


def short_items(seed, n_seq, most_rows, most_keys):
    """Requests of few rows over few keys, now and then one over many."""
    rng = np.random.default_rng(seed)
    lens = []
    for i in range(n_seq):
        n = int(rng.integers(0, most_rows + 1))
        kv = n + int(rng.integers(0, most_keys if i % 17 else 40 * most_keys))
        lens.append((n, kv))
    return lens + [(most_rows, most_rows)]


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (192, 128)])
@pytest.mark.parametrize("n_seq", [40, 200, 700])
def test_short_items(flh, gpu, act, cdt, dk, dv, n_seq):
    """Many strips of a tile or two per workgroup: shares end inside, at the begin
    and at the end of them."""
    c = Case(flh, gpu, act, cdt, 8, 1, dk, dv, 16, "head", short_items(n_seq, n_seq, 20, 70), 22)
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("n_seq", [30, 300])
def test_short_items_with_values_not_seen(flh, gpu, act, cdt, n_seq):
    """An infinite value at every request's last key, which only its last row sees."""
    c = Case(flh, gpu, act, cdt, 8, 1, 64, 64, 16, "head", short_items(n_seq + 1, n_seq, 20, 70), 23)
    for i, kv in enumerate(c.kv_len):
        if kv:
            j = int(kv) - 1
            c.cache.view[1][int(c.table[i, j // 16]), j % 16, 0, 5] = math.inf
    c.cache.push()
    c.run()
    c.check()


@pytest.mark.parametrize("act,cdt", TYPES)
def test_wide_groups(flh, gpu, act, cdt):
    """One token of more query heads per kv head than the streaming kernel has rows."""
    c = Case(flh, gpu, act, cdt, 96, 2, 64, 64, 16, "token", [(1, kv) for kv in (1, 63, 64, 65, 500, 3000)], 24)
    c.run()
    c.check()


def test_tiles_in_fours(flh, gpu):
    """Keys around multiples of four tiles of 64 (rows are found for four at once)."""
    lens = [(40, kv) for kv in (64, 128, 192, 255, 256, 257, 319, 320, 321, 448, 511, 512, 513, 768, 1023, 1025)]
    for window in (0, 200, 330):
        c = Case(flh, gpu, "BF16", "BF16", 4, 4, 128, 128, 8, "head", lens, 25, window=window)
        c.run()
        c.check()


def test_a_torch_stream(flh, gpu):
    """A stream that was made elsewhere."""
    c = Case(flh, gpu, "F32", "F16", 8, 2, 128, 128, 16, "head", [(1, 700), (30, 300)], 26)
    gpu.sync()
    t = torch.cuda.Stream()
    c.run(flh.Stream.wrap(t.cuda_stream))
    t.synchronize()
    c.check()


@pytest.mark.parametrize("act,cdt", TYPES)
@pytest.mark.parametrize("max_q", [1, 100])
def test_rows_of_no_request_alone(flh, gpu, act, cdt, max_q):
    """A padded step in which no request adds a token, behind one that left its notes in
    the workspace."""
    c = Case(flh, gpu, act, cdt, 4, 2, 128, 128, 16, "head", [(max_q, 5000), (max_q, 300)], 27)
    c.p.max_q = max_q
    c.ws()
    c.run()
    c.check()
    c.b["out"].upload(raw(c.out0), gpu)
    c.b["start"].upload(np.zeros(3, np.uint32), gpu)
    for _ in range(2):
        c.run()
        assert torch.equal(c.result(), c.out0)


@pytest.mark.parametrize("max_q", [1, 100])
def test_starts_that_do_not_ascend(flh, gpu, max_q):
    """35 requests that all claim the same rows, before 35 of none, give more units of work
    than 32 bits hold: nothing is done, and nothing out of bounds."""
    n, d, page = 1 << 20, 8, 65536
    cache = Cache(flh, gpu, "F16", 1, page, 1, d, d, "head", 0)
    cache.push()
    table = np.full((70, 16), NONE, np.uint32)
    start = np.array([0, n] * 35 + [0], np.uint32)
    kv = np.full(70, 1 << 20, np.uint32)
    q = torch.zeros(n, d, dtype=torch.float16)
    out0 = torch.full((n, d), 3.0, dtype=torch.float16)
    b = [put(flh, gpu, torch.from_numpy(x.view(np.int32))) for x in (start, kv, table)] + [put(flh, gpu, q), put(flh, gpu, out0)]
    p = flh.AttnP(q=b[3].ptr, out=b[4].ptr, q_start=b[0].ptr, kv_len=b[1].ptr, table=b[2].ptr, q_tok=d, q_head=d, o_tok=d, o_head=d,
                  dtype=flh.Dtype.F16, n_head=1, n_seq=70, n_tok=n, max_q=max_q, table_stride=16, scale=1.0, causal=0, window=0)
    p.ws_bytes = flh.paged_attn_ws_bytes(cache.c, p)
    ws = flh.DeviceBuffer(p.ws_bytes)
    p.ws = ws.ptr
    flh.paged_attn(cache.c, p, gpu)
    assert torch.equal(get(b[4], out0, gpu), out0)
