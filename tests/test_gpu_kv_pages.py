"""Pages between steps: requests forked, cut back and freed against a plain account of who
holds what; tokens copied and compacted in several layers."""
import numpy as np
import pytest
import torch

from paged_cases import Cache, NONE, TORCH

pytestmark = pytest.mark.gpu


def up(flh, s, a):
    return flh.DeviceBuffer.from_array(np.ascontiguousarray(a), s, extra=16)


def trim_oracle(kv_len, keep, table, free, taken, shared, page, n_pages):
    """The definition, one request and page after the other."""
    table, free = table.copy(), free.copy()
    shared = None if shared is None else shared.astype(np.int64).copy()
    n, width = table.shape
    held = np.minimum(kv_len, keep).astype(np.uint32)
    top, lost = min(int(taken), len(free)), 0
    src, dst, num = (np.full(n, NONE, np.uint32), np.full(n, NONE, np.uint32), np.zeros(n, np.uint32))
    left = []                                                 # pages that are left, in order
    own = {}
    if shared is not None:
        for s in range(n):
            k = int(held[s])
            if k % page and -(-k // page) <= width:
                j = -(-k // page) - 1
                e = int(table[s, j])
                if e < n_pages and shared[e] > 0:
                    own[s] = (j, e)
        for s, (j, e) in own.items():
            f = int(free[top]) if top < len(free) else NONE
            top = min(top + 1, len(free))
            if f < n_pages:
                src[s], dst[s], num[s] = e * page, f * page, held[s] % page
                table[s, j] = f
            else:
                table[s, j] = NONE
                lost += 1
    for s in range(n):
        if s in own:
            left.append(own[s][1])
        for j in range(min(-(-int(held[s]) // page), width), min(-(-int(kv_len[s]) // page), width)):
            left.append(int(table[s, j]))
            table[s, j] = NONE
    left = [e for e in left if e < n_pages]
    back = []
    for i, e in enumerate(left):
        if shared is None:
            back.append(e)
        elif e not in left[i + 1:]:                           # the last one that leaves it
            k = left.count(e)
            if k > shared[e]:
                back.append(e)
                shared[e] = 0
            else:
                shared[e] -= k
    done = 0
    for e in back:
        if top > 0:
            top -= 1
            free[top] = e
            done += 1
    lost += len(back) - done
    return dict(held=held, table=table, free=free, taken=top, shared=None if shared is None else shared.astype(np.uint32), src=src,
                dst=dst, num=num, info=[done, lost])


class Book:
    """The pages of a few requests, on the device."""

    def __init__(self, flh, s, page, n_seq, width, n_pages, seed, shared=True, n_free=None):
        rng = np.random.default_rng(seed)
        self.flh, self.s, self.page, self.n_seq, self.width, self.n_pages = flh, s, page, n_seq, width, n_pages
        self.free = rng.permutation(n_pages).astype(np.uint32)[:n_free]
        self.taken, self.table = np.uint32(0), np.full((n_seq, width), NONE, np.uint32)
        self.shared = np.zeros(n_pages, np.uint32) if shared else None
        self.kv_len = np.zeros(n_seq, np.uint32)

    def take(self, s, tokens):
        """Request s grows to `tokens`, as a plan would have it."""
        for j in range(-(-int(self.kv_len[s]) // self.page), -(-tokens // self.page)):
            self.table[s, j] = self.free[self.taken]
            self.taken += np.uint32(1)
        self.kv_len[s] = tokens

    def push(self, n_list):
        f, s = self.flh, self.s
        self.b = dict(table=up(f, s, self.table), free=up(f, s, self.free), taken=up(f, s, np.array([self.taken], np.uint32)),
                      kv=up(f, s, self.kv_len), info=up(f, s, np.array([7, 7], np.uint32)),
                      shared=up(f, s, self.shared) if self.shared is not None else None)
        self.lists = [up(f, s, np.full(max(n_list, 1), 0xABABABAB, np.uint32)) for _ in range(3)]
        self.n_list = n_list
        b = self.b
        return dict(kv_len=b["kv"].ptr, table=b["table"].ptr, free_pages=b["free"].ptr, taken=b["taken"].ptr,
                    shared=b["shared"].ptr if b["shared"] else None, info=b["info"].ptr, n_seq=self.n_seq, n_pages=self.n_pages,
                    page_size=self.page, n_free=len(self.free), table_stride=self.width,
                    **{k: x.ptr for k, x in zip(("copy_src", "copy_dst", "copy_n"), self.lists)})

    def read(self):
        s, b = self.s, self.b
        return dict(table=b["table"].download(np.uint32, self.table.size, s).reshape(self.table.shape),
                    free=b["free"].download(np.uint32, len(self.free), s), taken=int(b["taken"].download(np.uint32, 1, s)[0]),
                    shared=b["shared"].download(np.uint32, self.n_pages, s) if b["shared"] else None,
                    held=b["kv"].download(np.uint32, self.n_seq, s), info=b["info"].download(np.uint32, 2, s).tolist(),
                    **{k: x.download(np.uint32, self.n_list, s) for k, x in zip(("src", "dst", "num"), self.lists)})

    def trim(self, keep, held=None):
        p = self.push(self.n_seq)
        k = up(self.flh, self.s, np.array(keep, np.uint32))
        out = up(self.flh, self.s, np.full(self.n_seq, 5, np.uint32)) if held else None
        self.flh.kv_trim(self.flh.KvTrimP(keep=k.ptr, held=out.ptr if held else p["kv_len"], **p), self.s)
        got = self.read()
        if held:
            np.testing.assert_array_equal(got["held"], self.kv_len)
            got["held"] = out.download(np.uint32, self.n_seq, self.s)
        want = trim_oracle(self.kv_len, np.array(keep, np.uint32), self.table, self.free, self.taken, self.shared, self.page, self.n_pages)
        if self.shared is None:
            for x in ("src", "dst", "num"):
                assert (got[x] == 0xABABABAB).all()
                got.pop(x), want.pop(x)
        same(got, want)
        self.adopt(got)
        return got

    def fork(self, src, dst, length=None):
        p = self.push(len(src))
        a = [up(self.flh, self.s, np.array(x, np.uint32)) for x in (src, dst, length if length is not None else [0])]
        self.flh.kv_fork(self.flh.KvForkP(src=a[0].ptr, dst=a[1].ptr, len=a[2].ptr if length is not None else None, n_fork=len(src), **p),
                         self.s)
        got = self.read()
        want = dict(table=self.table.copy(), free=self.free, taken=int(self.taken), shared=self.shared.copy(), held=self.kv_len.copy(),
                    src=np.full(len(src), NONE, np.uint32), dst=np.full(len(src), NONE, np.uint32), num=np.zeros(len(src), np.uint32),
                    info=[0, 0])
        for i, (x, y) in enumerate(zip(src, dst)):
            if x >= self.n_seq or y >= self.n_seq or x == y:
                continue
            n = min(int(self.kv_len[x]), int(length[i]) if length is not None else 1 << 40, self.width * self.page)
            want["held"][y] = n
            for j in range(n // self.page):
                e = self.table[x, j]
                want["table"][y, j] = e if e < self.n_pages else NONE
                if e < self.n_pages:
                    want["shared"][e] += 1
            if n % self.page:
                j, e = n // self.page, int(self.table[x, n // self.page])
                want["table"][y, j] = NONE
                if e < self.n_pages:
                    f = int(self.free[want["taken"]]) if want["taken"] < len(self.free) else NONE
                    want["taken"] += 1
                    want["info"][0 if f < self.n_pages else 1] += 1
                    if f < self.n_pages:
                        want["table"][y, j] = f
                        want["src"][i], want["dst"][i], want["num"][i] = e * self.page, f * self.page, n % self.page
        same(got, want)
        self.adopt(got)
        return got

    def adopt(self, got):
        self.table, self.free, self.taken, self.kv_len = got["table"], got["free"], np.uint32(got["taken"]), got["held"]
        self.shared = got["shared"]

    def sound(self):
        """Every page is free once, or held by as many as its count says."""
        held = [int(e) for s in range(self.n_seq) for e in self.table[s, :-(-int(self.kv_len[s]) // self.page)] if e < self.n_pages]
        free = self.free[min(int(self.taken), len(self.free)):].tolist()
        count = np.bincount(held, minlength=self.n_pages) if held else np.zeros(self.n_pages, int)
        assert len(set(free)) == len(free) and not set(free) & set(held)
        assert len(free) + (count > 0).sum() == self.n_pages
        np.testing.assert_array_equal(self.shared, np.maximum(count - 1, 0))


def same(got, want):
    for k in want:
        np.testing.assert_array_equal(got[k], want[k], err_msg=k)


@pytest.mark.parametrize("page", [1, 16, 128])
@pytest.mark.parametrize("n_seq,width", [(1, 1), (7, 12), (60, 40), (2500, 6)])
def test_forked_and_trimmed(flh, gpu, page, n_seq, width):
    """Rounds of growth, forks (of forks, shorter ones, of several from one), cuts and frees; lengths of zero and one,
    whole pages, full tables."""
    rng = np.random.default_rng(n_seq + page)
    b = Book(flh, gpu, page, n_seq, width, 4 * n_seq * width + 9, 1)
    for _ in range(4):
        for s in range(n_seq):
            if rng.random() < 0.5:
                tokens = int(rng.choice([0, 1, page, width * page, rng.integers(0, width * page + 1)]))
                if tokens >= b.kv_len[s] and (b.kv_len[s] % page == 0 or tokens == b.kv_len[s] or
                                              b.shared[b.table[s, b.kv_len[s] // page]] == 0):
                    b.take(s, tokens)
        b.sound()
        empty = [s for s in range(n_seq) if b.kv_len[s] == 0]
        full = [s for s in range(n_seq) if b.kv_len[s]]
        if empty and full:
            dst = rng.permutation(empty)[:max(1, len(empty) // 2)].tolist()
            src = rng.choice(full, len(dst)).tolist()
            b.fork(src, dst, rng.integers(0, width * page + 9, len(dst)) if rng.random() < 0.5 else None)
            b.sound()
        keep = np.where(rng.random(n_seq) < 0.3, 0, np.where(rng.random(n_seq) < 0.5, 0xFFFFFFFF, rng.integers(0, width * page + 1, n_seq)))
        b.trim(keep.astype(np.uint32), held=rng.random() < 0.5)
        b.sound()
    b.trim(np.zeros(n_seq, np.uint32))
    b.sound()
    assert b.taken == 0 and len(set(b.free.tolist())) == b.n_pages


def test_many_pages(flh, gpu):
    """More pages than threads, of few requests: shared ones, those of the last holder, and whole rows."""
    b = Book(flh, gpu, 16, 6, 6000, 20000, 2)
    b.take(0, 6000 * 16 - 3)
    b.take(1, 5000 * 16)
    b.fork([0, 0, 1], [2, 3, 4])
    b.sound()
    b.trim([0xFFFFFFFF, 0, 0, 17, 4000 * 16 + 5, 9])
    b.sound()
    b.trim([0, 0, 0, 0, 4000 * 16 + 5, 0])
    b.sound()
    b.trim([0] * 6)
    b.sound()
    assert b.taken == 0


def test_a_shared_last_page(flh, gpu):
    """Holders of one partly filled page, each cut back inside it: each gets one of its own, the page
    itself goes back; with one who keeps it whole; and where the list has no page left."""
    for n_free, spare in ((None, 9), (4, 0)):
        b = Book(flh, gpu, 16, 5, 4, 4 + spare, 3, n_free=n_free)
        b.take(0, 64)
        b.fork([0, 0], [1, 2])
        b.trim([40, 41, 64, 0, 0])
        b.trim([40, 3, 0, 0, 0])
        if spare:
            b.sound()


def test_without_counts(flh, gpu):
    b = Book(flh, gpu, 16, 9, 5, 64, 4, shared=False)
    for s in range(9):
        b.take(s, 8 * s + 1)
    b.trim([0, 5, 0xFFFFFFFF, 16, 17, 0, 48, 0, 1])
    b.trim([0] * 9)
    assert b.taken == 0 and sorted(b.free.tolist()) == list(range(64))


def test_entries_that_are_no_pages(flh, gpu):
    """Entries behind a list that ran out, a list that gives no pages, forks of requests that are none, lengths
    behind the table, a taken behind the list; a list that has no room."""
    b = Book(flh, gpu, 16, 6, 4, 40, 5)
    for s in (0, 1):
        b.take(s, 40 + s)
    b.table[0, 1], b.table[1, 2] = NONE, 40
    b.fork([0, 1, 9, 0, 2], [2, 3, 4, 6, 2])
    b.trim([0, 30, 0xFFFFFFFF, 33, 0, 0])
    b = Book(flh, gpu, 16, 6, 4, 40, 6, n_free=4)
    b.take(0, 40)
    b.fork([0, 0, 0], [1, 2, 3])
    assert b.taken == 6
    b.trim([0xFFFFFFFF, 0, 35, 0, 0, 0])
    b = Book(flh, gpu, 16, 6, 4, 40, 7)
    b.take(0, 20)
    b.free[2:] = 1 << 20
    b.fork([0, 0], [1, 2])
    b = Book(flh, gpu, 16, 3, 2, 40, 8)
    b.take(0, 20)
    b.kv_len[:] = [1000, 0xFFFFFFFF, 0]
    b.fork([0, 1], [2, 5])
    b.trim([900, 7, 0])
    b = Book(flh, gpu, 16, 3, 4, 40, 9)
    for s in range(3):
        b.take(s, 64)
    b.taken = np.uint32(5)                                    # 12 pages, of which 5 came off the list
    assert b.trim([0, 0, 0])["info"] == [5, 7]
    b = Book(flh, gpu, 16, 3, 4, 40, 10)
    b.take(0, 64)
    b.table[1, 0] = b.table[0, 0]                             # a page of two, of which the count knows nothing
    b.kv_len[1] = 16
    b.trim([0, 0, 0])


# -------------------------------------------------------------------- tokens --
class Layers:
    def __init__(self, flh, s, n, dtype, n_pages, page, heads, dk, dv, order, pad=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.c = [Cache(flh, s, dtype, n_pages, page, heads, dk, dv, order, pad) for _ in range(n)]
        for c in self.c:
            for t in c.store:
                t.copy_(torch.randn(t.shape, generator=g).to(TORCH[dtype]))
            c.push()
        self.all = flh.KvCaches([c.c for c in self.c])
        self.page = page

    def check(self, moves):
        """moves: (from, to) slots, one after the other."""
        for c in self.c:
            for view, got in zip(c.view, c.pull()):
                for a, b in moves:
                    view[b // self.page, b % self.page] = view[a // self.page, a % self.page].clone()
                assert torch.equal(got, view)


SHAPES = [(1, "F16", 16, 8, 128, 128, "head", 0), (3, "BF16", 16, 2, 64, 64, "token", 8), (2, "F16", 1, 1, 8, 16, "head", 0),
          (66, "F16", 4, 1, 8, 8, "token", 0), (2, "BF16", 64, 5, 80, 40, "head", 16), (1, "F16", 256, 3, 256, 192, "token", 0)]


@pytest.mark.parametrize("layers,dtype,page,heads,dk,dv,order,pad", SHAPES)
def test_copy(flh, gpu, layers, dtype, page, heads, dk, dv, order, pad):
    """Whole pages, parts of them that begin inside, none, copies that reach behind a page's end, slots that are none."""
    rng = np.random.default_rng(1)
    ls = Layers(flh, gpu, layers, dtype, 24, page, heads, dk, dv, order, pad)
    perm = rng.permutation(24)
    src, dst, num, moves = [], [], [], []
    for i in range(9):
        a, b = (int(rng.integers(0, page)), int(rng.integers(0, page))) if i > 3 else (0, 0)
        n = [page, 1, 0, page - 1][i] if i < 4 else int(rng.integers(0, 2 * page))
        x, y = int(perm[2 * i]) * page + a, int(perm[2 * i + 1]) * page + b
        src.append(x), dst.append(y), num.append(n)
        moves += [(x + t, y + t) for t in range(min(n, page - a, page - b))]
    src += [NONE, 5, 24 * page]
    dst += [7, NONE, 3]
    num += [1, 1, 1]
    b = [up(flh, gpu, np.array(x, np.uint32)) for x in (src, dst, num)]
    flh.kv_copy(ls.all, b[0], b[1], b[2], len(src), gpu)
    ls.check(moves)
    flh.kv_copy(ls.all, None, None, None, 0, gpu)
    flh.kv_copy(flh.KvCaches([]), b[0], b[1], b[2], len(src), gpu)
    ls.check([])


@pytest.mark.parametrize("layers,dtype,page,heads,dk,dv,order,pad", SHAPES)
def test_compact(flh, gpu, layers, dtype, page, heads, dk, dv, order, pad):
    """Paths that stay, that move into each other's places, over page borders; tokens without slots, rows that are none,
    requests without rows or paths, paths longer than path_stride."""
    rng = np.random.default_rng(2)
    n = [1, 9, 0, 20, 7, 5, 12, 3]
    rows = sum(n)
    n_pages = max(24, -(-rows // page) + 2)
    ls = Layers(flh, gpu, layers, dtype, n_pages, page, heads, dk, dv, order, pad, 1)
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
    slot = np.concatenate([np.arange(rows - 30) + 1, rng.permutation(np.arange(rows, n_pages * page))[:30]]).astype(np.uint32)[:rows] \
        if n_pages * page - rows >= 30 else rng.permutation(n_pages * page)[:rows].astype(np.uint32)
    slot[int(start[3]) + 4] = NONE
    slot[int(start[6]) + 2] = n_pages * page
    paths = [[0], [0, 1, 2, 5, 8], [], [0, 2, 3, 4, 9, 10, 11, 12, 13, 14, 19], [0, 6], [0, 1, 2, 3, 4], [0, 3, 4, 12, 99], [0, 2]]
    stride, wide = 10, 7
    for stride in (10, 20):
        path = np.full((8, stride), NONE, np.uint32)
        n_path = np.array([len(p) for p in paths], np.uint32)
        n_path[7] = 0
        n_path[2] = 6
        moves = []
        for s, p in enumerate(paths):
            path[s, :min(len(p), stride)] = p[:stride]
            for j, r in enumerate(p[:min(stride, int(n_path[s]))]):
                if j < r < n[s] and j < n[s]:
                    a, b = int(slot[start[s] + r]), int(slot[start[s] + j])
                    if a < n_pages * page and b < n_pages * page:
                        moves.append((a, b))
        b = [up(flh, gpu, x) for x in (start, slot, n_path, path)]
        flh.kv_compact(ls.all, flh.KvCompactP(q_start=b[0].ptr, slot=b[1].ptr, n_path=b[2].ptr, path=b[3].ptr, n_seq=8, n_tok=rows,
                                              path_stride=stride), gpu)
        ls.check(moves)


def test_long_paths_compact(flh, gpu):
    """A path of more tokens than a workgroup has threads, each into the place of the one before."""
    n, page = 700, 16
    ls = Layers(flh, gpu, 2, "F16", 64, page, 2, 64, 64, "head", 0, 2)
    slot = np.random.default_rng(3).permutation(64 * page)[:n].astype(np.uint32)
    path = np.concatenate([[0], np.arange(2, n)]).astype(np.uint32)
    b = [up(flh, gpu, x) for x in (np.array([0, n], np.uint32), slot, np.array([len(path)], np.uint32), path)]
    flh.kv_compact(ls.all, flh.KvCompactP(q_start=b[0].ptr, slot=b[1].ptr, n_path=b[2].ptr, path=b[3].ptr, n_seq=1, n_tok=n,
                                          path_stride=len(path)), gpu)
    ls.check([(int(slot[r]), int(slot[j])) for j, r in enumerate(path) if r != j])


def test_offsets_past_32_bits(flh, gpu):
    """Caches of more than 4 GiB: the first and the last pages."""
    page, n_pages, heads, d = 256, 9000, 8, 128
    n = n_pages * page * heads * d
    buf = flh.DeviceBuffer(2 * n + 64)
    st = (page * heads * d, heads * d, d)
    cache = flh.KvCache(buf.ptr, buf.ptr, flh.Dtype.F16, n_pages, page, heads, d, d, st, st)
    row = heads * d * 2
    last = n_pages * page - 1
    want = np.random.default_rng(4).integers(0, 255, row, dtype=np.uint8)
    buf.upload(want, gpu, offset=last * row)
    b = [up(flh, gpu, np.array(x, np.uint32)) for x in ([last, last], [5, last - page], [1, 1])]
    flh.kv_copy(flh.KvCaches([cache]), b[0], b[1], b[2], 2, gpu)
    for at in (5, last - page):
        np.testing.assert_array_equal(buf.download(np.uint8, row, gpu, offset=at * row), want)
    buf.close()


def test_more_requests_and_copies_than_a_grid_has(flh, gpu):
    """70000 requests of two rows, of which the second one stands where the first was dropped, and as many copies."""
    n, page = 70000, 16
    pages = 2 * n // page + 1
    buf = flh.DeviceBuffer(pages * page * 64)
    rows = np.arange(pages * page, dtype=np.uint32)
    data = np.repeat(rows[:, None], 16, 1)                    # a token: 16 bytes of keys, 48 of values
    buf.upload(data, gpu)
    cache = flh.KvCache(buf.ptr, buf.ptr + 16, flh.Dtype.F16, pages, page, 1, 8, 24, (page * 32, 32, 8), (page * 32, 32, 8))
    start = (2 * np.arange(n + 1)).astype(np.uint32)
    b = [up(flh, gpu, x) for x in (start, np.arange(2 * n, dtype=np.uint32), np.full(n, 1, np.uint32), np.ones(n, np.uint32))]
    flh.kv_compact(flh.KvCaches([cache]), flh.KvCompactP(q_start=b[0].ptr, slot=b[1].ptr, n_path=b[2].ptr, path=b[3].ptr, n_seq=n,
                                                         n_tok=2 * n, path_stride=1), gpu)
    want = rows.copy()
    want[0:2 * n:2] = rows[1:2 * n:2]
    got = buf.download(np.uint32, data.size, gpu).reshape(data.shape)
    assert (got == want[:, None]).all()
    c = [up(flh, gpu, x) for x in (start[:n], start[:n] + np.uint32(1), np.ones(n, np.uint32))]
    buf.upload(data, gpu)
    flh.kv_copy(flh.KvCaches([cache]), c[0], c[1], c[2], n, gpu)
    want = rows.copy()
    want[1:2 * n:2] = rows[0:2 * n:2]
    got = buf.download(np.uint32, data.size, gpu).reshape(data.shape)
    assert (got == want[:, None]).all()


def test_captured(flh, gpu):
    """Fork, copy and trim as graphs of one kernel each, and as one, replayed: the requests go back and forth."""
    b = Book(flh, gpu, 16, 4, 8, 40, 11)
    b.take(0, 75)
    p = b.push(4)
    ls = Layers(flh, gpu, 3, "F16", 40, 16, 2, 64, 64, "head", 0, 5)
    a = [up(flh, gpu, np.array(x, np.uint32)) for x in ([0, 0], [1, 2], [0xFFFFFFFF, 0, 0, 0])]
    first = b.read()
    steps = [lambda: flh.kv_fork(flh.KvForkP(src=a[0].ptr, dst=a[1].ptr, n_fork=2, **p), gpu),
             lambda: flh.kv_copy(ls.all, b.lists[0], b.lists[1], b.lists[2], 2, gpu),
             lambda: flh.kv_trim(flh.KvTrimP(keep=a[2].ptr, held=p["kv_len"], **p), gpu)]
    graphs = []
    for group in ([steps[0]], [steps[1]], [steps[2]], steps):
        with flh.Graph.capture(gpu) as g:
            for f in group:
                f()
        graphs.append(g)
    for turn in range(4):
        if turn % 2:
            graphs[3].launch()
        else:
            graphs[0].launch()
            mid = b.read()
            assert mid["held"].tolist() == [75, 75, 75, 0] and mid["info"] == [2, 0] and mid["taken"] == 7
            assert (mid["shared"][first["table"][0, :4]] == 2).all() and mid["num"][:2].tolist() == [11, 11]
            graphs[1].launch()
            ls.check([(int(mid["src"][i]) + t, int(mid["dst"][i]) + t) for i in range(2) for t in range(11)])
            graphs[2].launch()
        got = b.read()
        assert got["taken"] == 5 and got["held"].tolist() == [75, 0, 0, 0] and got["info"] == [2, 0]
        np.testing.assert_array_equal(got["table"], first["table"])
        assert (got["shared"] == 0).all() and sorted(got["free"][5:].tolist()) == sorted(first["free"][5:].tolist())
    for g in graphs:
        g.close()
