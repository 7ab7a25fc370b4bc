"""Block tables and slot maps against the same rules written out request by
request, page by page, in Python."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


def oracle(held, add, page, free, taken, table, max_tok, slot, pos):
    table, slot, pos = table.copy(), slot.copy(), pos.copy()
    n, width = table.shape
    start, kv, row, lost = [], [], 0, 0
    for s in range(n):
        start.append(min(row, max_tok))
        fit = min(row + int(add[s]), max_tok) - min(row, max_tok)
        row += int(add[s])
        lost += int(add[s]) - fit
        h = int(held[s])
        kv.append(min(h + fit, NONE))
        for j in range(min(-(-h // page), width), min(-(-(h + fit) // page), width)):
            table[s, j] = free[taken] if taken < len(free) else NONE
            taken += 1
        for i in range(fit):
            at = h + i
            g = int(table[s, at // page]) if at // page < width else NONE
            v = NONE if g > (NONE - 1) // page else g * page + at % page
            if g <= (NONE - 1) // page and v >= NONE:
                v = NONE
            slot[start[s] + i] = v
            pos[start[s] + i] = np.int64(at).astype(np.int32)
            lost += v == NONE
    start.append(min(row, max_tok))
    slot[start[-1]:max_tok], pos[start[-1]:max_tok] = NONE, 0
    return dict(table=table, q_start=np.array(start, np.uint32), kv_len=np.array(kv, np.uint32), slot=slot, pos=pos,
                taken=np.array([taken], np.uint32), info=np.array([start[-1], lost], np.uint32))


class Plan:
    """Device buffers of one plan."""

    def __init__(self, flh, s, held, add, page, free, taken, table, max_tok, optional=True):
        u = lambda a: flh.DeviceBuffer.from_array(np.asarray(a), s, extra=16)     # noqa: E731
        self.flh, self.s, n = flh, s, len(held)
        self.slot0, self.pos0 = np.full(max_tok + 5, 77, np.uint32), np.full(max_tok + 5, -77, np.int32)
        self.start0 = np.full(n + 1, 5, np.uint32)
        self.b = dict(held=u(held), add=u(add), free=u(free), taken_in=u(np.array([taken], np.uint32)),
                      taken=u(np.zeros(1, np.uint32)), table=u(table), q_start=u(self.start0), kv_len=u(np.zeros(n, np.uint32)),
                      slot=u(self.slot0), pos=u(self.pos0), info=u(np.zeros(2, np.uint32)))
        b = self.b
        self.shape, self.n = table.shape, n
        self.p = flh.KvPlanP(held=b["held"].ptr, add=b["add"].ptr, free_pages=b["free"].ptr, taken_in=b["taken_in"].ptr,
                             taken=b["taken"].ptr, table=b["table"].ptr, q_start=b["q_start"].ptr, kv_len=b["kv_len"].ptr,
                             slot=b["slot"].ptr, pos=b["pos"].ptr if optional else None,
                             info=b["info"].ptr if optional else None, n_seq=n, page_size=page, n_free=len(free),
                             table_stride=table.shape[1], max_tok=max_tok)

    def read(self):
        d, b, s = {}, self.b, self.s
        d["table"] = b["table"].download(np.uint32, int(np.prod(self.shape)), s).reshape(self.shape)
        d["q_start"] = b["q_start"].download(np.uint32, self.n + 1, s)
        d["kv_len"] = b["kv_len"].download(np.uint32, self.n, s)
        d["slot"] = b["slot"].download(np.uint32, len(self.slot0), s)
        d["pos"] = b["pos"].download(np.int32, len(self.pos0), s)
        d["taken"] = b["taken"].download(np.uint32, 1, s)
        d["info"] = b["info"].download(np.uint32, 2, s)
        return d


def make_table(held, page, width, rng, n_pages):
    t = np.full((len(held), width), NONE, np.uint32)
    perm, at = rng.permutation(n_pages).astype(np.uint32), 0
    for s, h in enumerate(held):
        k = min(-(-int(h) // page), width)
        t[s, :k] = perm[at:at + k]
        at += k
    return t, perm[at:]


def check(got, want, skip=()):
    for k, v in want.items():
        if k not in skip:
            np.testing.assert_array_equal(got[k], v, err_msg=k)


CASES = [
    # requests, held up to, add lo..hi, page, table entries to spare, rows to spare, free pages short by
    (1, 0, 1, 1, 16, 1, 3, 0), (1, 100, 0, 0, 16, 0, 4, 0), (3, 50, 0, 20, 1, 2, 0, 0), (64, 8192, 1, 1, 16, 1, 0, 0),
    (65, 100, 0, 33, 16, 0, 7, 0), (65, 100, 0, 33, 16, 0, -50, 0), (40, 100, 0, 33, 16, -3, 2, 0), (40, 100, 0, 33, 16, 1, 2, 25),
    (40, 100, 5, 33, 8, 1, 2, 1000), (1023, 40, 0, 3, 4, 1, 1, 0), (1024, 40, 0, 3, 4, 1, 1, 3), (2500, 300, 0, 6, 32, 1, 9, 0),
    (500, 3000, 0, 257, 64, 1, 3, 0), (500, 3000, 0, 257, 64, 1, 3, 100), (7, 100000, 2000, 9000, 65536, 1, 11, 0),
    (2, 10, 9000, 9000, 2, 1, -1500, 40)]


@pytest.mark.parametrize("n,held_hi,lo,hi,page,spare,rows,short", CASES)
def test_plan(flh, gpu, n, held_hi, lo, hi, page, spare, rows, short):
    rng = np.random.default_rng(n * 1000 + page)
    held = rng.integers(0, held_hi + 1, n).astype(np.uint32)
    add = rng.integers(lo, hi + 1, n).astype(np.uint32)
    width = max(1, -(-(held_hi + hi) // page) + spare)
    total = sum(-(-(int(h) + int(a)) // page) for h, a in zip(held, add)) + 20
    table, free = make_table(held, page, width, rng, total)
    free = free[:max(1, len(free) - 20 - short + 4)] if short else free
    max_tok = max(0, int(add.sum()) + rows)
    p = Plan(flh, gpu, held, add, page, free, 4, table, max_tok)
    want = oracle(held, add, page, free, 4, table, max_tok, p.slot0, p.pos0)
    for _ in range(2):                                # the same again: nothing is kept between calls
        flh.kv_plan(p.p, gpu)
        check(p.read(), want)
    q = Plan(flh, gpu, held, add, page, free, 4, table, max_tok, optional=False)
    flh.kv_plan(q.p, gpu)
    got = q.read()
    check(got, want, skip=("pos", "info"))
    assert (got["pos"] == q.pos0).all()


def test_no_requests_and_no_rows(flh, gpu):
    table = np.full((1, 4), NONE, np.uint32)
    e = np.zeros(0, np.uint32)
    p = Plan(flh, gpu, e, e, 16, np.arange(3, dtype=np.uint32), 2, table, 0)
    flh.kv_plan(p.p, gpu)
    got = p.read()
    assert got["q_start"].tolist() == [0] and got["taken"].tolist() == [2] and got["info"].tolist() == [0, 0]
    p = Plan(flh, gpu, e, e, 16, np.arange(3, dtype=np.uint32), 2, table, 40000)      # the two-launch form
    flh.kv_plan(p.p, gpu)
    got = p.read()
    assert (got["slot"][:40000] == NONE).all() and (got["pos"][:40000] == 0).all() and (got["slot"][40000:] == 77).all()


def test_table_entries_that_are_no_page(flh, gpu):
    """A begun page that the table does not hold (or a number whose slots pass
    32 bits) gives its rows no slot."""
    held, add = np.array([5, 5, 5], np.uint32), np.array([3, 20, 3], np.uint32)
    table = np.array([[NONE, 0, 0], [NONE, 0, 0], [NONE // 16, 0, 0]], np.uint32)
    free = np.array([7, 9, 11], np.uint32)
    p = Plan(flh, gpu, held, add, 16, free, 0, table, 26)
    want = oracle(held, add, 16, free, 0, table, 26, p.slot0, p.pos0)
    flh.kv_plan(p.p, gpu)
    check(p.read(), want)


def test_lengths_that_pass_32_bits(flh, gpu):
    """Sums of lengths are 64-bit: a garbage length costs its own rows only."""
    held, add = np.array([3, 0xFFFFFFF0, 8], np.uint32), np.array([4, 0xFFFFFFFF, 0xFFFFFFFF], np.uint32)
    table = np.full((3, 4), NONE, np.uint32)
    table[0, 0], table[1, :], table[2, 0] = 1, [2, 3, 4, 5], 6
    free = np.array([7, 9, 11], np.uint32)
    p = Plan(flh, gpu, held, add, 16, free, 0, table, 30)
    flh.kv_plan(p.p, gpu)
    got = p.read()
    assert got["q_start"].tolist() == [0, 4, 30, 30] and got["kv_len"].tolist() == [7, 0xFFFFFFFF, 8]
    assert got["slot"][:4].tolist() == [16 + 3, 16 + 4, 16 + 5, 16 + 6] and (got["slot"][4:30] == NONE).all()
    assert got["info"].tolist() == [30, NONE] and (got["slot"][30:] == 77).all() and got["taken"].tolist() == [0]


@pytest.mark.parametrize("max_tok", [300, 20000])
def test_steps_in_place_and_captured(flh, gpu, max_tok):
    """kv_len may be held and taken taken_in: a captured step, replayed, walks the
    requests on; checked after every replay."""
    rng = np.random.default_rng(5)
    n, page = 37, 16
    held, add = rng.integers(0, 60, n).astype(np.uint32), rng.integers(0, 9, n).astype(np.uint32)
    table, free = make_table(held, page, 12, rng, 400)
    p = Plan(flh, gpu, held, add, page, free, 0, table, max_tok)
    p.p.kv_len, p.p.taken = p.p.held, p.p.taken_in
    p.b["kv_len"], p.b["taken"] = p.b["held"], p.b["taken_in"]
    with flh.Graph.capture(gpu) as g:
        flh.kv_plan(p.p, gpu)
    slot, pos, taken = p.slot0, p.pos0, 0
    for _ in range(5):
        want = oracle(held, add, page, free, taken, table, max_tok, slot, pos)
        g.launch()
        check(p.read(), want)
        held, table, taken, slot, pos = want["kv_len"], want["table"], int(want["taken"][0]), want["slot"], want["pos"]
    g.close()


@pytest.mark.parametrize("max_tok", [6143, 6144, 6145])
def test_rows_around_the_second_launch(flh, gpu, max_tok):
    """The rows of one launch and of two."""
    test_plan(flh, gpu, 76, 300, 80, 80, 16, 3, max_tok - 76 * 80, 0)
