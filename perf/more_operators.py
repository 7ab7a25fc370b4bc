"""A speculative step with trees of drafted tokens over a paged key/value cache, as cases to time.

Five operators, in the order in which a serving step calls them:

  plan     ancestor bits, depths and positions of drafted trees from parents.
  attn     attention of the trees' tokens: each sees the cached tokens and its
           own ancestors.
  verify   which drafted tokens stand against the target's distribution, and
           the token behind them, from given random numbers.
  compact  the accepted path's keys and values moved into place, in all layers.
  pages    requests forked into candidates that share full pages (a partly
           filled page is copied, in all layers) and the candidates dropped again.

Row counts, context lengths and paths belong to the case ("lens" seeds them); every
other value comes from the seed.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # one step of a small batch: trees of up to 16 tokens
        {"name": "plan_step", "op": "plan", "seqs": 8, "q_lo": 5, "q_hi": 16, "window": 0, "lens": 1},
        # a large batch of wide trees, a window that deep nodes feel
        {"name": "plan_wide", "op": "plan", "seqs": 300, "q_lo": 1, "q_hi": 100, "window": 6, "lens": 2},
        # the latency case: one request, a small tree
        {"name": "attn_one", "op": "attn", "act": "f32", "cache": "f16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 16, "order": "head", "seqs": 1, "q_lo": 8, "q_hi": 8, "kv_lo": 4001, "kv_hi": 4001, "window": 0, "lens": 3},
        # a serving batch: ragged trees behind contexts of every length
        {"name": "attn_batch", "op": "attn", "act": "f32", "cache": "f16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 16, "order": "head", "seqs": 32, "q_lo": 1, "q_hi": 25, "kv_lo": 32, "kv_hi": 8192, "window": 0, "lens": 4},
        # wide trees behind long contexts, a sliding window's layer, 16-bit activations
        {"name": "attn_long", "op": "attn", "act": "bf16", "cache": "bf16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 64, "order": "token", "seqs": 4, "q_lo": 64, "q_hi": 64, "kv_lo": 65536, "kv_hi": 65536, "window": 40000,
         "lens": 5},
        # one request whose draft came without a distribution (a suffix match): a chain, the benchmark's vocabulary
        {"name": "verify_one", "op": "verify", "dtype": "f32", "vocab": 128256, "seqs": 1, "q_lo": 5, "q_hi": 5, "kids": 1,
         "draft": False, "greedy": 0.0, "masked": 0.0, "lens": 6},
        # a serving batch of chains from a small model, some requests greedy
        {"name": "verify_chain", "op": "verify", "dtype": "f32", "vocab": 128256, "seqs": 32, "q_lo": 2, "q_hi": 6, "kids": 1,
         "draft": True, "greedy": 0.2, "masked": 0.0, "lens": 7},
        # trees with several candidates a node, an odd vocabulary, tokens that a grammar forbids
        {"name": "verify_tree", "op": "verify", "dtype": "bf16", "vocab": 50257, "seqs": 16, "q_lo": 7, "q_hi": 21, "kids": 3,
         "draft": True, "greedy": 0.1, "masked": 0.5, "lens": 8},
        # one request, all layers of a model
        {"name": "compact_one", "op": "compact", "layers": 32, "cache": "f16", "kv_heads": 8, "d": 128, "page": 16,
         "order": "head", "seqs": 1, "q_lo": 16, "q_hi": 16, "lens": 9},
        # a serving batch
        {"name": "compact_batch", "op": "compact", "layers": 32, "cache": "bf16", "kv_heads": 8, "d": 128, "page": 64,
         "order": "token", "seqs": 64, "q_lo": 1, "q_hi": 25, "lens": 10},
        # one prompt, eight candidates
        {"name": "pages_samples", "op": "pages", "layers": 32, "cache": "f16", "kv_heads": 8, "d": 128, "page": 16,
         "order": "head", "seqs": 1, "fork": 8, "len_lo": 2009, "len_hi": 2009, "lens": 11},
        # a batch of beams over contexts of every length
        {"name": "pages_beams", "op": "pages", "layers": 16, "cache": "bf16", "kv_heads": 8, "d": 128, "page": 64,
         "order": "token", "seqs": 32, "fork": 4, "len_lo": 1, "len_hi": 1500, "lens": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["plan", "attn", "attn", "attn", "verify", "verify", "verify", "compact", "pages"])
    lens = rng.randrange(1 << 30)
    if op == "plan":
        return {"op": op, "seqs": _log_int(rng, 1, 512), "q_lo": rng.randint(0, 2), "q_hi": _log_int(rng, 2, 128),
                "window": rng.choice([0, 0, rng.randint(1, 10)]), "lens": lens}
    if op == "verify":
        kids = rng.choice([1, 1, 2, 3, 4])
        vocab = _log_int(rng, 1000, 256000) if rng.random() < 0.7 else rng.choice([32000, 50257, 128256])
        dtype = rng.choice(["f32", "f32", "f16", "bf16"])
        q_hi = rng.randint(2, 9) if kids == 1 else rng.randint(3, 30)
        return {"op": op, "dtype": dtype, "vocab": vocab, "seqs": _log_int(rng, 1, max(2, 13000000 // (q_hi * vocab))),
                "q_lo": rng.choice([1, 2, q_hi]), "q_hi": q_hi, "kids": kids, "draft": rng.random() < 0.7,
                "greedy": rng.choice([0.0, 0.3]), "masked": rng.choice([0.0, 0.0, 0.9]), "lens": lens}
    cache = rng.choice(["f16", "bf16"])
    page, order = rng.choice([16, 16, 32, 64, 128]), rng.choice(["head", "token"])
    if op in ("compact", "pages"):
        c = {"op": op, "layers": rng.randint(1, 16), "cache": cache, "kv_heads": rng.choice([1, 2, 4, 8, 8]),
             "d": rng.choice([64, 80, 128, 128, 256]), "page": page, "order": order}
        if op == "compact":
            q_hi = _log_int(rng, 2, 64)
            c.update(seqs=_log_int(rng, 1, 2048 // q_hi), q_lo=rng.choice([1, q_hi]), q_hi=q_hi)
        else:
            seqs, fork = _log_int(rng, 1, 24), rng.randint(1, 6)
            len_hi = _log_int(rng, 1, 24000 // seqs)
            c.update(seqs=seqs, fork=fork, len_lo=rng.choice([1, len_hi]), len_hi=len_hi)
        return dict(c, lens=lens)
    act = rng.choice(["f32", cache])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
    dk, dv = rng.choice([(128, 128), (128, 128), (128, 128), (64, 64), (80, 80), (96, 96), (192, 128), (256, 256)])
    seqs = _log_int(rng, 1, 64)
    q_hi = _log_int(rng, 2, 128)
    most = min(131072, 180000000 // (seqs * kv_heads * (dk + dv)), 500000000 // (seqs * heads * q_hi))
    kv_hi = _log_int(rng, q_hi, max(q_hi + 1, most))
    return {"op": op, "act": act, "cache": cache, "heads": heads, "kv_heads": kv_heads, "dk": dk, "dv": dv, "page": page,
            "order": order, "seqs": seqs, "q_lo": rng.choice([1, q_hi]), "q_hi": q_hi,
            "kv_lo": rng.choice([1, (kv_hi + 1) // 2, kv_hi]), "kv_hi": kv_hi,
            "window": _log_int(rng, 2, 8192) if rng.random() < 0.25 else 0, "lens": lens}


# ----------------------------------------------------------------- inputs --
def _gen(seed, k):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + k) % (1 << 62))
    return g


def _randn(seed, k, shape, dtype=torch.float32):
    return torch.randn(shape, generator=_gen(seed, k), device=DEV, dtype=dtype)


def _rand(seed, k, shape):
    return torch.rand(shape, generator=_gen(seed, k), device=DEV)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _up(a, b):
    return -(-a // b)


def _counts(c):
    """Rows of each request; the first has the most."""
    r = random.Random(c["lens"])
    return [c["q_hi"]] + [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["seqs"] - 1)]


def _starts(n):
    at = [0]
    for x in n:
        at.append(at[-1] + x)
    return _ints(at)


def _place(start, rows):
    """Request and index inside it of each row."""
    at = torch.arange(rows, device=DEV)
    s = torch.searchsorted(start[1:].long().contiguous(), at, right=True)
    return s, at - start.long()[s]


def _parents(seed, index):
    """Trees as a draft model grows them: a token hangs on one of the four before it."""
    back = (_rand(seed, 90, index.shape) * index.clamp(max=4)).long()
    return (index - 1 - back).int()


def _prepare_plan(c, seed):
    n = _counts(c)
    rows, start, words = sum(n), _starts(n), _up(max(n), 32)
    _, index = _place(start, rows)
    return {"c": c, "start": start, "parent": _parents(seed, index), "rows": rows, "words": words,
            "kv_len": start[1:] - start[:-1] + torch.randint(0, 9000, (c["seqs"],), generator=_gen(seed, 2), device=DEV,
                                                             dtype=torch.int32),
            "mask": torch.zeros(rows, words, dtype=torch.int32, device=DEV),
            "depth": torch.zeros(rows, dtype=torch.int32, device=DEV), "pos": torch.zeros(rows, dtype=torch.int32, device=DEV)}


def _attn_lens(c):
    r = random.Random(c["lens"] + 1)
    n = _counts(c)
    return n, [max(a, b) for a, b in zip(n, [c["kv_hi"]] + [r.randint(c["kv_lo"], c["kv_hi"]) for _ in n[1:]])]


def _stored(c, t):
    """[..][page][token][head][d] in the order that the case stores it in."""
    return (t.transpose(-2, -3) if c["order"] == "head" else t).contiguous()


def _by_token(c, t):
    return t.transpose(-2, -3) if c["order"] == "head" else t


def _prepare_attn(c, seed):
    n, kl = _attn_lens(c)
    page, hk, h = c["page"], c["kv_heads"], c["heads"]
    stride = _up(max(kl), page) + 1
    pages = [_up(k, page) for k in kl]
    n_pages = sum(pages) + 3
    perm = torch.randperm(n_pages, generator=_gen(seed, 0), device=DEV).to(torch.int32)
    table = torch.full((c["seqs"], stride), -1, dtype=torch.int32, device=DEV)
    table[torch.arange(stride, device=DEV)[None, :] < _ints(pages)[:, None]] = perm[: sum(pages)]
    kv = [_randn(seed, 10 + i, (n_pages, page, hk, d), DT[c["cache"]]) for i, d in enumerate((c["dk"], c["dv"]))]
    kv[0].mul_(torch.where(_rand(seed, 12, (c["dk"],)) < 0.03, 3.0, 1.0).to(kv[0].dtype))
    # what no request has written yet is no number
    used = torch.zeros(n_pages, page, dtype=torch.bool, device=DEV)
    inside = (torch.arange(stride * page, device=DEV)[None, :] < _ints(kl)[:, None]).view(c["seqs"], stride, page)
    there = table >= 0
    used[table[there].long()] = inside[there]
    for t in kv:
        t.masked_fill_(~used[:, :, None, None], float("nan"))
    kc, vc = [_stored(c, t) for t in kv]
    rows = sum(n)
    x = _randn(seed, 1, (rows, h * c["dk"] + hk * (c["dk"] + c["dv"])))   # rows of one product
    x.mul_(torch.where(_rand(seed, 3, (x.shape[1],)) < 0.02, 4.0, 1.0))
    x = x.to(DT[c["act"]])
    plan = _prepare_plan(c, seed)
    bits = _tree(plan)
    return {"c": c, "x": x, "q": x[:, : h * c["dk"]].unflatten(1, (h, c["dk"])), "kc": kc, "vc": vc, "n_pages": n_pages,
            "table": table, "start": plan["start"], "kv_len": _ints(kl), "max_q": max(n), "max_kv": max(kl), "rows": rows,
            "parent": plan["parent"], "mask": bits["mask"], "depth": bits["depth"],
            "out": torch.zeros(rows, h, c["dv"], device=DEV, dtype=DT[c["act"]])}


def _prepare_verify(c, seed):
    n = _counts(c)
    rows, start, v = sum(n), _starts(n), c["vocab"]
    s, index = _place(start, rows)
    parent = ((index - 1) // c["kids"]).int() if c["kids"] > 1 else (index - 1).int()
    at = (start.long()[s] + parent.clamp(min=0)).clamp(max=rows - 1)     # the parent's row
    # a few likely tokens above many unlikely ones, as a language model has them
    target = _randn(seed, 20, (rows, v)).mul_(2.0)
    target += 14.0 * _rand(seed, 21, (rows, v)).sub_(1 - 64.0 / v).clamp_(min=0).mul_(v / 64.0)
    draft = target + 0.6 * _randn(seed, 22, (rows, v)) if c["draft"] else None
    if c["masked"]:
        no = _rand(seed, 23, (rows, v)) < c["masked"]
        target.masked_fill_(no, -math.inf)
        if c["draft"]:
            draft.masked_fill_(no, -math.inf)
    target = target.to(DT[c["dtype"]])
    draft = draft.to(DT[c["dtype"]]) if c["draft"] else None
    temp = 0.6 + 0.6 * _rand(seed, 24, (c["seqs"],))
    inv_temp = torch.where(_rand(seed, 25, (c["seqs"],)) < c["greedy"], math.inf, 1 / temp).float()
    hot = torch.where(torch.isinf(inv_temp), 8.0, inv_temp)[s]
    noise = _rand(seed, 26, (rows, v)).clamp_(min=1e-12).log_().neg_().log_().neg_()
    token = ((draft if c["draft"] else target).float()[at] * hot[:, None] + noise).argmax(1).int()
    z = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)                    # noqa: E731
    path = max(n)
    return {"c": c, "target": target, "draft": draft, "start": start, "token": token, "parent": parent, "inv_temp": inv_temp,
            "u_accept": _rand(seed, 27, (rows,)), "u_next": _rand(seed, 28, (c["seqs"],)), "rows": rows, "max_path": path,
            "kv_len": start[1:] - start[:-1] + 1000, "n_path": z(c["seqs"]), "path": z(c["seqs"], path), "next": z(c["seqs"]),
            "logp": torch.zeros(c["seqs"], path, device=DEV), "len": z(c["seqs"])}


def _paths(c):
    """Accepted rows of each request, up to eight and the root: [(index of the row, ..), ..]"""
    r = random.Random(c["lens"] + 2)
    got = []
    for n in _counts(c):
        k = r.randint(0, min(n - 1, 8)) if n else 0
        got.append([0] + sorted(r.sample(range(1, n), k)) if n else [])
    return got


def _layers(c, seed, n_pages):
    """Keys and values of all layers: [layer][page].."""
    return [_stored(c, _randn(seed, 30 + i, (c["layers"], n_pages, c["page"], c["kv_heads"], c["d"]), DT[c["cache"]]))
            for i in range(2)]


def _prepare_compact(c, seed):
    n, paths = _counts(c), _paths(c)
    rows = sum(n)
    n_pages = _up(2 * rows, c["page"]) + 5
    slot = torch.randperm(n_pages * c["page"], generator=_gen(seed, 4), device=DEV)[:rows].to(torch.int32)
    kc, vc = _layers(c, seed, n_pages)
    wide = max(len(p) for p in paths)
    path = torch.full((c["seqs"], wide), -1, dtype=torch.int32)
    for s, p in enumerate(paths):
        path[s, : len(p)] = torch.tensor(p, dtype=torch.int32)
    return {"c": c, "kc": kc, "vc": vc, "n_pages": n_pages, "start": _starts(n), "slot": slot, "rows": rows, "path": path.to(DEV),
            "n_path": _ints([len(p) for p in paths])}


def _page_lens(c):
    r = random.Random(c["lens"])
    return [c["len_hi"]] + [r.randint(c["len_lo"], c["len_hi"]) for _ in range(c["seqs"] - 1)]


def _prepare_pages(c, seed):
    lens = _page_lens(c)
    page, f = c["page"], c["seqs"] * c["fork"]
    n_seq = c["seqs"] + f
    stride = _up(max(lens), page) + 1
    pages = [_up(x, page) for x in lens]
    held = sum(pages)
    n_pages = held + f + 9
    perm = torch.randperm(n_pages, generator=_gen(seed, 0), device=DEV).to(torch.int32)
    row = torch.randperm(n_seq, generator=_gen(seed, 1), device=DEV)     # table rows, in any order
    src, dst = row[: c["seqs"]], row[c["seqs"]:]
    table = torch.full((n_seq, stride), -1, dtype=torch.int32, device=DEV)
    part = torch.full((c["seqs"], stride), -1, dtype=torch.int32, device=DEV)
    part[torch.arange(stride, device=DEV)[None, :] < _ints(pages)[:, None]] = perm[:held]
    table[src] = part
    kv_len = torch.zeros(n_seq, dtype=torch.int32, device=DEV)
    kv_len[src] = _ints(lens)
    keep = torch.full((n_seq,), -1, dtype=torch.int32, device=DEV)       # all that they hold
    keep[dst] = 0
    kc, vc = _layers(c, seed, n_pages)
    lists = lambda n: torch.zeros(3, n, dtype=torch.int32, device=DEV)                       # noqa: E731
    return {"c": c, "kc": kc, "vc": vc, "n_pages": n_pages, "table": table, "kv_len": kv_len, "keep": keep, "free": perm.clone(),
            "taken": _ints([held]), "shared": torch.zeros(n_pages, dtype=torch.int32, device=DEV),
            "src": src.repeat_interleave(c["fork"]).int(), "dst": dst.int(), "n_seq": n_seq, "copies": lists(f),
            "last": lists(n_seq), "info": torch.zeros(2, 2, dtype=torch.int32, device=DEV)}


def prepare(case, seed):
    return {"plan": _prepare_plan, "attn": _prepare_attn, "verify": _prepare_verify, "compact": _prepare_compact,
            "pages": _prepare_pages}[case["op"]](case, seed)


# ------------------------------------------------------------ plain forms --
def _ancestors(parent, start, rows):
    """[row][index]: the row at that index of its request is the row or above it."""
    s, index = _place(start, rows)
    wide = int((start[1:] - start[:-1]).max())
    up = torch.zeros(start.shape[0] - 1, wide + 1, wide + 1, device=DEV)  # (a place behind the last one takes the roots)
    up[s, index, torch.where(parent >= 0, parent.long(), wide)] = 1.0
    up[:, :, wide] = 0.0
    see = (up + torch.eye(wide + 1, device=DEV)).clamp(max=1)
    for _ in range(max(1, math.ceil(math.log2(wide + 1)))):              # twice as far each time
        see = torch.matmul(see, see).clamp(max=1)
    return see[s, index, :wide] > 0


def _tree(st):
    c, start, rows = st["c"], st["start"], st["rows"]
    s, _ = _place(start, rows)
    see = _ancestors(st["parent"], start, rows)
    depth = see.sum(1) - 1
    if c["window"]:
        at = (start.long()[s][:, None] + torch.arange(see.shape[1], device=DEV)).clamp(max=rows - 1)
        see = see & (depth[:, None] - depth[at] < c["window"])
    pad = st["words"] * 32 - see.shape[1]
    bits = torch.cat([see, see.new_zeros(rows, pad)], 1).view(rows, st["words"], 32).long()
    words = (bits << torch.arange(32, device=DEV)).sum(2)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).int()
    n = start[1:] - start[:-1]
    return {"mask": words, "depth": depth.int(), "pos": (st["kv_len"] - n)[s].int() + depth.int()}


def _plain_attn(st):
    c = st["c"]
    hk, g, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["page"]
    start, kl = st["start"].long(), st["kv_len"].long()
    n, mq, mk = kl.shape[0], st["max_q"], st["max_kv"]
    j = torch.arange(mk, device=DEV)
    there = j[None, :] < kl[:, None]
    pg = st["table"][:, j // page].long().clamp(min=0)
    k, v = [_by_token(c, t)[pg, j % page].float().masked_fill_(~there[:, :, None, None], 0.0).transpose(1, 2)
            for t in (st["kc"], st["vc"])]
    i = torch.arange(mq, device=DEV)
    ql = start[1:] - start[:-1]
    real = i[None, :] < ql[:, None]
    at = (start[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][at].float().unflatten(2, (hk, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (c["dk"] ** -0.5)
    p0 = (kl - ql)[:, None, None]
    see = (j < p0).expand(n, mq, mk)
    if c["window"]:
        see = see & (j > p0 + st["depth"].long()[at][:, :, None] - c["window"])
    b = (j - p0).clamp(min=0, max=st["mask"].shape[1] * 32 - 1).expand(n, mq, mk)
    bit = (st["mask"][at].gather(2, b >> 5) >> (b & 31)) & 1
    see = (see | ((j >= p0) & (bit > 0))) & there[:, None, :]
    s = s.unflatten(2, (g, mq)).masked_fill_(~see[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top > float("-inf"), top, 0.0)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.flatten(2, 3), v).unflatten(2, (g, mq))
    o = torch.where(total > 0, o / total, 0.0)
    out = st["out"].clone()
    out[at[real]] = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[real].to(out.dtype)
    return {"out": out}


def _probs(x, it):
    """exp(it x) over its sum, in 64 bits; the first of the largest for an infinite it (greedy)."""
    x, it = x.double(), it.double()[:, None]
    top = x.amax(1, keepdim=True)
    e = ((x - top) * torch.where(torch.isinf(it), 1.0, it)).exp_()
    e = e.div_(e.sum(1, keepdim=True))
    first = torch.where(x == top, torch.arange(x.shape[1], device=DEV), x.shape[1]).amin(1, keepdim=True)
    return torch.where(torch.isinf(it), torch.zeros_like(e).scatter_(1, first, 1.0), e)


def _plain_verify(st):
    # In 64 bits throughout: a random number may lie next to a border between two tokens.
    c, start, rows = st["c"], st["start"], st["rows"]
    s, index = _place(start, rows)
    n_seq, wide = c["seqs"], st["max_path"]
    it = st["inv_temp"][s]
    p = _probs(st["target"], it)
    # (a greedy request's tokens stand where they are the target's choice, however they were drafted)
    q = _probs(st["draft"], it).masked_fill_(torch.isinf(it)[:, None], 0.0) if c["draft"] else None
    parent, token = st["parent"].long(), st["token"].long()
    is_child = parent >= 0
    at = torch.where(is_child, start.long()[s] + parent, 0)              # the parent's row
    row = torch.arange(rows, device=DEV)
    same = (at[:, None] == at[None, :]) & is_child[:, None] & is_child[None, :]
    rank = (same & (row[None, :] < row[:, None])).sum(1)                 # siblings in front
    kids = torch.zeros(rows, dtype=torch.long, device=DEV).index_add_(0, at, is_child.long())
    pc = p[at, token]
    u = st["u_accept"].double()
    if c["draft"]:
        # p_i = max(p - t_i q, 0) / n_i is what is left when i siblings are rejected
        t, norm = [p.new_zeros(rows)], [p.new_ones(rows)]
        for _ in range(c["kids"]):
            t.append(t[-1] + norm[-1])
            norm.append((p - t[-1][:, None] * q).clamp_(min=0).sum(1))
        t, norm = torch.stack(t, 1), torch.stack(norm, 1)
        qc = q[at, token]
        ok = is_child & (u * qc * norm[at, rank] < (pc - t[at, rank] * qc).clamp(min=0))
    else:
        twice = (same & (row[None, :] < row[:, None]) & (token[None, :] == token[:, None])).any(1)
        gone = (torch.where(twice, 0.0, pc)[None, :] * (same & (row[None, :] < row[:, None]))).sum(1)
        ok = is_child & ~twice & (u * (1 - gone) < pc)
    ok = ok & ~(same & (row[None, :] < row[:, None]) & ok[None, :]).any(1)     # the first that is accepted
    see = _ancestors(st["parent"], start, rows)
    anc = (start.long()[s][:, None] + torch.arange(see.shape[1], device=DEV)).clamp(max=rows - 1)
    on = (~see | ok[anc] | ~is_child[anc]).all(1) & (see.any(1))         # accepted with all above it
    n_path = torch.zeros(n_seq, dtype=torch.long, device=DEV).index_add_(0, s, on.long())
    place = torch.cumsum(on, 0) - 1
    place = place - (torch.cumsum(n_path, 0) - n_path)[s]
    path = torch.full((n_seq, wide), -1, dtype=torch.long, device=DEV)
    path[s[on], place[on]] = index[on]
    end = start.long()[:-1] + path.gather(1, (n_path - 1)[:, None])[:, 0]      # the last accepted row
    pe = p[end]
    if c["draft"]:
        left = (pe - t[end, kids[end]][:, None] * q[end]).clamp_(min=0)
    else:
        left = pe.clone()
        below = is_child & (at == end[s])
        left[s[below], token[below]] = 0.0
    left = torch.where(left.sum(1, keepdim=True) > 0, left, pe)
    cum = left.cumsum(1)
    over = cum > st["u_next"].double()[:, None] * cum[:, -1:]
    nxt = torch.where(over, torch.arange(c["vocab"], device=DEV), c["vocab"]).amin(1)
    logp = torch.zeros(n_seq, wide, dtype=torch.float64, device=DEV)
    below = on & is_child
    logp[s[below], place[below] - 1] = pc[below].log()
    logp.scatter_(1, (n_path - 1)[:, None], pe.gather(1, nxt[:, None]).log())
    n = start[1:] - start[:-1]
    return {"n_path": n_path.int(), "path": path.int(), "next": nxt.int(), "logp": logp.float(),
            "len": st["kv_len"] - n + n_path.int()}


def _plain_compact(st):
    c, page = st["c"], st["c"]["page"]
    path, n_path = st["path"].long(), st["n_path"].long()
    j = torch.arange(path.shape[1], device=DEV)
    moved = (j[None, :] < n_path[:, None]) & (path != j)
    first = st["start"].long()[:-1, None]
    src, dst = st["slot"][(first + path)[moved]].long(), st["slot"][(first + j)[moved]].long()
    for t in (st["kc"], st["vc"]):
        t = _by_token(c, t)
        t[:, dst // page, dst % page] = t[:, src // page, src % page]
    return {"k": st["kc"], "v": st["vc"]}


def _copies(some, src, dst, n):
    """The copies of whole or partly filled pages: from which slot, to which, how many tokens."""
    return torch.stack([torch.where(some, src, -1), torch.where(some, dst, -1), torch.where(some, n, 0)]).int()


def _plain_copy(st, lists):
    c, page = st["c"], st["c"]["page"]
    src, dst, n = lists.long()
    j = torch.arange(page, device=DEV)
    on = j[None, :] < n[:, None]
    src, dst = (src[:, None] + j)[on], (dst[:, None] + j)[on]
    for t in (st["kc"], st["vc"]):
        t = _by_token(c, t)
        t[:, dst // page, dst % page] = t[:, src // page, src % page]


def _plain_pages(st):
    c, page, n_pages = st["c"], st["c"]["page"], st["n_pages"]
    table, free, kv_len, shared = st["table"], st["free"], st["kv_len"], st["shared"]
    n_free, taken = free.shape[0], st["taken"].long()
    j = torch.arange(table.shape[1], device=DEV)[None, :]
    # fork: full pages are shared, a partly filled one is a fresh one's source
    src, dst = st["src"].long(), st["dst"].long()
    held = kv_len[src].long()
    full, rest = held // page, held % page
    at = taken + torch.cumsum(rest > 0, 0) - (rest > 0).long()
    fresh = torch.where(at < n_free, free[at.clamp(max=n_free - 1)], -1)
    mine = table[src]
    last = mine.gather(1, full[:, None].clamp(max=table.shape[1] - 1))[:, 0]
    table[dst] = torch.where(j < full[:, None], mine, torch.where((j == full[:, None]) & (rest > 0)[:, None], fresh[:, None], table[dst]))
    pages = mine[j < full[:, None]].long()
    shared.index_add_(0, pages, torch.ones_like(pages, dtype=torch.int32))
    kv_len[dst] = held.int()
    some = (rest > 0) & (fresh >= 0)
    st["copies"].copy_(_copies(some, last * page, fresh * page, rest))
    st["info"][0] = torch.stack([(some).sum(), ((rest > 0) & (fresh < 0)).sum()]).int()
    taken = taken + (rest > 0).sum()
    _plain_copy(st, st["copies"])
    # trim: to the lengths kept; a last page that others hold too is left to them
    held = kv_len.long()
    keep = torch.where(st["keep"] < 0, held, torch.minimum(held, st["keep"].long()))
    before, after, rest = _up(held, page), _up(keep, page), keep % page
    last = table.gather(1, (after - 1).clamp(min=0)[:, None])[:, 0]
    own_one = (rest > 0) & (last >= 0) & (shared[last.clamp(min=0).long()] > 0)
    at = taken + torch.cumsum(own_one, 0) - own_one.long()
    fresh = torch.where(at < n_free, free[at.clamp(max=n_free - 1)], -1)
    some = own_one & (fresh >= 0)
    st["last"].copy_(_copies(some, last * page, fresh * page, rest))
    top = torch.clamp(taken + own_one.sum(), max=n_free)
    begin = torch.where(own_one, after - 1, after)[:, None]
    gone = (j >= begin) & (j < before[:, None])
    drop = table[gone]
    drop = drop[drop >= 0].long()
    i = torch.arange(drop.shape[0], device=DEV)
    count = torch.zeros(n_pages, dtype=torch.int32, device=DEV).index_add_(0, drop, torch.ones_like(drop, dtype=torch.int32))
    final = torch.full((n_pages,), -1, dtype=torch.long, device=DEV).scatter_reduce_(0, drop, i, "amax")
    back = drop[(final[drop] == i) & (count[drop] > shared[drop])]
    shared.copy_((shared - count).clamp(min=0))
    table.masked_fill_(gone, -1)
    table.copy_(torch.where(own_one[:, None] & (j == after[:, None] - 1), fresh[:, None], table))
    to = top - 1 - torch.arange(back.shape[0], device=DEV)                # one after another: the last is taken next
    free[to[to >= 0]] = back[to >= 0].int()
    kv_len.copy_(keep.int())
    st["taken"].copy_((top - back.shape[0]).clamp(min=0).int())
    st["info"][1] = torch.stack([(to >= 0).sum(), (to < 0).sum() + (own_one & (fresh < 0)).sum()]).int()
    _plain_copy(st, st["last"])
    return {k: st[v] for k, v in PAGES.items()}


PAGES = {"k": "kc", "v": "vc", "table": "table", "kv_len": "kv_len", "free": "free", "taken": "taken", "shared": "shared",
         "copies": "copies", "last": "last", "info": "info"}


# -------------------------------------------------- the framework's calls --
_flh = None


def _lib():
    global _flh
    if _flh is None:
        import __graft_entry__
        _flh = __graft_entry__._pkg()
        _flh.init(0)
    return _flh


def _stream(flh):
    return flh.Stream.wrap(torch.cuda.current_stream().cuda_stream)


def _cache(flh, c, k, v, n_pages, dk, dv):
    """The cache as the library sees it: element strides of a page, a token, a head."""
    page, hk = c["page"], c["kv_heads"]

    def strides(d):
        return (page * hk * d, d, page * d) if c["order"] == "head" else (page * hk * d, hk * d, d)
    return flh.KvCache(k.data_ptr(), v.data_ptr(), flh.Dtype[c["cache"].upper()], n_pages, page, hk, dk, dv, strides(dk), strides(dv))


def _own_plan(st):
    flh = _lib()
    if "p" not in st:
        st["p"] = flh.TreePlanP(
            q_start=st["start"].data_ptr(), parent=st["parent"].data_ptr(), kv_len=st["kv_len"].data_ptr(),
            mask=st["mask"].data_ptr(), depth=st["depth"].data_ptr(), pos=st["pos"].data_ptr(), n_seq=st["c"]["seqs"],
            n_tok=st["rows"], mask_stride=st["words"], window=st["c"]["window"])
    flh.tree_plan(st["p"], _stream(flh))
    return {k: st[k] for k in ("mask", "depth", "pos")}


def _own_attn(st):
    flh, c = _lib(), st["c"]
    if "p" not in st:
        st["cache"] = _cache(flh, c, st["kc"], st["vc"], st["n_pages"], c["dk"], c["dv"])
        q, o = st["q"], st["out"]
        p = flh.AttnP(
            q=q.data_ptr(), out=o.data_ptr(), q_start=st["start"].data_ptr(), kv_len=st["kv_len"].data_ptr(),
            table=st["table"].data_ptr(), q_tok=q.stride(0), q_head=q.stride(1), o_tok=o.stride(0), o_head=o.stride(1),
            dtype=flh.Dtype[c["act"].upper()], n_head=c["heads"], n_seq=c["seqs"], n_tok=st["rows"], max_q=st["max_q"],
            table_stride=st["table"].shape[1], scale=c["dk"] ** -0.5, causal=1, window=c["window"])
        p.ws_bytes = flh.tree_attn_ws_bytes(st["cache"], p)
        st["ws"] = torch.empty(max(p.ws_bytes, 1), dtype=torch.uint8, device=DEV)
        p.ws = st["ws"].data_ptr()
        st["p"] = p
        st["t"] = flh.TreeP(mask=st["mask"].data_ptr(), depth=st["depth"].data_ptr(), mask_stride=st["mask"].shape[1])
    flh.tree_attn(st["cache"], st["p"], st["t"], _stream(flh))
    return {"out": st["out"]}


def _own_verify(st):
    flh, c = _lib(), st["c"]
    if "p" not in st:
        p = flh.VerifyP(
            target=st["target"].data_ptr(), draft=st["draft"].data_ptr() if c["draft"] else None,
            q_start=st["start"].data_ptr(), token=st["token"].data_ptr(), parent=st["parent"].data_ptr(),
            inv_temp=st["inv_temp"].data_ptr(), u_accept=st["u_accept"].data_ptr(), u_next=st["u_next"].data_ptr(),
            kv_len=st["kv_len"].data_ptr(), n_path=st["n_path"].data_ptr(), path=st["path"].data_ptr(),
            next=st["next"].data_ptr(), logp=st["logp"].data_ptr(), len=st["len"].data_ptr(), t_row=c["vocab"], d_row=c["vocab"],
            dtype=flh.Dtype[c["dtype"].upper()], n_seq=c["seqs"], n_tok=st["rows"], vocab=c["vocab"],
            path_stride=st["max_path"], max_child=c["kids"])
        p.ws_bytes = flh.spec_verify_ws_bytes(p)
        st["ws"] = torch.empty(max(p.ws_bytes, 1), dtype=torch.uint8, device=DEV)
        p.ws = st["ws"].data_ptr()
        st["p"] = p
    flh.spec_verify(st["p"], _stream(flh))
    return {k: st[k] for k in ("n_path", "path", "next", "logp", "len")}


def _all_layers(flh, st):
    c = st["c"]
    return flh.KvCaches([_cache(flh, c, st["kc"][i], st["vc"][i], st["n_pages"], c["d"], c["d"]) for i in range(c["layers"])])


def _own_compact(st):
    flh = _lib()
    if "p" not in st:
        st["caches"] = _all_layers(flh, st)
        st["p"] = flh.KvCompactP(
            q_start=st["start"].data_ptr(), slot=st["slot"].data_ptr(), n_path=st["n_path"].data_ptr(),
            path=st["path"].data_ptr(), n_seq=st["c"]["seqs"], n_tok=st["rows"], path_stride=st["path"].shape[1])
    flh.kv_compact(st["caches"], st["p"], _stream(flh))
    return {"k": st["kc"], "v": st["vc"]}


def _own_pages(st):
    flh, c = _lib(), st["c"]
    if "fork" not in st:
        st["caches"] = _all_layers(flh, st)
        both = dict(kv_len=st["kv_len"].data_ptr(), table=st["table"].data_ptr(), free_pages=st["free"].data_ptr(),
                    taken=st["taken"].data_ptr(), shared=st["shared"].data_ptr(), n_seq=st["n_seq"], n_pages=st["n_pages"],
                    page_size=c["page"], n_free=st["free"].shape[0], table_stride=st["table"].shape[1])
        lists = lambda t: dict(copy_src=t[0].data_ptr(), copy_dst=t[1].data_ptr(), copy_n=t[2].data_ptr())   # noqa: E731
        st["fork"] = flh.KvForkP(src=st["src"].data_ptr(), dst=st["dst"].data_ptr(), n_fork=st["src"].shape[0],
                                 info=st["info"][0].data_ptr(), **both, **lists(st["copies"]))
        st["trim"] = flh.KvTrimP(keep=st["keep"].data_ptr(), held=st["kv_len"].data_ptr(), info=st["info"][1].data_ptr(),
                                 **both, **lists(st["last"]))
    s = _stream(flh)
    flh.kv_fork(st["fork"], s)
    flh.kv_copy(st["caches"], *[t.data_ptr() for t in st["copies"]], st["copies"].shape[1], s)
    flh.kv_trim(st["trim"], s)
    flh.kv_copy(st["caches"], *[t.data_ptr() for t in st["last"]], st["last"].shape[1], s)
    return {k: st[v] for k, v in PAGES.items()}


def run(state):
    op = state["c"]["op"]
    if own:
        return {"plan": _own_plan, "attn": _own_attn, "verify": _own_verify, "compact": _own_compact, "pages": _own_pages}[op](state)
    return {"plan": _tree, "attn": _plain_attn, "verify": _plain_verify, "compact": _plain_compact, "pages": _plain_pages}[op](state)


# ------------------------------------------------------------------- work --
def work(case):
    c = case
    if c["op"] == "plan":
        n = _counts(c)
        return {"bytes": 4 * sum(n) * (3 + _up(max(n), 32)) + 8 * len(n), "flops": 0}
    if c["op"] == "verify":
        n = _counts(c)
        inner = [0 if a == 0 else _up(a - 1, c["kids"]) for a in n]      # rows with children
        el = BYTES[c["dtype"]] * c["vocab"]
        return {"bytes": el * (sum(n) + (sum(inner) if c["draft"] else 0)) + 20 * sum(n) + 24 * len(n),
                "flops": 3 * c["vocab"] * (sum(n) + (sum(inner) if c["draft"] else 0))}
    if c["op"] == "compact":
        moved = sum(sum(a != i for i, a in enumerate(p)) for p in _paths(c))
        return {"bytes": moved * c["layers"] * c["kv_heads"] * c["d"] * 2 * 2 * 2 + 4 * sum(_counts(c)), "flops": 0}
    if c["op"] == "pages":
        lens, page = _page_lens(c), c["page"]
        copied = c["fork"] * sum(x % page for x in lens)
        entries = c["fork"] * sum(_up(x, page) for x in lens)            # copied, counted, taken off and cleared again
        return {"bytes": copied * c["layers"] * c["kv_heads"] * c["d"] * 2 * 2 * 2 + entries * 4 * 7, "flops": 0}
    pairs = keys = 0
    w = c["window"]
    for n, k in zip(*_attn_lens(c)):
        old = min(k - n, w) if w else k - n
        pairs, keys = pairs + n * (old + min(n, 8)), keys + old + n      # (an ancestor line is about eight long)
    rows = sum(_counts(c))
    return {"bytes": rows * c["heads"] * (c["dk"] + c["dv"]) * BYTES[c["act"]]
            + keys * c["kv_heads"] * (c["dk"] + c["dv"]) * BYTES[c["cache"]],
            "flops": 2 * pairs * c["heads"] * (c["dk"] + c["dv"])}


# ------------------------------------------------------------------ exact --
def _exact_attn(c, st):
    n, kl = _attn_lens(c)
    g, r0 = c["heads"] // c["kv_heads"], 0
    out = torch.zeros(st["rows"], c["heads"], c["dv"], dtype=torch.float64, device=DEV)
    parent = st["parent"].tolist()
    for s, (ql, k_len) in enumerate(zip(n, kl)):
        pages = st["table"][s, : _up(k_len, c["page"])].long()
        k, v = [_by_token(c, t[pages]).flatten(0, 1)[:k_len] for t in (st["kc"], st["vc"])]
        old = k_len - ql
        hide = torch.ones(ql, k_len, dtype=torch.bool)
        for i in range(ql):
            line, a = [], i
            while a >= 0:                                                # up to the root
                line.append(a)
                a = parent[r0 + a]
            if c["window"]:
                hide[i, max(0, old + len(line) - c["window"]): old] = False
                line = line[: c["window"]]
            else:
                hide[i, :old] = False
            hide[i, [old + a for a in line]] = False
        hide = hide.to(DEV)
        for h in range(c["kv_heads"]):
            q = st["q"][r0: r0 + ql, h * g: (h + 1) * g].double()
            w = torch.einsum("rgd,kd->rgk", q, k[:, h].double()) / math.sqrt(c["dk"])
            w = torch.softmax(w.masked_fill(hide[:, None], -math.inf), -1)
            out[r0: r0 + ql, h * g: (h + 1) * g] = torch.einsum("rgk,kd->rgd", w, v[:, h].double())
        r0 += ql
    return {"out": out}


def _exact_verify(c, st):
    start, parent, token = st["start"].tolist(), st["parent"].tolist(), st["token"].tolist()
    u, un, inv = st["u_accept"].double().tolist(), st["u_next"].double().tolist(), st["inv_temp"].tolist()
    logp = torch.zeros(c["seqs"], st["max_path"], dtype=torch.float64, device=DEV)

    def soft(x, it):
        x = x.double()
        if math.isinf(it):
            return torch.zeros_like(x).index_fill_(0, (x == x.max()).nonzero()[0], 1.0)
        return torch.softmax(x * it, 0)
    for s in range(c["seqs"]):
        r0, n, at, j = start[s], start[s + 1] - start[s], 0, 0
        while True:
            p = soft(st["target"][r0 + at], inv[s])
            q = soft(st["draft"][r0 + at], inv[s]) if c["draft"] else None
            if c["draft"] and math.isinf(inv[s]):
                q.zero_()
            left, took = p, None
            for i in range(at + 1, n):
                if parent[r0 + i] != at:
                    continue
                x = token[r0 + i]
                if c["draft"]:
                    if u[r0 + i] * float(q[x]) < float(left[x]):
                        took = i
                        break
                    left = (left - q).clamp(min=0)
                else:
                    if u[r0 + i] < float(left[x]):
                        took = i
                        break
                    left = left.clone()
                    left[x] = 0.0
                total = left.sum()
                left = left / total if float(total) > 0 else p
            if took is None:
                break
            logp[s, j] = p[token[r0 + took]].log()
            at, j = took, j + 1
        cum = left.cumsum(0)
        logp[s, j] = p[int(torch.searchsorted(cum, un[s] * cum[-1], right=True).clamp(max=c["vocab"] - 1))].log()
    return {"n_path": None, "path": None, "next": None, "logp": logp, "len": None}


def exact(case, seed):
    if case["op"] not in ("attn", "verify"):
        return None                                                      # whole numbers, and values that are moved
    st = prepare(case, seed)
    return _exact_attn(case, st) if case["op"] == "attn" else _exact_verify(case, st)
