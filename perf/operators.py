"""Decoder attention over a paged key/value cache, as cases to time.

Three operators, in the order in which a decoder step calls them:

  plan    block tables and slot maps from request lengths: pages are taken off
          a free list for the tokens that each request adds, and every token
          gets its cache slot and its position.
  rope    rotary positions (one axis, or time / height / width) on the queries
          and keys of the new tokens, keys and values written to their slots.
  attn    attention of the new tokens over the cache: one token a sequence, a
          few (speculative verify), a chunk of a prompt, or not causal at all
          (an encoder's states as the cache).

Shapes: activations are rows of a fused query/key/value product, so queries,
keys and values are strided views; the cache's pages lie in any order, stored
head by head inside a page or token by token.  Request lengths belong to the
case ("lens" seeds them); every value comes from the seed.
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
        # one decode step of a serving batch: a token each, a page now and then
        {"name": "plan_decode", "op": "plan", "seqs": 64, "held": 8192, "add_lo": 1, "add_hi": 1, "page": 16, "lens": 1},
        # a step that mixes prompt chunks of every length with requests that add nothing
        {"name": "plan_ragged", "op": "plan", "seqs": 500, "held": 3001, "add_lo": 0, "add_hi": 257, "page": 64, "lens": 2},
        # the latency case: one token of the benchmark's decoder layer
        {"name": "rope_token", "op": "rope", "act": "f32", "cache": "f16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "n_rot": 128, "first": 0, "style": "pairs", "axes": 1, "tokens": 1, "page": 16, "order": "head", "far": 8192},
        # a prompt with images: three position axes, 16-bit activations
        {"name": "rope_image", "op": "rope", "act": "bf16", "cache": "bf16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "n_rot": 128, "first": 0, "style": "halves", "axes": 3, "tokens": 4999, "page": 64, "order": "token", "far": 4096},
        # the rotated part of a head behind an unrotated one, far positions
        {"name": "rope_tail", "op": "rope", "act": "f32", "cache": "f16", "heads": 16, "kv_heads": 16, "dk": 192, "dv": 128,
         "n_rot": 64, "first": 128, "style": "pairs", "axes": 1, "tokens": 1000, "page": 16, "order": "head", "far": 1 << 20},
        # one token of one request
        {"name": "attn_token", "op": "attn", "act": "f32", "cache": "f16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 16, "order": "head", "seqs": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 4001, "kv_hi": 4001, "causal": True,
         "window": 0, "lens": 3},
        # one token of each request of a serving batch, contexts of every length
        {"name": "attn_batch", "op": "attn", "act": "f32", "cache": "f16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 16, "order": "head", "seqs": 64, "q_lo": 1, "q_hi": 1, "kv_lo": 1, "kv_hi": 8192, "causal": True,
         "window": 0, "lens": 4},
        # a few requests over very long contexts
        {"name": "attn_long", "op": "attn", "act": "bf16", "cache": "bf16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 64, "order": "head", "seqs": 4, "q_lo": 1, "q_hi": 1, "kv_lo": 131072, "kv_hi": 131072, "causal": True,
         "window": 0, "lens": 5},
        # a speculative verify step with a sliding window, pages token by token
        {"name": "attn_verify", "op": "attn", "act": "f32", "cache": "bf16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 32, "order": "token", "seqs": 16, "q_lo": 1, "q_hi": 8, "kv_lo": 100, "kv_hi": 10000, "causal": True,
         "window": 4096, "lens": 6},
        # a whole prompt
        {"name": "attn_prompt", "op": "attn", "act": "bf16", "cache": "bf16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 64, "order": "head", "seqs": 1, "q_lo": 8192, "q_hi": 8192, "kv_lo": 8192, "kv_hi": 8192, "causal": True,
         "window": 0, "lens": 7},
        # prompt chunks behind cached contexts, ragged, in the fp32 of the quantized products
        {"name": "attn_chunk", "op": "attn", "act": "f32", "cache": "f16", "heads": 32, "kv_heads": 8, "dk": 128, "dv": 128,
         "page": 16, "order": "head", "seqs": 5, "q_lo": 1, "q_hi": 1000, "kv_lo": 1000, "kv_hi": 8000, "causal": True,
         "window": 0, "lens": 8},
        # cross attention: a decoder's tokens over an encoder's states of another length
        {"name": "attn_cross", "op": "attn", "act": "f16", "cache": "f16", "heads": 20, "kv_heads": 20, "dk": 64, "dv": 64,
         "page": 128, "order": "token", "seqs": 8, "q_lo": 5, "q_hi": 448, "kv_lo": 1500, "kv_hi": 1500, "causal": False,
         "window": 0, "lens": 9},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["plan", "rope", "rope", "attn", "attn", "attn", "attn", "attn"])
    lens = rng.randrange(1 << 30)
    if op == "plan":
        seqs = _log_int(rng, 1, 1500)
        hi = rng.choice([1, rng.randint(2, 16), _log_int(rng, 16, max(17, 120000 // seqs))])
        return {"op": "plan", "seqs": seqs, "held": _log_int(rng, 16, 16384), "add_lo": rng.randint(0, 1), "add_hi": hi,
                "page": rng.choice([16, 32, 64, 128, 256]), "lens": lens}
    act, cache = rng.choice([("f32", "f16"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 7, 8] if kv_heads <= 8 else [1, 2])
    dk, dv = rng.choice([(128, 128), (128, 128), (128, 128), (64, 64), (80, 80), (96, 96), (192, 128), (256, 256)])
    c = {"op": op, "act": act, "cache": cache, "heads": heads, "kv_heads": kv_heads, "dk": dk, "dv": dv,
         "page": rng.choice([16, 16, 32, 64, 128]), "order": rng.choice(["head", "token"])}
    if op == "rope":
        n_rot = rng.choice([dk, dk, dk // 2])
        c.update(n_rot=n_rot, first=rng.choice([0, dk - n_rot]), style=rng.choice(["halves", "pairs"]),
                 axes=rng.choice([1, 1, 3]), tokens=_log_int(rng, 1, 8192), far=_log_int(rng, 1024, 1 << 20))
        return c
    seqs = _log_int(rng, 1, 128)
    kind = rng.choice(["one", "one", "few", "chunk", "chunk"])
    q_hi = 1 if kind == "one" else rng.randint(2, 16) if kind == "few" else 0
    if kind == "chunk":
        seqs = _log_int(rng, 1, 16)
        kv_hi = _log_int(rng, 64, 32768 // seqs)
        q_hi = _log_int(rng, 17, max(18, min(kv_hi, 4096, int(2.6e11 / (dk + dv) / (seqs * heads * kv_hi)))))
    else:
        kv_hi = _log_int(rng, 32, min(131072, 10 ** 9 // (seqs * kv_heads * (dk + dv))))
    c.update(seqs=seqs, q_lo=rng.choice([1, q_hi]), q_hi=q_hi, kv_lo=rng.choice([1, (kv_hi + 1) // 2, kv_hi]), kv_hi=kv_hi,
             causal=rng.random() < 0.85, window=0, lens=lens)
    if c["causal"] and rng.random() < 0.25:
        c["window"] = _log_int(rng, 16, 8192)
    return c


# ----------------------------------------------------------------- inputs --
def _gen(seed, k):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + k) % (1 << 62))
    return g


def _randn(seed, k, shape, dtype=torch.float32):
    return torch.randn(shape, generator=_gen(seed, k), device=DEV, dtype=dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _lens(c):
    """(rows, keys) of each sequence; the first has the most of both."""
    r = random.Random(c["lens"])
    q = [c["q_hi"]] + [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["seqs"] - 1)]
    kv = [c["kv_hi"]] + [r.randint(c["kv_lo"], c["kv_hi"]) for _ in range(c["seqs"] - 1)]
    if c["causal"]:                                 # a chunk's own keys are in the cache
        q = [min(a, b) for a, b in zip(q, kv)]
    return q, kv


def _plan_lens(c):
    r = random.Random(c["lens"])
    held = [r.randint(0, c["held"]) for _ in range(c["seqs"])]
    add = [r.randint(c["add_lo"], c["add_hi"]) for _ in range(c["seqs"])]
    return held, add


def _up(a, b):
    return -(-a // b)


def _prepare_plan(c, seed):
    held, add = _plan_lens(c)
    page, n = c["page"], c["seqs"]
    stride = _up(c["held"] + c["add_hi"], page) + 1
    pages = [_up(h, page) for h in held]
    need = sum(_up(h + a, page) - p for h, a, p in zip(held, add, pages))
    total = sum(pages) + need + 17
    perm = torch.randperm(total, generator=_gen(seed, 0), device=DEV).to(torch.int32)
    table = torch.full((n, stride), -1, dtype=torch.int32, device=DEV)
    at = torch.arange(stride, device=DEV)[None, :] < _ints(pages)[:, None]
    table[at] = perm[: sum(pages)]
    cap = sum(add) + 3                              # rows behind the last token have no slot
    return {"c": c, "held": _ints(held), "add": _ints(add), "free": perm[sum(pages):].contiguous(), "table": table,
            "taken_in": _ints([5]), "taken": _ints([0]), "q_start": _ints([0] * (n + 1)), "kv_len": _ints([0] * n),
            "slot": torch.full((cap,), -7, dtype=torch.int32, device=DEV),
            "pos": torch.full((cap,), -7, dtype=torch.int32, device=DEV), "info": _ints([0, 0])}


def _cache(c, n_pages, tensors):
    """The pages in the order that the case stores them in, from [page][token][head][d]."""
    return [(t.permute(0, 2, 1, 3) if c["order"] == "head" else t).contiguous() for t in tensors]


def _fused(c, seed, n):
    """Queries, keys and values of n tokens: views of the rows of one product."""
    h, hk, dk, dv = c["heads"], c["kv_heads"], c["dk"], c["dv"]
    x = _randn(seed, 1, (max(n, 1), h * dk + hk * dk + hk * dv))
    x.mul_(torch.where(torch.rand(x.shape[1], generator=_gen(seed, 2), device=DEV) < 0.02, 4.0, 1.0))
    x = x.to(DT[c["act"]])
    q, k, v = x.split([h * dk, hk * dk, hk * dv], 1)
    return x, q.unflatten(1, (h, dk)), k.unflatten(1, (hk, dk)), v.unflatten(1, (hk, dv))


def _axis(c):
    """The position axis of every rotated pair: a quarter turns with time, the
    rest is height's and width's, one after the other."""
    p = c["n_rot"] // 2
    if c["axes"] == 1:
        return [0] * p
    t = p // 4
    return [0] * t + [1] * ((p - t) // 2) + [2] * (p - t - (p - t) // 2)


ROPE_BASE = 500000.0


def _prepare_rope(c, seed):
    n, page = c["tokens"], c["page"]
    x, q, k, v = _fused(c, seed, n)
    n_pages = _up(n + n // 8 + 8, page)
    slot = torch.randperm(n_pages * page, generator=_gen(seed, 3), device=DEV)[:n].to(torch.int32)
    if n > 16:
        slot[torch.randint(0, n, (n // 16,), generator=_gen(seed, 4), device=DEV)] = -1   # tokens that found no page
    pos = torch.randint(0, c["far"], (c["axes"], n), generator=_gen(seed, 5), device=DEV).to(torch.int32)
    kc, vc = _cache(c, n_pages, [torch.zeros(n_pages, page, c["kv_heads"], d, device=DEV, dtype=DT[c["cache"]])
                                 for d in (c["dk"], c["dv"])])
    return {"c": c, "x": x, "q": q, "k": k, "v": v, "slot": slot, "pos": pos, "kc": kc, "vc": vc, "n_pages": n_pages,
            "axis": _axis(c), "q_out": torch.zeros(n, c["heads"], c["dk"], device=DEV, dtype=DT[c["act"]])}


def _prepare_attn(c, seed):
    ql, kl = _lens(c)
    page, hk, n = c["page"], c["kv_heads"], c["seqs"]
    stride = _up(max(kl), page) + 1
    pages = [_up(k, page) for k in kl]
    n_pages = sum(pages) + 3
    perm = torch.randperm(n_pages, generator=_gen(seed, 0), device=DEV).to(torch.int32)
    table = torch.full((n, stride), -1, dtype=torch.int32, device=DEV)
    at = torch.arange(stride, device=DEV)[None, :] < _ints(pages)[:, None]
    table[at] = perm[: sum(pages)]
    rows = sum(ql)
    x, q, _, _ = _fused(c, seed, rows + 2)
    kv = [_randn(seed, 10 + i, (n_pages, page, hk, d), DT[c["cache"]]) for i, d in enumerate((c["dk"], c["dv"]))]
    kv[0].mul_(torch.where(torch.rand(c["dk"], generator=_gen(seed, 12), device=DEV) < 0.03, 3.0, 1.0).to(kv[0].dtype))
    # what no request has written yet is no number
    used = torch.zeros(n_pages, page, dtype=torch.bool, device=DEV)
    j = torch.arange(stride * page, device=DEV)
    inside = (j[None, :] < _ints(kl)[:, None]).view(n, stride, page)
    used[table[at].long()] = inside[at]
    for t in kv:
        t.masked_fill_(~used[:, :, None, None], float("nan"))
    kc, vc = _cache(c, n_pages, kv)
    start = [0]
    for a in ql:
        start.append(start[-1] + a)
    return {"c": c, "x": x, "q": q, "kc": kc, "vc": vc, "n_pages": n_pages, "table": table, "q_start": _ints(start),
            "kv_len": _ints(kl), "max_q": max(ql), "max_kv": max(kl), "rows": rows,
            "out": torch.zeros(rows + 2, c["heads"], c["dv"], device=DEV, dtype=DT[c["act"]])}


def prepare(case, seed):
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attn": _prepare_attn}[case["op"]](case, seed)


# ------------------------------------------------------------ plain forms --
def _plain_plan(st):
    c, page = st["c"], st["c"]["page"]
    held, add, free, table = st["held"].long(), st["add"].long(), st["free"], st["table"]
    cap, width, n_free = st["slot"].shape[0], table.shape[1], free.shape[0]
    end = add.cumsum(0).clamp(max=cap)
    start = torch.cat([end.new_zeros(1), end])
    kv = held + end - start[:-1]
    before, after = ((held + page - 1) // page).clamp(max=width), ((kv + page - 1) // page).clamp(max=width)
    need = after - before
    first = st["taken_in"].long() + need.cumsum(0) - need
    j = torch.arange(width, device=DEV)[None, :]
    at = first[:, None] + j - before[:, None]
    fresh = torch.where(at < n_free, free[at.clamp(0, n_free - 1)], -1)
    table = torch.where((j >= before[:, None]) & (j < after[:, None]), fresh, table)
    t = torch.arange(cap, device=DEV)
    s = torch.searchsorted(end, t, right=True).clamp(max=held.shape[0] - 1)
    p = held[s] + t - start[s]
    pg = torch.where(p // page < width, table[s, (p // page).clamp(max=width - 1)], -1)
    slot = torch.where(pg >= 0, pg * page + p % page, -1).int()
    live = t < end[-1]
    lost = add.sum() - ((slot >= 0) & live).sum()
    return {"table": table, "q_start": start.int(), "kv_len": kv.int(), "slot": torch.where(live, slot, -1),
            "pos": torch.where(live, p, 0).int(), "taken": (st["taken_in"] + need.sum()).int(),
            "info": torch.stack([end[-1], lost]).int()}


def _turn(c, x, pos, axis):
    """x [token][head][d] with its pairs rotated; angles in 64 bits, the rest in 32."""
    p = c["n_rot"] // 2
    freq = ROPE_BASE ** (-torch.arange(p, device=DEV, dtype=torch.float64) / p)
    ang = pos.double()[torch.tensor(axis, device=DEV)].t() * freq          # [token][pair]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    y = x.float().clone()
    part = y[..., c["first"]: c["first"] + c["n_rot"]]
    pair = part.unflatten(-1, (2, p)) if c["style"] == "halves" else part.unflatten(-1, (p, 2)).transpose(-1, -2)
    a, b = pair[..., 0, :].clone(), pair[..., 1, :].clone()
    pair[..., 0, :] = a * cos - b * sin
    pair[..., 1, :] = a * sin + b * cos
    return y


def _plain_rope(st):
    c = st["c"]
    q = _turn(c, st["q"], st["pos"], st["axis"]).to(DT[c["act"]])
    k = _turn(c, st["k"], st["pos"], st["axis"])
    live = st["slot"] >= 0
    slot = st["slot"][live].long()
    for cache, new in ((st["kc"], k), (st["vc"], st["v"])):
        by_token = cache.transpose(1, 2) if c["order"] == "head" else cache
        by_token[slot // c["page"], slot % c["page"]] = new[live].to(cache.dtype)
    return {"q": q, "k": st["kc"], "v": st["vc"]}


def _plain_attn(st):
    c = st["c"]
    hk, g, page = c["kv_heads"], c["heads"] // c["kv_heads"], c["page"]
    start, kl = st["q_start"].long(), st["kv_len"].long()
    n, mq, mk = kl.shape[0], st["max_q"], st["max_kv"]
    j = torch.arange(mk, device=DEV)
    there = j[None, :] < kl[:, None]
    pg = st["table"][:, j // page].long().clamp(min=0)
    by_token = [t.transpose(1, 2) if c["order"] == "head" else t for t in (st["kc"], st["vc"])]
    k, v = [t[pg, j % page].float().masked_fill_(~there[:, :, None, None], 0.0).transpose(1, 2) for t in by_token]
    i = torch.arange(mq, device=DEV)
    ql = start[1:] - start[:-1]
    real = i[None, :] < ql[:, None]
    at = (start[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][at].float()                                               # [seq][row][head][d]
    q = q.unflatten(2, (hk, g)).permute(0, 2, 3, 1, 4).flatten(2, 3)      # [seq][kv head][g * row][d]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (c["dk"] ** -0.5)
    pos = (kl - ql)[:, None] + i                                          # [seq][row]
    see = there[:, None, :].expand(n, mq, mk)
    if c["causal"]:
        see = see & (j[None, None, :] <= pos[:, :, None])
        if c["window"]:
            see = see & (j[None, None, :] > pos[:, :, None] - c["window"])
    s = s.unflatten(2, (g, mq)).masked_fill_(~see[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(top > float("-inf"), top, 0.0)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.flatten(2, 3), v).unflatten(2, (g, mq))
    o = torch.where(total > 0, o / total, 0.0)
    out = st["out"].clone()
    out[at[real]] = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[real].to(out.dtype)
    return {"out": out}


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


def _kv(flh, c, st):
    """The cache as the library sees it: element strides of a page, a token, a head."""
    page, hk = c["page"], c["kv_heads"]

    def strides(d):
        return (page * hk * d, d, page * d) if c["order"] == "head" else (page * hk * d, hk * d, d)
    return flh.KvCache(st["kc"].data_ptr(), st["vc"].data_ptr(), flh.Dtype[c["cache"].upper()], st["n_pages"], page, hk,
                       c["dk"], c["dv"], strides(c["dk"]), strides(c["dv"]))


def _own_plan(st):
    flh = _lib()
    if "p" not in st:
        st["p"] = flh.KvPlanP(
            held=st["held"].data_ptr(), add=st["add"].data_ptr(), free_pages=st["free"].data_ptr(),
            taken_in=st["taken_in"].data_ptr(), taken=st["taken"].data_ptr(), table=st["table"].data_ptr(),
            q_start=st["q_start"].data_ptr(), kv_len=st["kv_len"].data_ptr(), slot=st["slot"].data_ptr(),
            pos=st["pos"].data_ptr(), info=st["info"].data_ptr(), n_seq=st["c"]["seqs"], page_size=st["c"]["page"],
            n_free=st["free"].shape[0], table_stride=st["table"].shape[1], max_tok=st["slot"].shape[0])
    flh.kv_plan(st["p"], _stream(flh))
    return {k: st[k] for k in ("table", "q_start", "kv_len", "slot", "pos", "taken", "info")}


def _own_rope(st):
    flh, c = _lib(), st["c"]
    if "p" not in st:
        st["cache"] = _kv(flh, c, st)
        st["rope"] = flh.RopeTable(c["n_rot"], base=ROPE_BASE, axis=st["axis"], n_axis=c["axes"], first=c["first"],
                                   layout=flh.RopeLayout.HALVES if c["style"] == "halves" else flh.RopeLayout.PAIRS)
        q, k, v, o = st["q"], st["k"], st["v"], st["q_out"]
        st["p"] = flh.RopeKvP(
            q=q.data_ptr(), q_out=o.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), pos=st["pos"].data_ptr(),
            slot=st["slot"].data_ptr(), q_tok=q.stride(0), q_head=q.stride(1), qo_tok=o.stride(0), qo_head=o.stride(1),
            k_tok=k.stride(0), k_head=k.stride(1), v_tok=v.stride(0), v_head=v.stride(1),
            dtype=flh.Dtype[c["act"].upper()], n_tok=c["tokens"], n_head=c["heads"], pos_stride=c["tokens"])
    flh.rope_kv_append(st["rope"], st["cache"], st["p"], _stream(flh))
    return {"q": st["q_out"], "k": st["kc"], "v": st["vc"]}


def _own_attn(st):
    flh, c = _lib(), st["c"]
    if "p" not in st:
        st["cache"] = _kv(flh, c, st)
        q, o = st["q"], st["out"]
        p = flh.AttnP(
            q=q.data_ptr(), out=o.data_ptr(), q_start=st["q_start"].data_ptr(), kv_len=st["kv_len"].data_ptr(),
            table=st["table"].data_ptr(), q_tok=q.stride(0), q_head=q.stride(1), o_tok=o.stride(0), o_head=o.stride(1),
            dtype=flh.Dtype[c["act"].upper()], n_head=c["heads"], n_seq=c["seqs"], n_tok=st["rows"], max_q=st["max_q"],
            table_stride=st["table"].shape[1], scale=c["dk"] ** -0.5, causal=int(c["causal"]), window=c["window"])
        p.ws_bytes = flh.paged_attn_ws_bytes(st["cache"], p)
        st["ws"] = torch.empty(max(p.ws_bytes, 1), dtype=torch.uint8, device=DEV)
        p.ws = st["ws"].data_ptr()
        st["p"] = p
    flh.paged_attn(st["cache"], st["p"], _stream(flh))
    return {"out": st["out"]}


def run(state):
    op = state["c"]["op"]
    if own:
        return {"plan": _own_plan, "rope": _own_rope, "attn": _own_attn}[op](state)
    return {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn}[op](state)


# ------------------------------------------------------------------- work --
def _seen(c):
    """(query, key) pairs that are visible, and keys that some query sees, over the sequences."""
    pairs = keys = 0
    for q, k in zip(*_lens(c)):
        if not c["causal"]:
            pairs, keys = pairs + q * k, keys + k
            continue
        w = c["window"] or k
        lo, hi = k - q + 1, k                       # keys at or before the first and the last row
        full = max(0, min(q, hi - max(lo, w) + 1))  # rows that see a whole window
        part = q - full
        pairs += full * w + part * (2 * lo + part - 1) // 2
        keys += min(k, q - 1 + w)
    return pairs, keys


def work(case):
    c = case
    if c["op"] == "plan":
        held, add = _plan_lens(c)
        fresh = sum(_up(h + a, c["page"]) - _up(h, c["page"]) for h, a in zip(held, add))
        return {"bytes": 4 * (4 * c["seqs"] + 3 * sum(add) + 2 * fresh), "flops": 0}
    if c["op"] == "rope":
        row = c["heads"] * c["dk"] * 2 * BYTES[c["act"]] + c["kv_heads"] * (c["dk"] + c["dv"]) * (BYTES[c["act"]] + BYTES[c["cache"]])
        return {"bytes": c["tokens"] * (row + 4 * c["axes"] + 4), "flops": 3 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["n_rot"]}
    pairs, keys = _seen(c)
    rows = sum(_lens(c)[0])
    return {"bytes": rows * c["heads"] * (c["dk"] + c["dv"]) * BYTES[c["act"]]
            + keys * c["kv_heads"] * (c["dk"] + c["dv"]) * BYTES[c["cache"]],
            "flops": 2 * pairs * c["heads"] * (c["dk"] + c["dv"])}


# ------------------------------------------------------------------ exact --
def _exact_rope(c, st):
    n, p = c["tokens"], c["n_rot"] // 2
    i = torch.arange(p, device=DEV)
    ia, ib = (i, i + p) if c["style"] == "halves" else (2 * i, 2 * i + 1)
    where = torch.empty(p, n, dtype=torch.float64, device=DEV)
    for r in range(p):
        where[r] = st["pos"][st["axis"][r]].double() * math.exp(-math.log(ROPE_BASE) * r / p)
    z = torch.polar(torch.ones_like(where), where).t()[:, None, :]        # e^(i angle)

    def turned(x):
        y = x.double()
        w = torch.complex(y[..., c["first"] + ia], y[..., c["first"] + ib]) * z
        y[..., c["first"] + ia], y[..., c["first"] + ib] = w.real, w.imag
        return y
    out = {"q": turned(st["q"])}
    for name, cache, new in (("k", st["kc"], turned(st["k"])), ("v", st["vc"], st["v"].double())):
        flat = torch.zeros(st["n_pages"] * c["page"], new.shape[1], new.shape[2], dtype=torch.float64, device=DEV)
        keep = st["slot"] >= 0
        flat[st["slot"][keep].long()] = new[keep]
        flat = flat.unflatten(0, (st["n_pages"], c["page"]))
        out[name] = flat.permute(0, 2, 1, 3).contiguous() if c["order"] == "head" else flat
    return out


def _exact_attn(c, st):
    out = torch.zeros(st["rows"] + 2, c["heads"], c["dv"], dtype=torch.float64, device=DEV)
    g, r0 = c["heads"] // c["kv_heads"], 0
    for s, (ql, kl) in enumerate(zip(*_lens(c))):
        pages = st["table"][s, : _up(kl, c["page"])].long()
        k, v = st["kc"][pages], st["vc"][pages]
        if c["order"] == "head":
            k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
        k, v = k.flatten(0, 1)[:kl], v.flatten(0, 1)[:kl]
        col = torch.arange(kl, device=DEV)
        for h in range(c["kv_heads"]):
            kh, vh = k[:, h].double(), v[:, h].double()
            for b0 in range(0, ql, 2048):
                b1 = min(ql, b0 + 2048)
                q = st["q"][r0 + b0: r0 + b1, h * g: (h + 1) * g].double()
                w = torch.einsum("rgd,kd->rgk", q, kh) / math.sqrt(c["dk"])
                if c["causal"]:
                    last = (kl - ql + torch.arange(b0, b1, device=DEV))[:, None, None]
                    hide = col > last
                    if c["window"]:
                        hide = hide | (col <= last - c["window"])
                    w = w.masked_fill(hide, -math.inf)
                out[r0 + b0: r0 + b1, h * g: (h + 1) * g] = torch.einsum("rgk,kd->rgd", torch.softmax(w, -1), vh)
        r0 += ql
    return {"out": out}


def exact(case, seed):
    if case["op"] == "plan":
        return None
    st = prepare(case, seed)
    return _exact_rope(case, st) if case["op"] == "rope" else _exact_attn(case, st)
