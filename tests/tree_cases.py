"""Oracles of drafted trees, their verification and the pages between steps: plain
sequential code in 64 bits, from the definitions."""
import math

import numpy as np
import torch

NONE = 0xFFFFFFFF


def random_parents(n, rng, back=4):
    """A tree as drafts grow: each row hangs on one of the few before it."""
    return np.array([-1] + [int(rng.integers(max(0, i - back), i)) for i in range(1, n)], np.int32)[:n]


def lines(parent):
    """The rows of each row's line, itself first, up to its root."""
    out = []
    for r in range(len(parent)):
        line, x = [r], r
        while 0 <= parent[x] < x:
            x = int(parent[x])
            line.append(x)
        out.append(line)
    return out


def plan_oracle(parents, kv_len, stride, window):
    """mask, depth, pos of the requests' rows, one after the other."""
    mask, depth, pos = [], [], []
    for parent, kv in zip(parents, kv_len):
        for line in lines(parent):
            words = np.zeros(stride, np.uint64)
            for d, x in enumerate(line):
                if x < 32 * stride and (window == 0 or d < window):
                    words[x // 32] |= np.uint64(1 << (x % 32))
            mask.append(words.astype(np.uint32))
            depth.append(len(line) - 1)
            pos.append(int(kv) - len(parent) + len(line) - 1)
    return (np.array(mask, np.uint32).reshape(-1, stride), np.array(depth, np.uint32), np.array(pos, np.int32))


def tree_attn_oracle(q, rows, kv_len, table, cache, group, scale, window, mask, depth, cut=None):
    """As paged_cases.attn_oracle, for trees: row i of n sees the keys in front of the tree (by
    its depth in the window) and those that its bits name.  cut: rows that the requests have beside those in `rows`."""
    H, dv, page = q.shape[1], cache.dv, cache.page
    out = torch.zeros(q.shape[0], H, dv, dtype=torch.float64)
    mag, amp = torch.zeros_like(out), torch.zeros(q.shape[0], H, dtype=torch.float64)
    kall, vall = cache.view
    for s, (r0, r1) in enumerate(rows):
        n = r1 - r0
        if n <= 0:
            continue
        kv = int(kv_len[s])
        j = np.arange(min(kv, table.shape[1] * page))
        pg = table[s][j // page] if len(j) else np.zeros(0, np.uint32)
        ok = pg < cache.n_pages
        j, pg = j[ok], pg[ok].astype(np.int64)
        k = kall[torch.from_numpy(pg), torch.from_numpy(j % page)].double()
        v = vall[torch.from_numpy(pg), torch.from_numpy(j % page)].double()
        old = kv - n - (cut[s] if cut is not None else 0)
        see = np.zeros((n, len(j)), bool)
        for i in range(n):
            d = min(int(depth[r0 + i]), n - 1)
            see[i] = (j < old) & ((j > old + d - window) if window else True)
            b = j - old
            t = (b >= 0) & (b < 32 * mask.shape[1])
            see[i][t] = (mask[r0 + i][b[t] // 32] >> (b[t] % 32).astype(np.uint32)) & 1
        see = torch.from_numpy(see)
        for h in range(H):
            qh, kh, vh = q[r0:r1, h].double(), k[:, h // group], v[:, h // group]
            t = ((qh @ kh.T) * scale).masked_fill(~see, -math.inf)
            t = torch.where(see, t, -math.inf)
            top = t.max(1, keepdim=True).values if t.shape[1] else torch.full((n, 1), -math.inf, dtype=torch.float64)
            e = torch.exp(t - torch.where(torch.isinf(top), torch.zeros_like(top), top)).masked_fill(~see, 0.0)
            l = e.sum(1, keepdim=True)
            w = torch.where(l == 0, torch.zeros_like(e), e / l)
            for i in range(n):                                # (keys not seen have no part in a row, whatever they are)
                out[r0 + i, h] = w[i][see[i]] @ vh[see[i]]
                mag[r0 + i, h] = w[i][see[i]] @ vh[see[i]].abs()
                a = (qh[i].abs() * kh[see[i]].abs()).sum(1) * scale
                amp[r0 + i, h] = a.max() if len(a) else 0.0
    return out, mag, amp


# ------------------------------------------------------------------ verify --
def clean(x):
    """Logits in 64 bits: what is no number is -infinity, infinity the largest float."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    return np.minimum(x, float(np.finfo(np.float32).max))


def soft(x, it):
    """softmax(it x); 1 at the first of the largest for an infinite it; all zeros where nothing is allowed."""
    x = clean(x)
    top = x.max()
    if top == -np.inf:
        return np.zeros_like(x)
    if math.isinf(it):
        return (np.arange(len(x)) == np.argmax(x)).astype(np.float64)
    with np.errstate(invalid="ignore"):
        e = np.where(x == -np.inf, 0.0, np.exp((x - top) * it))
    return e / e.sum()


def verify_oracle(target, draft, starts, token, parent, inv_temp, u_accept, u_next, path_stride, max_child, vocab):
    """(n_path, path, next, logp) of the definition: p is renormalised after each child that does not stand.
    Also how near the nearest decision was to its border (relative to 1)."""
    n_seq = len(starts) - 1
    path = np.full((n_seq, path_stride), NONE, np.uint32)
    logp = np.zeros((n_seq, path_stride))
    n_path, nxt, near = np.zeros(n_seq, np.uint32), np.full(n_seq, NONE, np.uint32), 1.0
    for s in range(n_seq):
        r0, n = int(starts[s]), min(256, int(starts[s + 1]) - int(starts[s]))
        if n <= 0:
            continue
        it = 1.0 if inv_temp is None else float(inv_temp[s])
        it = it if it >= 0 else 0.0
        par = [-1] + [(i - 1 if parent is None else int(parent[r0 + i])) for i in range(1, n)]
        at, j = 0, 0
        while True:
            path[s, j] = at
            p = soft(target[r0 + at], it)
            kids = [i for i in range(at + 1, n) if par[i] == at][:max_child]
            left, took = p, None
            for i in kids:
                x = int(token[r0 + i])
                inside = x < vocab
                if math.isinf(it):
                    ok = inside and p[x] > 0
                else:
                    q = soft(draft[r0 + at], it) if draft is not None else None
                    qx = (q[x] if q is not None else 1.0) if inside else 0.0
                    px = left[x] if inside else 0.0
                    ok = float(u_accept[r0 + i]) * qx < px
                    near = min(near, abs(float(u_accept[r0 + i]) * qx - px) / max(qx, 1e-300) if inside and qx > 0 else 1.0)
                if ok:
                    took = i
                    break
                if not math.isinf(it):
                    left = np.maximum(left - q, 0.0) if q is not None else np.where(np.arange(vocab) == x, 0.0, left)
                    total = left.sum()
                    if total > 0:
                        left = left / total
                    else:
                        left = np.zeros_like(left)
            if took is not None and j + 1 < path_stride:
                logp[s, j] = math.log(p[int(token[r0 + took])])
                at, j = took, j + 1
                continue
            if took is not None or left.sum() <= 0:
                left = p
            n_path[s] = j + 1
            if p.sum() > 0:
                cum = np.cumsum(left)
                want = float(u_next[s]) * cum[-1]
                nxt[s] = int(np.argmax(cum > want)) if (cum > want).any() else int(np.nonzero(left)[0][-1])
                live = cum[left > 0]
                near = min(near, float(np.abs(live[:-1] - want).min()) if len(live) > 1 else 1.0)
                logp[s, j] = math.log(p[nxt[s]])
            break
    return n_path, path, nxt, logp, near
