"""Inputs and 64-bit oracles of the paged cache, rotary and attention tests."""
import math

import numpy as np
import torch

TORCH = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
NONE = 0xFFFFFFFF


def half_step(name):
    """Largest relative error of one rounding to the type."""
    return torch.finfo(TORCH[name]).eps / 2


def raw(t):
    """A torch tensor's bytes as a numpy array."""
    return t.contiguous().view(torch.uint8).numpy().reshape(-1) if t.numel() else np.zeros(0, np.uint8)


def put(flh, s, t):
    return flh.DeviceBuffer.from_array(raw(t) if isinstance(t, torch.Tensor) else t, s, extra=16)


def get(buf, like, s):
    """The device buffer's contents, with the shape and type of a torch tensor."""
    n = like.numel() * like.element_size()
    return torch.from_numpy(buf.download(np.uint8, n, s)).view(like.dtype).reshape(like.shape)


class Cache:
    """A paged cache on the host ([page][token][head][d] views of one storage
    order) and on the device; everything starts as NaN."""

    def __init__(self, flh, s, dtype, n_pages, page, heads, dk, dv, order="head", pad=0):
        self.flh, self.s, self.dtype, self.page, self.n_pages, self.heads, self.dk, self.dv = \
            flh, s, dtype, page, n_pages, heads, dk, dv
        self.store, self.view, strides = [], [], []
        for d in (dk, dv):
            w = d + pad                                       # pad: elements between rows (a multiple of 8)
            shape = (n_pages, heads, page, w) if order == "head" else (n_pages, page, heads, w)
            t = torch.full(shape, float("nan"), dtype=TORCH[dtype])
            v = t.transpose(1, 2) if order == "head" else t
            self.store.append(t)
            self.view.append(v[..., :d])
            st = v.stride()
            strides.append((st[0], st[1], st[2]))
        self.buf = [put(flh, s, t) for t in self.store]
        self.c = flh.KvCache(self.buf[0], self.buf[1], flh.Dtype[dtype], n_pages, page, heads, dk, dv, *strides)

    def push(self):
        for b, t in zip(self.buf, self.store):
            b.upload(raw(t), self.s)

    def pull(self):
        """The device's pages, as views like .view."""
        out = []
        for b, t, v in zip(self.buf, self.store, self.view):
            got = get(b, t, self.s)
            out.append(torch.as_strided(got, v.shape, v.stride()))
        return out


def attn_oracle(q, rows, kv_len, table, cache, group, scale, causal, window):
    """q [row][head][d]; rows: (first, end) per request.  Returns out and, per
    element, sum_j p_j |v_j| and per (row, head) the largest sum_i |q_i k_ji|
    scale over the visible keys (what rounding errors scale with); all float64."""
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
        k = kall[torch.from_numpy(pg), torch.from_numpy(j % page)].double()          # [key][kv head][d]
        v = vall[torch.from_numpy(pg), torch.from_numpy(j % page)].double()
        p = kv - n + np.arange(n)
        see = np.ones((n, len(j)), bool)
        if causal:
            see = j[None, :] <= p[:, None]
            if window:
                see &= j[None, :] > p[:, None] - window
        see = torch.from_numpy(see)
        for h in range(H):
            qh, kh, vh = q[r0:r1, h].double(), k[:, h // group], v[:, h // group]
            t = (qh @ kh.T) * scale
            t = t.masked_fill(~see, -math.inf)
            top = t.max(1, keepdim=True).values if t.shape[1] else torch.full((n, 1), -math.inf, dtype=torch.float64)
            e = torch.exp(t - torch.where(torch.isinf(top), torch.zeros_like(top), top)).masked_fill(~see, 0.0)
            l = e.sum(1, keepdim=True)
            w = torch.where(l == 0, torch.zeros_like(e), e / l)
            # keys not seen have no part in a row, whatever their values are
            if torch.isfinite(vh).all():
                out[r0:r1, h] = w @ vh
                mag[r0:r1, h] = w @ vh.abs()
            else:
                for i in range(n):
                    out[r0 + i, h] = w[i][see[i]] @ vh[see[i]]
                    mag[r0 + i, h] = w[i][see[i]] @ vh[see[i]].abs()
            a = ((qh.abs() @ kh.abs().T) * scale).masked_fill(~see, 0.0)
            amp[r0:r1, h] = a.max(1).values if a.shape[1] else 0.0
    return out, mag, amp


def attn_bound(out, mag, amp, act, d, keys):
    """How far an output may be off.  A score is a sum of d products whose fp32
    roundings add up like sqrt(d) of them (4 standard deviations; half of 2^-23
    each, relative to sum |q_i k_i|), e = exp(score) is off by that, the exponent's
    own rounding and the exponential's (2^-22 of |score| <= amp and of 1), and so is the
    sum below it: twice that, times sum p |v|.  The sums over the keys round like
    sqrt(keys) of 2^-24, 4 standard deviations.  fp32 activations split queries
    and weights into 16-bit terms that leave 2^-21.  16-bit activations take one
    rounding of the weights to their type, and every result one to its own."""
    u = half_step(act)
    e = amp * (4 * math.sqrt(d) * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -22 + 4 * math.sqrt(max(keys, 1)) * 2.0 ** -24
    rel = 2 * e + (2.0 ** -21 * (1 + 2 * amp) if act == "F32" else u)
    tiny = {"F32": 2.0 ** -126, "F16": 2.0 ** -24, "BF16": 2.0 ** -126}[act]
    return mag * rel[..., None] + out.abs() * u + tiny
