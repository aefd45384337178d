"""Plain restatement of the paged key/value cache and its attention (test
infrastructure): page bookkeeping with Python lists and sets, attention in 64
bits, one query row at a time; the 4-bit form of the pool, and the position
rotation of heads."""
from __future__ import annotations

import numpy as np
import torch


class ListCache:
    """The cache's state as lists: rows[i] the pages of slot i, lengths[i] its
    tokens, data [pages, layers, 2, kv_heads, page_size, head_dim]."""

    def __init__(self, data, slots, table_pages, dtype=None):
        """dtype: the 16-bit type beside a 4-bit pool (data uint8, its last two dimensions a block)."""
        self.data, self.dtype = data, dtype
        self.rows = [[] for _ in range(slots)]
        self.lengths = [0] * slots
        self.status = [0] * slots
        self.refused = [False] * slots
        self.table_pages = table_pages

    @property
    def pages(self):
        return self.data.shape[0]

    @property
    def page_size(self):
        return self.data.shape[4]

    def used(self):
        return {p for r in self.rows for p in r}

    def refs(self):
        n = [0] * self.pages
        for r in self.rows:
            for p in r:
                n[p] += 1
        return n

    def table(self):
        return [r + [-1] * (self.table_pages - len(r)) for r in self.rows]

    def free(self, mask):
        for i, m in enumerate(mask):
            if m:
                self.rows[i], self.lengths[i], self.refused[i] = [], 0, False

    def extend(self, counts):
        free = sorted(set(range(self.pages)) - self.used())
        asked = 0
        for i, c in enumerate(counts):
            self.refused[i] = False
            if c == 0:
                continue
            self.refused[i] = True
            want = -(-(self.lengths[i] + c) // self.page_size)
            if c < 0 or want > self.table_pages:
                self.status[i] = 1
                continue
            need = want - len(self.rows[i])
            asked += need
            if need and asked > len(free):
                self.status[i] = 2
                continue
            self.status[i], self.refused[i] = 0, False
            self.rows[i] += free[asked - need:asked]
            self.lengths[i] += c

    def fork(self, source, deep=False):
        before = [list(r) for r in self.rows]
        lengths = list(self.lengths)
        free = sorted(set(range(self.pages)) - self.used())
        asked = 0
        for d, s in enumerate(source):
            if s == -1 or s == d:
                continue
            if s < 0 or s >= len(before):
                self.status[d] = 1
                continue
            first = 0 if deep else lengths[s] // self.page_size
            need = len(before[s]) - first
            asked += need
            if need and asked > len(free):
                self.status[d] = 2
                continue
            self.status[d] = 0
            fresh = free[asked - need:asked]
            for old, new in zip(before[s][first:], fresh):
                self.data[new] = self.data[old]
            self.rows[d] = before[s][:first] + fresh
            self.lengths[d], self.refused[d] = lengths[s], False

    def compact(self):
        used = sorted(self.used())
        live = len(used)
        holes = [p for p in range(live) if p not in set(used)]
        to = dict(zip([p for p in used if p >= live], holes))
        for p, h in to.items():
            self.data[h] = self.data[p]
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return live

    def store(self, k, v, offsets, layers):
        """k, v [layers, rows, kv_heads, head_dim]; layers: the cache's layers they go to."""
        refs = self.refs()
        for i in range(len(self.rows)):
            a, b = offsets[i], offsets[i + 1]
            if self.refused[i]:
                continue
            if b - a > self.lengths[i]:
                self.status[i] = 1
                continue
            for r in range(a, b):
                t = self.lengths[i] - b + r
                page = self.rows[i][t // self.page_size]
                if refs[page] > 1:
                    self.status[i] = 3
                    continue
                for n, layer in enumerate(layers):
                    for kv, x in enumerate((k, v)):
                        if self.dtype is None:
                            self.data[page, layer, kv, :, t % self.page_size] = x[n, r]
                        else:
                            put4(self.data[page, layer, kv], t % self.page_size, x[n, r])


GROUP = 64
ORDER = (0, 2, 4, 6, 1, 3, 5, 7)  # of every 8 dims, from the word's lowest bits up


def quantised(x):
    """(codes, step, low) of x [..., d]: codes int64, step and low [..., groups] of x's type.  Single precision where the
    format says so, one operation at a time."""
    g = x.reshape(*x.shape[:-1], -1, GROUP).float().numpy()
    low, high = g.min(-1), g.max(-1)
    with np.errstate(all="ignore"):
        spread = high - low
        step = torch.from_numpy(np.where(np.isfinite(spread), spread / np.float32(15), np.float32("nan"))).to(x.dtype)
        s32 = step.float().numpy()
        inverse = np.where(s32 >= np.float32(2.0 ** -126), np.float32(1) / s32, np.float32(0))
        at = (g - low[..., None]) * inverse[..., None]
    codes = np.rint(np.clip(np.nan_to_num(at, nan=0.0, posinf=15.0, neginf=0.0), 0, 15))
    return torch.from_numpy(codes).long().reshape(x.shape), step, torch.from_numpy(low).to(x.dtype)


def put4(blocks, t, x):
    """Token t's x [heads, d] into blocks [heads, page_size, bytes]."""
    heads, ps, _ = blocks.shape
    d = x.shape[-1]
    codes, step, low = quantised(x)
    flat = blocks.view(heads, -1)
    words = codes.reshape(heads, -1, 8)[..., list(ORDER)]
    flat[:, t * d // 2:(t + 1) * d // 2] = (words[..., 0::2] + 16 * words[..., 1::2]).reshape(heads, -1).to(torch.uint8)
    pairs = torch.stack([step, low], -1).reshape(heads, -1).contiguous().view(torch.uint8)
    at = ps * d // 2 + t * d // 16
    flat[:, at:at + d // 16] = pairs


def held(data, dtype):
    """The values of a 4-bit pool, in 64 bits: [pages, layers, 2, kv_heads, page_size, head_dim]."""
    ps, d = data.shape[4], data.shape[5] * 16 // 9
    flat = data.reshape(*data.shape[:4], -1)
    byte = flat[..., :ps * d // 2].reshape(*data.shape[:4], ps, d // 8, 4).long()
    words = torch.stack([byte % 16, byte // 16], -1).reshape(*data.shape[:4], ps, d // 8, 8)
    codes = torch.empty_like(words)
    codes[..., list(ORDER)] = words
    pairs = flat[..., ps * d // 2:].contiguous().view(dtype).double().reshape(*data.shape[:4], ps, d // GROUP, 2)
    step, low = (pairs[..., i].repeat_interleave(GROUP, -1) for i in range(2))
    return low + step * codes.reshape(*data.shape[:4], ps, d).double()


def rotated(x, positions, rotary_dim, frequencies, interleaved=False, weight=None, eps=1e-6):
    """(y, size) in 64 bits: the heads x [rows, heads, d] normed and turned, one pair at a time; size is |a| + |b| of each
    pair before the turn (|x| past rotary_dim), which rounding errors are measured by."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    out, size = y.clone(), y.abs()
    for i in range(rotary_dim // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
        t = positions.double() * float(frequencies[i])
        cos, sin = torch.cos(t)[:, None], torch.sin(t)[:, None]
        out[..., a] = y[..., a] * cos - y[..., b] * sin
        out[..., b] = y[..., b] * cos + y[..., a] * sin
        size[..., a] = size[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, size


def attention(pool, table, lengths, layer, q, offsets, window=0, sinks=0, scale=None, key_mask=None):
    """(out, lse, weight) in 64 bits: weight = sum_j p_j |v_j|, the size that
    rounding errors of the probabilities are measured by.  CPU tensors."""
    hkv, ps, d = pool.shape[3:]
    group = q.shape[1] // hkv
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    weight = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64)
    for i in range(len(lengths)):
        a, b, n = offsets[i], offsets[i + 1], int(lengths[i])
        if b <= a or n == 0 or b - a > n:
            continue
        j = np.arange(n)
        page = torch.as_tensor(np.asarray(table[i])[j // ps], dtype=torch.long)
        k = pool[page, layer, 0, :, j % ps].double()        # [n, hkv, d]
        v = pool[page, layer, 1, :, j % ps].double()
        p = n - (b - a) + np.arange(b - a)[:, None]
        see = j[None] <= p
        if window:
            see &= (p - j[None] < window) | (j[None] < sinks)
        if key_mask is not None:
            see &= key_mask[i, :n].numpy()[None]
        for r in range(b - a):
            keys = torch.from_numpy(np.flatnonzero(see[r]))
            if not len(keys):
                continue
            x = q[a + r].double().reshape(hkv, group, d)
            s = torch.einsum("hgd,khd->hgk", x, k[keys]) * scale
            w = torch.softmax(s, -1)
            out[a + r] = torch.einsum("hgk,khd->hgd", w, v[keys]).reshape(-1, d)
            weight[a + r] = torch.einsum("hgk,khd->hgd", w, v[keys].abs()).reshape(-1, d)
            lse[a + r] = torch.logsumexp(s, -1).reshape(-1)
    return out, lse, weight
