"""Plain models of the 4-bit relay cache in numpy: 64-bit arithmetic, and loops where the kernels are
parallel (sequences one after another, pages one by one)."""
from __future__ import annotations

import numpy as np

TILE, GROUP = 16, 32


def to_bf16(x, up):
    """x (float64) rounded down or up to the 8 significant bits of bf16."""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(x)
    step = np.ldexp(1.0, np.maximum(e - 8, -133))
    return np.where(np.isfinite(x), (np.ceil(x / step) if up else np.floor(x / step)) * step, x)


def quantise(x):
    """(scale, minimum, code) of the groups of x [..., D]."""
    x = np.asarray(x, np.float64)
    x = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(all="ignore"):
        low = to_bf16(x.min(-1), False)
        span = x.max(-1) - low
        scale = np.where(span < 2.0 ** -100, 0.0, to_bf16(span / 15, True))
        bad = ~(np.abs(span) <= np.finfo(np.float32).max)
        d, s = x - low[..., None], scale[..., None]
        code = np.zeros(x.shape, np.int64)
        for c in range(15):
            code += d > (c + 0.5) * s
    code[np.broadcast_to((bad | (scale == 0))[..., None], code.shape)] = 0
    return np.where(bad, np.nan, scale), np.where(bad, np.nan, low), code


def values(x):
    """What the cache keeps of x [..., D]."""
    scale, low, code = quantise(x)
    return (low[..., None] + scale[..., None] * code).reshape(np.shape(x))


def bf16_bits(x):
    u = np.asarray(x, np.float32).view(np.uint32) >> 16
    return np.where(np.isnan(x), 0x7FFF, u).astype(np.uint16)


def pack_token(tile, k, which, x):
    """Writes one token's key or value x [D] at place k of a tile (uint8 [20 D])."""
    d = x.shape[-1]
    g = d // GROUP
    scale, low, code = quantise(x)
    base = 0 if which == "k" else 10 * d
    for c in range(d):
        j, i = divmod(c, GROUP)
        if which == "k":
            nibble = ((k * 4 + i // 8) * g + j) * 8 + i % 8
        else:
            nibble = ((((k // 8) * 8 + i // 4) * 8 + k % 8) * g + j) * 4 + i % 4
        at = base + nibble // 2
        shift = 4 * (nibble % 2)
        tile[at] = (int(tile[at]) & ~(15 << shift)) | int(code[j, i]) << shift
    words = np.stack([bf16_bits(scale), bf16_bits(low)], -1).reshape(-1).view(np.uint8)
    tile[base + 8 * d + k * 4 * g:base + 8 * d + (k + 1) * 4 * g] = words


def attention(q, k, v, own, prefix_k=None, prefix_v=None, scale=None):
    """q [N,Tq,H,D]; k, v lists of [len,Hkv,D] (values of the cache), own lens; prefix [Lp,Hkv,D].
    Returns o, row_max, row_sum and the two scales that rounding errors go by: sum p |v| / l and
    max over keys of scale * sum |q k|."""
    n, tq, h, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    o, mx, sm = np.zeros(q.shape), np.zeros(q.shape[:3]), np.ones(q.shape[:3])
    size, mass = np.zeros(q.shape), np.zeros(q.shape[:3])
    for i in range(n):
        for t in range(tq):
            end = max(0, own[i] - tq + t + 1)
            kk, vv = k[i][:end], v[i][:end]
            if prefix_k is not None:
                kk, vv = np.concatenate([prefix_k, kk]), np.concatenate([prefix_v, vv])
            if len(kk) == 0:
                continue
            group = h // kk.shape[1]
            for a in range(h):
                kh, vh = kk[:, a // group], vv[:, a // group]
                s = kh @ q[i, t, a] * scale
                m = s.max()
                p = np.exp(s - m)
                l = p.sum()
                o[i, t, a], mx[i, t, a], sm[i, t, a] = p @ vh / l, m, l
                size[i, t, a], mass[i, t, a] = p @ np.abs(vh) / l, (np.abs(kh) @ np.abs(q[i, t, a])).max() * abs(scale)
    return o, mx, sm, size, mass


class Pages:
    """The page table, lengths and reference counts, one sequence after another."""

    def __init__(self, table, lengths, refs, page):
        self.table, self.lengths, self.refs = (np.array(x, np.int64) for x in (table, lengths, refs))
        self.page = page
        self.copies = []  # (src, dst, tiles)

    def release(self, sequences):
        for s in sequences:
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s], self.lengths[s] = -1, 0

    def fork(self, parents, children):
        for a, b in zip(parents, children):
            held = -(-self.lengths[a] // self.page)
            self.table[b, :held], self.lengths[b] = self.table[a, :held], self.lengths[a]
            for p in self.table[b, :held]:
                self.refs[p] += 1

    def reserve(self, counts):
        before = self.table.copy(), self.refs.copy()
        free = [p for p in range(len(self.refs)) if self.refs[p] == 0]
        width, want, taken, copies = self.table.shape[1], 0, [], []
        asks = {}
        for s, c in enumerate(counts):
            if c > 0 and self.lengths[s] % self.page and self.table[s, self.lengths[s] // self.page] >= 0:
                asks.setdefault(self.table[s, self.lengths[s] // self.page], []).append(s)
        refs = self.refs.copy()
        for s, c in enumerate(counts):
            if c <= 0:
                continue
            length = self.lengths[s]
            slots = []
            at = length // self.page
            if length % self.page and self.table[s, at] >= 0:
                p = self.table[s, at]
                if refs[p] > 1 and not (len(asks[p]) == refs[p] and asks[p][-1] == s):
                    slots.append(at)
            slots += [w for w in range(-(-length // self.page), -(-(length + c) // self.page))
                      if w < width and self.table[s, w] < 0]
            for w in slots:
                taken.append((s, w))
        if len(taken) > len(free):
            return len(taken) - len(free)
        for p, (s, w) in zip(free, taken):
            if self.table[s, w] >= 0:
                self.refs[self.table[s, w]] -= 1
                copies.append((self.table[s, w], p, -(-(self.lengths[s] % self.page) // TILE)))
            self.table[s, w], self.refs[p] = p, 1
        self.copies = copies
        return 0

    def compact(self):
        used = int((self.refs > 0).sum())
        holes = [p for p in range(used) if self.refs[p] == 0]
        movers = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        self.copies = []
        for a, b in zip(movers, holes):
            self.table[self.table == a] = b
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.copies.append((a, b, None))
        return used

    def apply(self, pool):
        """The copies on a pool (uint8 array), all reading before any writes."""
        pool = pool.copy()
        read = [(b, t, pool[a].copy()) for a, b, t in self.copies]
        for b, t, data in read:
            pool[b, :, :t] = data[:, :t]
        return pool
