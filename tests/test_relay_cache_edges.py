"""The 4-bit relay cache where its state or its numbers are unusual: lengths that were lowered or lie past the table,
rows that hold pages before they hold tokens, values and queries of all sizes, host threads, streams and graphs."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import delta_block_lm_b200 as dbl
import relay_cache_model as M
from delta_block_lm_b200 import relay_cache as R
from test_relay_cache import _device_code, _fill, _i32, _ok, _same, _state, _tables, _three

gpu = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U32 = 2.0 ** -23  # spacing of f32


# ------------------------------------------------------------------------------------------ pages
class Pages(M.Pages):
    """The sequential model with the rule for every page that the next tokens are written to, whatever was done to the
    lengths: a page that others hold too is replaced (with its tokens, where it holds some below the length), except
    for the last of its holders where all of them are about to write to it."""

    def written(self, s, count):
        first, end = self.lengths[s] // self.page, -(-(self.lengths[s] + count) // self.page)
        return range(first, min(end, self.table.shape[1])) if count > 0 else range(0)

    def reserve(self, counts):
        free = [p for p in range(len(self.refs)) if self.refs[p] == 0]
        asks, taken = {}, []
        for s, c in enumerate(counts):
            for w in self.written(s, c):
                if self.table[s, w] >= 0:
                    asks.setdefault(self.table[s, w], []).append(s)
        for s, c in enumerate(counts):
            for w in self.written(s, c):
                p = self.table[s, w]
                if p < 0:
                    if w * self.page >= self.lengths[s]:
                        taken.append((s, w))
                elif self.refs[p] > 1 and not (len(asks[p]) == self.refs[p] and asks[p][-1] == s):
                    taken.append((s, w))
        if len(taken) > len(free):
            return len(taken) - len(free)
        self.copies = []
        for p, (s, w) in zip(free, taken):
            old = self.table[s, w]
            if old >= 0:
                self.refs[old] -= 1
                if w * self.page < self.lengths[s]:
                    self.copies.append((old, p, -(-(self.lengths[s] % self.page) // M.TILE)))
            self.table[s, w], self.refs[p] = p, 1
        return 0


@gpu
@pytest.mark.parametrize("rows,width,page,pages", [(6, 4, 16, 40), (40, 9, 64, 400), (300, 40, 32, 12000), (3, 150, 16, 500)])
def test_reserve_after_lengths_were_lowered(cuda, native_lib, rows, width, page, pages):
    """Forks, then lengths cut back to any place, page boundaries among them: every page in the range to be written is the
    sequence's own afterwards, and the rest follows the sequential model to the byte."""
    rng = np.random.default_rng(rows)
    for turn in range(6):
        s = _state(rng, rows, width, page, pages, max(1, rows // 2), width * page * 3 // 4)
        m = Pages(s.table, s.lengths, s.refs, page)
        pool = torch.randint(0, 256, (pages, 1, page // 16, 1280), device=cuda, dtype=torch.uint8)
        full = [i for i in range(rows) if m.lengths[i] > 0]
        children = [i for i in range(rows) if m.lengths[i] == 0 and (m.table[i] < 0).all()] if full else []
        m.fork([int(rng.choice(full)) for _ in children], children)
        for i in range(rows):
            kind = rng.integers(0, 4)
            if kind == 1:
                m.lengths[i] = rng.integers(0, m.lengths[i] + 1)
            elif kind == 2:
                m.lengths[i] = m.lengths[i] // page * page
            elif kind == 3:
                m.lengths[i] = rng.integers(0, m.lengths[i] // page + 1) * page
        counts = [int(rng.integers(1, 3 * page)) if rng.random() < 0.7 else 0 for _ in range(rows)]
        counts = [min(c, width * page - int(m.lengths[i])) for i, c in enumerate(counts)]
        old, state = pool.cpu().numpy().copy(), _three(m, cuda)
        table, refs, missing = dbl.relay_cache_reserve(pool, *state, _i32(counts, cuda),
                                                       out=(state[0], state[2]) if turn % 2 else None)
        short = m.reserve(counts)
        assert missing.tolist() == [short]
        _same([table, refs], m, what=2)
        assert np.array_equal(pool.cpu().numpy(), m.apply(old) if not short else old)
        if not short:
            held = table.cpu().numpy()
            for i, c in enumerate(counts):
                for w in m.written(i, c):
                    assert (held == held[i, w]).sum() == 1, (i, w)
        assert np.array_equal(np.bincount(m.table[m.table >= 0], minlength=pages), m.refs)
    _ok()


@gpu
@pytest.mark.parametrize("cut,more", [(10, 20), (16, 20), (20, 25), (32, 8), (0, 40), (39, 1)])
def test_a_cut_fork_leaves_the_other_sequence_alone(cuda, native_lib, cut, more):
    """Fork at 40 tokens (pages of 16), drop the child's tokens past `cut`, reserve and append `more`: the parent's tokens
    stay, and the child holds its first `cut` and the new ones."""
    rng = np.random.default_rng(cut)
    pool = dbl.relay_cache_pool(12, 2, 64, 16, device=cuda)
    state = [torch.full((2, 5), -1, device=cuda, dtype=torch.int32), _i32([0, 0], cuda), _i32([0] * 12, cuda)]
    k, v = (torch.as_tensor(rng.standard_normal((2, 40, 2, 64))).to(cuda, BF16) for _ in "kv")

    def write(state, counts, k, v):
        table, refs, missing = dbl.relay_cache_reserve(pool, *state, _i32(counts, cuda))
        assert missing.tolist() == [0]
        return [table, dbl.relay_cache_append(pool, table, state[1], k, v, counts=_i32(counts, cuda)), refs]

    state = write(state, [40, 0], k, v)
    state = list(dbl.relay_cache_fork(pool, *state, _i32([0], cuda), _i32([1], cuda)))
    before = dbl.relay_cache_read(pool, state[0], state[1], tokens=40, dtype=F32)
    state[1] = _i32([40, cut], cuda)
    state = write(state, [0, more], k, v)
    after = dbl.relay_cache_read(pool, state[0], state[1], tokens=cut + more, dtype=F32)
    for b, a, x in zip(before, after, (k, v)):
        assert torch.equal(a[0, :40], b[0, :cut + more])
        assert torch.equal(a[1, :cut], b[0, :cut])
        new = M.values(x[1, :more].double().cpu().numpy()).astype(np.float32)
        assert np.array_equal(a[1, cut:].cpu().numpy(), new)
    _ok()


@gpu
def test_fork_into_a_row_that_holds_pages(cuda, native_lib):
    """A sequence without tokens that reserve has given pages, or one with tokens: fork gives the pages back."""
    pool = dbl.relay_cache_pool(8, 1, 64, 16, device=cuda)
    state = [torch.full((3, 4), -1, device=cuda, dtype=torch.int32), _i32([0, 0, 0], cuda), _i32([0] * 8, cuda)]
    table, refs, _ = dbl.relay_cache_reserve(pool, *state, _i32([20, 33, 1], cuda))
    assert refs.tolist() == [1, 1, 1, 1, 1, 1, 0, 0]
    for out in (False, True):
        state = [table.clone(), _i32([20, 0, 0], cuda), refs.clone()]
        got = dbl.relay_cache_fork(pool, *state, _i32([0, 0], cuda), _i32([1, 2], cuda), out=state if out else None)
        assert got[0].tolist() == [[0, 1, -1, -1]] * 3 and got[1].tolist() == [20, 20, 20]
        assert got[2].tolist() == [3, 3, 0, 0, 0, 0, 0, 0]
    # a child that held tokens of its own
    state = [table.clone(), _i32([20, 33, 1], cuda), refs.clone()]
    got = dbl.relay_cache_fork(pool, *state, _i32([0], cuda), _i32([1], cuda))
    assert got[0].tolist() == [[0, 1, -1, -1], [0, 1, -1, -1], [5, -1, -1, -1]] and got[1].tolist() == [20, 20, 1]
    assert got[2].tolist() == [2, 2, 0, 0, 0, 1, 0, 0]
    # a child that held the parent's own page already
    state = [_i32([[0, 1], [1, -1]], cuda), _i32([20, 0], cuda), _i32([1, 2, 0, 0, 0, 0, 0, 0], cuda)]
    got = dbl.relay_cache_fork(pool, *state, _i32([0], cuda), _i32([1], cuda))
    assert got[0].tolist() == [[0, 1], [0, 1]] and got[2].tolist() == [2, 2, 0, 0, 0, 0, 0, 0]
    _ok()


# ------------------------------------------------------------------------------------------ append and read
@gpu
@pytest.mark.parametrize("length", [-1, -3, -31, -100, -2 ** 31])
def test_append_at_a_negative_length_is_recorded(cuda, native_lib, length):
    """A call of many tokens does what single tokens do: those at negative positions are left out and recorded."""
    rng = np.random.default_rng(4)
    h, d, page, t = 2, 64, 16, 40
    k, v = (torch.as_tensor(rng.standard_normal((2, t, h, d))).to(cuda, BF16) for _ in "kv")
    tab = _i32([[0, 1, 2], [3, 4, 5]], cuda)
    pools = [dbl.relay_cache_pool(6, h, d, page, device=cuda) for _ in "ab"]
    dbl.relay_cache_append(pools[0], tab, _i32([length, 3], cuda), k, v)
    assert _device_code() == 102
    for i in range(t):
        dbl.relay_cache_append(pools[1], tab, _i32([length + i, 3 + i], cuda), k[:, i:i + 1], v[:, i:i + 1])
        assert (_device_code() == 102) == (length + i < 0)
    assert torch.equal(*pools)
    dbl.relay_cache_append(pools[0], tab, _i32([length, 3], cuda), k, v, counts=_i32([0, 1], cuda))
    _ok()


@gpu
def test_read_that_starts_far_past_the_end(cuda, native_lib):
    """Zeros and no error, whatever the number of tokens, up to the last position that 32 bits hold."""
    pool, tab, held, _, _ = _fill(cuda, np.random.default_rng(0), [40, 3], 1, 64, 16)
    for start in (48, 2 ** 31 - 1, 2 ** 31 - 17, 2 ** 31 - 40):
        for tokens in (1, 70):
            k, v = dbl.relay_cache_read(pool, tab, held, start=_i32([start, start], cuda), tokens=tokens, dtype=F32)
            assert not k.any() and not v.any()
            _ok()
    for tokens in (5, 70):  # and far before the beginning
        k, v = dbl.relay_cache_read(pool, tab, held, start=_i32([-2 ** 31, -2 ** 31 + 9], cuda), tokens=tokens, dtype=F32)
        assert not k.any() and not v.any()
        _ok()


# ------------------------------------------------------------------------------------------ attention
def _attend(q, kk, vv, lens, pre=(None, None), scale=None):
    """The model's result and, for each row and channel, sum p (|minimum| + 8 scale) / l and max p scale / l of what the
    cache holds of its group: the sizes that the rounding of p goes by.  kk, vv: lists of (scale, minimum, code)."""
    full = lambda x: (x[1][..., None] + x[0][..., None] * x[2]).reshape(*x[0].shape[:-1], -1)  # noqa: E731
    join = lambda a, b: b if a is None else tuple(np.concatenate([x, y]) for x, y in zip(a, b))  # noqa: E731
    n, tq, h, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    o, mx, sm = np.zeros(q.shape), np.zeros(q.shape[:3]), np.ones(q.shape[:3])
    size, most, mass = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3])
    count = np.ones(q.shape[:3])
    for i in range(n):
        for t in range(tq):
            end = max(0, lens[i] - tq + t + 1)
            keys, vals = (join(p, tuple(y[:end] for y in x[i])) for p, x in zip(pre, (kk, vv)))
            if len(keys[0]) == 0:
                continue
            kf, vf = full(keys), full(vals)
            for a in range(h):
                b = a // (h // kf.shape[1])
                s = kf[:, b] @ q[i, t, a] * scale
                m = s.max()
                p = np.exp(s - m)
                l = p.sum()
                o[i, t, a], mx[i, t, a], sm[i, t, a] = p @ vf[:, b] / l, m, l
                per = p[:, None] * (np.abs(vals[1][:, b]) + 8 * vals[0][:, b]) / l
                size[i, t, a] = np.repeat(per.sum(0), M.GROUP)
                most[i, t, a] = np.repeat((p[:, None] * vals[0][:, b] / l).max(0), M.GROUP)
                mass[i, t, a] = (np.abs(kf[:, b]) @ np.abs(q[i, t, a])).max() * abs(scale)
                count[i, t, a] = len(s)
    return o, mx, sm, size, most, mass, count


def _check(got, want, dtype):
    """Channel by channel.  A score is off by 2 d + 8 roundings of its terms (f32 sums) and p by 2 more units; p scale
    is rounded to f16 once (bf16 rows: 2^-12 of it) or twice (f32 rows: 2^-22 at the least), with a floor of 2^-25 where
    the largest is 2^7, so 2^-32 of the largest for each of at most `count` keys and codes up to 8 from zero; p to two
    bf16 parts for the minima (2^-17); sums over the keys; the output's own rounding."""
    o, mx, sm = (x.double().cpu().numpy().reshape(w.shape) for x, w in zip(got, want))
    eo, em, es, size, most, mass, count = want
    d = eo.shape[-1]
    ds = (2 * d + 8) * U32 * mass + 4 * U32 + U32 * np.abs(em)
    tail = np.sqrt(count) * 4 * U32
    assert (np.abs(mx - em) <= ds).all()
    assert (np.abs(sm - es) <= es * (2 * ds + tail) + U32).all()
    dp = 2.0 ** -12 + 2.0 ** -17 if dtype == BF16 else 2.0 ** -22
    tol = size * (2 * ds + tail + dp)[..., None] + count[..., None] * 2.0 ** -29 * most
    tol = tol * (1 + 2.0 ** -7) + np.abs(eo) * (2.0 ** -8 if dtype == BF16 else U32)
    assert np.isfinite(o).all()
    assert (np.abs(o - eo) <= tol).all(), float((np.abs(o - eo) / np.maximum(tol, 1e-300)).max())


def _kept(tiles, length):
    """((scale, minimum, code) of the keys, of the values) in the bytes of tiles [n, Hkv, 20 D], tokens [length, Hkv, ...].
    (How append rounds to them is tested to the byte elsewhere.)"""
    n, h, size = tiles.shape
    d, g = size // 20, size // 20 // M.GROUP
    out = []
    for at, shape in ((0, (16, 4, g, 8)), (10 * d, (2, 8, 8, g, 4))):
        x = tiles[..., at:at + 8 * d]
        x = np.stack([x & 15, x >> 4], -1).reshape(n, h, *shape)
        if at:  # [n, h, half, part, token, group, code] -> [n, half, token, h, group, part, code]
            x = x.transpose(0, 2, 4, 1, 5, 3, 6)
        else:  # [n, h, token, part, group, code] -> [n, token, h, group, part, code]
            x = x.transpose(0, 2, 1, 4, 3, 5)
        words = np.ascontiguousarray(tiles[..., at + 8 * d:at + 10 * d]).view(np.uint16).reshape(n, h, 16, g, 2)
        words = (words.astype(np.uint32) << 16).view(np.float32).astype(np.float64).transpose(0, 2, 1, 3, 4)
        words, x = words.reshape(n * 16, h, g, 2)[:length], x.reshape(n * 16, h, g, M.GROUP)[:length]
        out.append((words[..., 0], words[..., 1], x.astype(np.int64)))
    return out


def _cache(dev, k, v, page):
    """A pool that holds the sequences k[i], v[i] [length, Hkv, D] (tensors on the device), its table and lengths, and
    what it keeps of them."""
    lens = [len(x) for x in k]
    table, pages, _ = _tables(np.random.default_rng(0), lens, page)
    pool = dbl.relay_cache_pool(pages, k[0].shape[1], k[0].shape[2], page, device=dev)
    pool.fill_(255)
    tab, zero = _i32(table, dev), _i32([0], dev)
    for i, n in enumerate(lens):
        dbl.relay_cache_append(pool, tab[i:i + 1], zero, k[i][None], v[i][None])
    tiles = [pool[tab[i, :-(-n // page)].long()].transpose(1, 2).flatten(0, 1).cpu().numpy() for i, n in enumerate(lens)]
    kept = [_kept(x, n) for x, n in zip(tiles, lens)]
    return pool, tab, _i32(lens, dev), [x[0] for x in kept], [x[1] for x in kept]


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tq,g,prefix,n", [(1, 1, 0, 2), (1, 2, 21, 3), (2, 1, 0, 2), (9, 1, 0, 2), (9, 2, 37, 2), (3, 1, 33000, 4)])
def test_attention_lengths_past_the_table(cuda, native_lib, dtype, tq, g, prefix, n):
    """A table of 2 pages of 16 tokens and lengths up to 40: the queries count from the length, the tokens that the table
    has no pages for are left out and recorded."""
    rng = np.random.default_rng(tq)
    hkv, d, page = 4, 64, 16
    assert prefix == 33000 or n * hkv * prefix < 1 << 19  # with and without a launch of the prefix's own
    lens = [32] * n
    k, v = ([torch.as_tensor(rng.standard_normal((x, hkv, d))).to(cuda, BF16) for x in [prefix] + lens] for _ in "kv")
    pool, tab, held, kk, vv = _cache(cuda, k, v, page)
    own = tab[1:, :2].contiguous()
    q = torch.as_tensor(rng.standard_normal((n, tq, hkv * g, d))).to(cuda, dtype)
    kw = dict(prefix_pages=tab[0], prefix_len=prefix) if prefix else {}
    pre = (kk[0], vv[0]) if prefix else (None, None)
    for past in (0, 1, 8, 40, 2 ** 31 - 33):
        now = [32 + past] + [32] * (n - 1)
        got = dbl.relay_cache_attention(q, pool, own, _i32(now, cuda), **kw)
        assert _device_code() == (102 if past else 0)
        _check(got, _attend(q.double().cpu().numpy(), kk[1:], vv[1:], now, pre), dtype)
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_values_near_the_largest(cuda, native_lib, dtype, d):
    """Values of 2^120, and scores that rise by 5.4 after the running maximum was set: the sums stay in range where p is
    at most 1 (264 tokens of 2^120), and so does the result."""
    rng = np.random.default_rng(d)
    t = 264
    k = rng.standard_normal((t, 1, d)) * 1e-3
    k[260:] += 5.4 / d ** 0.5
    v = rng.uniform(1.8, 1.99, (t, 1, d)) * 2.0 ** 119
    k, v = (torch.as_tensor(x).to(cuda, BF16) for x in (k, v))
    pool, tab, held, kk, vv = _cache(cuda, [k], [v], 16)
    q = torch.ones((1, 1, 1, d), device=cuda, dtype=dtype)
    _check(dbl.relay_cache_attention(q, pool, tab, held), _attend(q.double().cpu().numpy(), kk, vv, [t]), dtype)
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tq,g", [(1, 1), (1, 6), (1, 14), (5, 1)])
@pytest.mark.parametrize("sizes", [(0, -2, -4, -6), (-1, -3, -5, -7), (0, -8, -10, -12), (3, 3, -20, -25), (-9, 0), (-5, -7)])
def test_attention_value_groups_of_different_sizes(cuda, native_lib, dtype, tq, g, sizes):
    """Groups of 32 channels whose values are powers of ten apart: every channel is as exact as its own group allows.
    Small queries, so that the scores' own error does not hide it."""
    rng = np.random.default_rng(g + len(sizes))
    d, hkv, lens = 32 * len(sizes), 2, [300, 33]
    size = np.repeat(10.0 ** np.array(sizes), 32)
    k, v = ([torch.as_tensor(rng.standard_normal((n, hkv, d)) * x).to(cuda, F32) for n in lens] for x in (1, size))
    pool, tab, held, kk, vv = _cache(cuda, k, v, 16)
    q = torch.as_tensor(rng.standard_normal((2, tq, hkv * g, d)) * 1e-3).to(cuda, dtype)
    _check(dbl.relay_cache_attention(q, pool, tab, held), _attend(q.double().cpu().numpy(), kk, vv, lens), dtype)
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("g,d", [(1, 128), (3, 64), (7, 128), (16, 64)])
@pytest.mark.parametrize("prefix,rise", [(0, 0.02), (50, 0.02), (0, -0.02), (50, -0.02), (0, 3.0), (50, 3.0), (0, 400.0),
                                         (70000, 0.02), (70000, 3.0)])
def test_attention_scores_that_rise_and_values_that_change(cuda, native_lib, dtype, g, d, prefix, rise):
    """Scores that rise (or fall) from token to token, up to far past what one power of two of p covers, with value
    sizes that differ by token and by group, each in its own order."""
    rng = np.random.default_rng(g + prefix)
    n, t = 4, 700
    lens, hkv = [t, 1, 130, 0], 2
    assert (prefix == 70000) == (n * hkv * prefix >= 1 << 19)  # with a launch of the prefix's own
    k, v = [], []
    for x in [prefix] + lens:
        y = rng.standard_normal((x, hkv, d)) * 1e-2
        y[..., 0] = (np.arange(x) % t)[:, None] * rise  # channel 0 carries the score
        z = rng.standard_normal((x, hkv, d // 32, 32)) * 10.0 ** rng.integers(-6, 7, (x, hkv, d // 32, 1))
        k.append(torch.as_tensor(y).to(cuda, F32)), v.append(torch.as_tensor(z.reshape(x, hkv, d)).to(cuda, F32))
    pool, tab, held, kk, vv = _cache(cuda, k, v, 64)
    q = torch.as_tensor(rng.standard_normal((n, 1, hkv * g, d)) * 1e-2)
    q[..., 0] = d ** 0.5 / torch.arange(1, hkv * g + 1)
    q = q.to(cuda, dtype)
    kw = dict(prefix_pages=tab[0], prefix_len=prefix) if prefix else {}
    want = _attend(q.double().cpu().numpy(), kk[1:], vv[1:], lens, (kk[0], vv[0]) if prefix else (None, None))
    _check(dbl.relay_cache_attention(q[:, 0], pool, tab[1:], held[1:], **kw), want, dtype)
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("exponent", [10, 24, 31, 40, 80, 118])
@pytest.mark.parametrize("tq,g,prefix", [(1, 1, 0), (1, 7, 40), (3, 4, 0)])
def test_attention_scores_of_all_sizes(cuda, native_lib, dtype, exponent, tq, g, prefix):
    """Scores up to 2^118: the largest has the weight 1 (as many times as it occurs), the others what their distance
    gives, however coarse the scores are."""
    rng = np.random.default_rng(exponent + g)
    d, lens = 64, [300, 61]
    k, v = ([torch.as_tensor(rng.uniform(-1, 1, (n, 2, d))).to(cuda, BF16) for n in [prefix] + lens] for _ in "kv")
    k[1][200] = k[1][7]  # the same key twice, in the steps of different warps
    pool, tab, held, kk, vv = _cache(cuda, k, v, 32)
    q = torch.as_tensor(rng.uniform(-1, 1, (2, tq, 2 * g, d)) * 2.0 ** (exponent // 2)).to(cuda, dtype)
    q[0, :, 0] = k[1][7, 0].to(dtype) * 2.0 ** (exponent // 2)  # which the query finds
    scale = 2.0 ** (exponent - exponent // 2)
    kw = dict(prefix_pages=tab[0], prefix_len=prefix) if prefix else {}
    got = dbl.relay_cache_attention(q, pool, tab[1:], held[1:], scale=scale, **kw)
    want = _attend(q.double().cpu().numpy(), kk[1:], vv[1:], lens, (kk[0], vv[0]) if prefix else (None, None), scale)
    o, mx, sm = (x.double().cpu().numpy().reshape(w.shape) for x, w in zip(got, want))
    ds = (2 * d + 8) * U32 * want[5]
    far = ds > 0.1
    assert (np.abs(mx - want[1]) <= ds + 4 * U32 + U32 * np.abs(want[1])).all()
    near = torch.as_tensor(~far, device=cuda)
    _check([x.reshape(w.shape)[near] for x, w in zip(got, want)], [x[~far] for x in want], dtype)
    # the first rows find one key twice: 2 of its weight, its value rows averaged; with another key as near as the
    # scores' rounding the weights may differ, so the others are looked at for what every softmax keeps
    assert np.isfinite(o).all() and (sm >= 1 - 1e-5).all() and (sm <= max(lens) + prefix + 1).all()
    values = np.concatenate([(x[1][..., None] + x[0][..., None] * x[2]).reshape(-1, 2, d) for x in vv])
    assert (np.abs(o) <= np.abs(values).max() * (1 + 2.0 ** -7)).all()
    if exponent >= 31:
        both = values[prefix + 7] + values[prefix + 200]
        assert np.allclose(sm[0, :, 0], 2, rtol=1e-6)
        assert (np.abs(o[0, :, 0] - both[0] / 2) <= 2.0 ** -8 * (np.abs(both[0]) + 15 * max(vv[1][0][7, 0].max(), vv[1][0][200, 0].max()))).all()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("exponents,k_exponent,scale", [
    ((90, 111, 112, 118, 121, 123, 125, 126), 0, 2.0 ** -124), ((-112, -118, -122, -125), 112, 0.25),
    ((127, 120, 112, -3), -60, None), ((126, 126, 124, 3, 126, 122, 117, 111, 126, 125, 126), -8, None)])
@pytest.mark.parametrize("tq", [1, 3])
def test_attention_queries_of_all_sizes(cuda, native_lib, dtype, exponents, k_exponent, scale, tq):
    """Queries of 2^-125 to the largest that the type holds, where the scores are finite."""
    rng = np.random.default_rng(len(exponents))
    d, lens, h = 64, [200, 40], len(exponents)
    k, v = ([torch.as_tensor(rng.uniform(-1, 1, (n, 1, d)) * x).to(cuda, F32) for n in lens] for x in (2.0 ** k_exponent, 1))
    pool, tab, held, kk, vv = _cache(cuda, k, v, 32)
    q = rng.uniform(-1, 1, (2, tq, h, d)) * 2.0 ** np.array(exponents)[:, None]
    q[..., 1, 5] = np.sign(q[..., 1, 5]) * 1.9 * 2.0 ** exponents[1]
    q = torch.as_tensor(q).to(cuda, dtype)
    want = _attend(q.double().cpu().numpy(), kk, vv, lens, scale=scale)
    assert np.abs(want[5]).max() < 2.0 ** 127
    got = dbl.relay_cache_attention(q, pool, tab, held, scale=scale)
    # where the scores' rounding is as large as their softmax resolves, one key has all of the weight
    ds = (2 * d + 8) * U32 * want[5]
    far, near = ds > 0.1, torch.as_tensor(ds <= 0.1, device=cuda)
    assert (want[2][far] < 1 + 1e-6).all()
    _check([x.reshape(w.shape)[near] for x, w in zip(got, want)], [x[~far] for x in want], dtype)
    o, mx, _ = (x.double().cpu().numpy().reshape(w.shape) for x, w in zip(got, want))
    assert (np.abs(mx - want[1])[far] <= (ds + U32 * np.abs(want[1]))[far]).all()
    tol = (2.0 ** -8 if dtype == BF16 else 2.0 ** -20) * (np.abs(want[0]) + want[3])
    assert (np.abs(o - want[0])[far] <= tol[far]).all()
    _ok()


@gpu
@pytest.mark.parametrize("d,g", [(64, 7), (128, 1)])
def test_attention_long_sums_of_f32_rows(cuda, native_lib, d, g):
    """95000 tokens whose values average out, ten sequences on the same pages, so that one warp sums 34 steps: the result
    is small beside its terms, and no term of one sign may grow in a sum that drops bits.  A warp adds 136 times
    (34 steps of 2 tiles and 2 parts), each time dropping at most 2^-23 of a sum, half of it on average."""
    rng = np.random.default_rng(d)
    n, hkv, t = 10, 2, 95000
    k, v = (torch.as_tensor(rng.standard_normal((t, hkv, d))).to(cuda, BF16) for _ in "kv")
    pool, tab, held, kk, vv = _cache(cuda, [k], [v], 64)
    q = torch.as_tensor(rng.standard_normal((n, 1, hkv * g, d)) * 0.05).to(cuda, F32)
    got = dbl.relay_cache_attention(q, pool, tab.expand(n, -1).contiguous(), held.expand(n).contiguous())
    want = _attend(q.double().cpu().numpy(), kk * n, vv * n, [t] * n)
    err = got[0].double().cpu().numpy() - want[0]
    assert np.linalg.norm(err) <= 136 * 2.0 ** -24 * np.linalg.norm(want[0])
    _ok()


@gpu
def test_attention_long_sums_of_bf16_rows(cuda, native_lib):
    """16 sequences on the same 131072 tokens, whose values average out: beside the rounding of the output to bf16 there is
    the rounding of p scale to f16 (a tenth of it) and no more, however many steps a warp sums (443 in one run)."""
    torch.manual_seed(1)
    n, t, h, d, page = 16, 131072, 16, 64, 64
    pool = dbl.relay_cache_pool(t // page, h, d, page, device=cuda)
    tab, held = torch.randperm(t // page, device=cuda).to(torch.int32)[None], _i32([0], cuda)
    for _ in range(8):
        k, v = (torch.randn(1, t // 8, h, d, device=cuda) for _ in "kv")
        held = dbl.relay_cache_append(pool, tab, held, k, v)
    q = (torch.randn(n, h, d, device=cuda) * 0.05).bfloat16()
    o, _, _ = dbl.relay_cache_attention(q, pool, tab.expand(n, -1).contiguous(), held.expand(n).contiguous())
    k, v = dbl.relay_cache_read(pool, tab, held, tokens=t, dtype=F32)
    for a in (0, 7, 15):
        p = torch.softmax(q[:, a].double() @ k[0, :, a].double().T * d ** -0.5, -1)
        want = p @ v[0, :, a].double()
        assert (o[:, a].double() - want).norm() <= 1.1 * (want.bfloat16().double() - want).norm()
    _ok()


# ------------------------------------------------------------------------------------------ threads, streams, graphs
def test_threads_do_not_share_a_workspace(monkeypatch):
    """A call can be two launches that hand results over in its workspace, and the interpreter lock is let go in between:
    host threads on one stream need workspaces of their own, and one thread keeps its own from call to call."""
    real = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: real(*a, **kw))
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: False)
    ready, got = threading.Barrier(2, timeout=30), [None, None]

    def work(i):
        mine = R._workspace("attention", 9000, 0, 7)
        ready.wait()
        got[i] = mine.data_ptr(), R._workspace("attention", 8500, 0, 7).data_ptr(), mine
        ready.wait()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got[0][0] != got[1][0]
    assert all(first == again for first, again, _ in got)


@gpu
def test_two_threads_on_one_stream(cuda, native_lib):
    """Attention with a launch of the prefix's own, reserve with copies and compact, from two host threads on the default
    stream, each with its own state: every result is the one that the thread gets alone."""
    rng = np.random.default_rng(3)

    def job(i):
        n, hkv, d, page, prefix = 8, 16, 64, 64, 4096 + 64 * i
        pool = dbl.relay_cache_pool(100 + n, hkv, d, page, device=cuda)
        tab = torch.arange(100 + n, device=cuda, dtype=torch.int32)
        k, v = (torch.as_tensor(rng.standard_normal((1, prefix + 40 * n, hkv, d))).to(cuda, BF16) for _ in "kv")
        dbl.relay_cache_append(pool, tab[None], _i32([0], cuda), k, v)
        q = torch.as_tensor(rng.standard_normal((n, hkv, d))).to(cuda, BF16)
        own, lens = tab[60:60 + n, None].contiguous(), _i32(range(5, 5 + n), cuda)
        # pages 0 .. 9 of two sequences, the second a fork of the first, holes between them
        table = torch.full((4, 12), -1, device=cuda, dtype=torch.int32)
        table[0, :10] = torch.arange(0, 30, 3, device=cuda) + i
        table[1:3] = table[0]
        refs = torch.zeros(len(pool), device=cuda, dtype=torch.int32)
        refs[table[0, :10].long()] = 3
        small = pool.clone()

        def attend():
            return dbl.relay_cache_attention(q, pool, own, lens, prefix_pages=tab[:66], prefix_len=prefix)

        def pages():
            p = small.clone()
            t, r, missing = dbl.relay_cache_reserve(p, table, _i32([600, 600, 600, 0], cuda), refs, 30)
            t, r, used = dbl.relay_cache_compact(p, t, r)
            return p, t, r, missing, used

        return attend, pages

    jobs = [job(i) for i in range(2)]
    want = [[f() for f in j] for j in jobs]
    torch.cuda.synchronize()
    wrong, failures = [torch.zeros(1, device=cuda, dtype=torch.int64) for _ in jobs], []
    ready = threading.Barrier(2, timeout=60)

    def work(i):
        try:
            ready.wait()
            for _ in range(150):
                for f, w in zip(jobs[i], want[i]):
                    for a, b in zip(f(), w):
                        wrong[i] += (a != b).any()
        except Exception as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures and [int(x) for x in wrong] == [0, 0]
    _ok()


@gpu
@pytest.mark.parametrize("prefix", [37, 20000])
def test_a_serving_loop_in_a_graph(cuda, native_lib, prefix):
    """Release, fork, reserve, append, attention, read and compact captured as one graph that updates its state in place:
    every replay gives what the same calls give outside a graph, from the same state."""
    rng = np.random.default_rng(prefix)
    n, hkv, d, page = 14, 2, 64, 16
    assert (prefix == 20000) == (n * hkv * prefix >= 1 << 19)  # with a launch of the prefix's own
    width = -(-prefix // page)
    pool = dbl.relay_cache_pool(width + 12 * n, hkv, d, page, device=cuda)
    pool.fill_(255)
    table = torch.full((n + 1, width + 8), -1, device=cuda, dtype=torch.int32)  # the last row: the shared prompt
    state = [table, _i32([0] * (n + 1), cuda), _i32([0] * len(pool), cuda)]

    def write(pool, state, counts, k, v, out=False):
        table, refs, missing = dbl.relay_cache_reserve(pool, *state, counts, out=(state[0], state[2]) if out else None)
        lengths = dbl.relay_cache_append(pool, table, state[1], k, v, counts=counts, out=state[1] if out else None)
        return [table, lengths, refs], missing

    def tokens(t):
        return [torch.as_tensor(rng.standard_normal((n + 1, t, hkv, d))).to(cuda, BF16) for _ in "kv"]

    state, missing = write(pool, state, _i32([0] * n + [prefix], cuda), *tokens(prefix))
    state, missing = write(pool, state, _i32([20 + i for i in range(n)] + [0], cuda), *tokens(40))
    assert missing.tolist() == [0]
    # the inputs of a step, which the graph reads where they are
    gone, parents = _i32([0, 0], cuda), _i32([0, 0], cuda)
    counts, q = _i32([1] * n + [0], cuda), torch.zeros((n, 3 * hkv, d), device=cuda, dtype=BF16)
    k, v = tokens(1)

    def step(pool, state, out):
        state = list(dbl.relay_cache_release(pool, *state, gone, out=state if out else None))
        state = list(dbl.relay_cache_fork(pool, *state, parents, gone, out=state if out else None))
        state, missing = write(pool, state, counts, k, v, out)
        got = dbl.relay_cache_attention(q, pool, state[0][:n], state[1][:n], prefix_pages=state[0][n], prefix_len=prefix)
        back = dbl.relay_cache_read(pool, state[0], state[1], tokens=50, dtype=F32)
        table, refs, used = dbl.relay_cache_compact(pool, state[0], state[2], out=(state[0], state[2]) if out else None)
        return [table, state[1], refs], [*got, *back, missing, used]

    gone.copy_(_i32([1, 5], cuda)), parents.copy_(_i32([3, 3], cuda))
    step(pool.clone(), [x.clone() for x in state], True)  # everything is loaded before the capture
    torch.cuda.synchronize()
    graph, kept, kept_pool = torch.cuda.CUDAGraph(), [x.clone() for x in state], pool.clone()
    with torch.cuda.graph(graph):
        after, outputs = step(kept_pool, kept, True)
    for _ in range(12):
        two = rng.permutation(n)[:4]
        gone.copy_(_i32(two[:2], cuda)), parents.copy_(_i32(two[2:], cuda))
        q.copy_(torch.as_tensor(rng.standard_normal(q.shape)))
        for x, y in zip((k, v), tokens(1)):
            x.copy_(y)
        graph.replay()
        state, want = step(pool, state, False)
        assert all(torch.equal(a, b) for a, b in zip(outputs, want))
        assert all(torch.equal(a, b) for a, b in zip(after, state)) and torch.equal(kept_pool, pool)
        assert outputs[-2].tolist() == [0] and torch.isfinite(outputs[0]).all()
    _ok()


@gpu
def test_two_streams_at_once(cuda, native_lib):
    """Reserve with copies, compact and attention on two streams at the same time, each on its own state."""
    rng = np.random.default_rng(12)
    jobs = []
    for i in range(2):
        n, hkv, d, page, pages = 40, 4, 128, 32, 4600
        pool = torch.randint(0, 200, (pages, hkv, page // 16, 20 * d), device=cuda, dtype=torch.uint8)
        pool[..., 8 * d:10 * d] = 1  # scales and minima that are numbers
        pool[..., 18 * d:] = 1
        m = Pages(np.full((n, 60), -1), rng.integers(1, 1500, n), np.zeros(pages, int), page)
        order = list(rng.permutation(pages))
        for s in range(0, n, 2):
            for w in range(-(-m.lengths[s] // page)):
                m.table[s, w] = order.pop()
                m.refs[m.table[s, w]] = 1
            m.lengths[s + 1] = 0
        m.fork(range(0, n, 2), range(1, n, 2))
        q = torch.as_tensor(rng.standard_normal((n, 8, d))).to(cuda, BF16)
        jobs.append((pool, _three(m, cuda), q, torch.cuda.Stream()))

    def run(pool, state, q):
        p = pool.clone()
        table, refs, missing = dbl.relay_cache_reserve(p, *state, 40)
        table, refs, used = dbl.relay_cache_compact(p, table, refs)
        return [p, table, refs, missing, used, *dbl.relay_cache_attention(q, p, table, state[1])]

    want = [run(*job[:3]) for job in jobs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = [None, None]
        for i, (pool, state, q, stream) in enumerate(jobs):
            with torch.cuda.stream(stream):
                got[i] = run(pool, state, q)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    _ok()


