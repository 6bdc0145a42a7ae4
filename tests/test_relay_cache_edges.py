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


