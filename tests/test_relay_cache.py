"""The 4-bit relay cache: the format, the refusals and the host side on the CPU; every kernel against
the 64-bit models of relay_cache_model.py on the GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

import delta_block_lm_b200 as dbl
import relay_cache_model as M
from delta_block_lm_b200 import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------ CPU
def test_struct_layout_matches_header(tmp_path):
    structs = {"dbl_relay_cache": N.RelayCache, "dbl_relay_cache_append_args": N.RelayCacheAppendArgs,
               "dbl_relay_cache_read_args": N.RelayCacheReadArgs,
               "dbl_relay_cache_attention_args": N.RelayCacheAttentionArgs,
               "dbl_relay_cache_pages_args": N.RelayCachePagesArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>",
             f'#include "{os.path.join(ROOT, "include", "dbl_gdn2.h")}"', "int main(void) {"]
    want = []
    for name, py in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(py))
        for field, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(py, field).offset)
    lines.append("return 0; }")
    (tmp_path / "layout.c").write_text("\n".join(lines))
    subprocess.check_call(["gcc", "-std=c11", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "layout")], text=True).split()]
    assert got == want


def _random(rng, *shape):
    return torch.as_tensor(rng.standard_normal(shape), dtype=F32).bfloat16().double().numpy()


@pytest.mark.parametrize("d", [64, 128])
def test_model_error_is_half_a_step(d):
    rng = np.random.default_rng(d)
    x = rng.standard_normal((50, d)) * np.exp(rng.uniform(-20, 20, (50, 1))) + rng.standard_normal((50, 1))
    x = x.astype(np.float32)
    scale, low, code = M.quantise(x)
    assert code.min() >= 0 and code.max() <= 15
    err = np.abs(M.values(x) - x).reshape(50, -1, 32)
    assert (err <= scale[..., None] / 2).all()
    assert (low <= x.reshape(50, -1, 32).min(-1)).all()


def test_refusals_of_the_library(native_lib):
    """Every refusal comes back as a status before anything is launched (there is no GPU here)."""
    L = native_lib
    good = N.RelayCache(4, 2, 64, 16, 256)
    bad = [(N.RelayCache(0, 2, 64, 16, 256), N.DBL_ERR_INVALID_ARGUMENT, b"positive"),
           (N.RelayCache(4, 2, 96, 16, 256), N.DBL_ERR_UNSUPPORTED, b"head_dim"),
           (N.RelayCache(4, 2, 64, 24, 256), N.DBL_ERR_UNSUPPORTED, b"page_size"),
           (N.RelayCache(4, 2, 64, 16, None), N.DBL_ERR_INVALID_ARGUMENT, b"pool"),
           (N.RelayCache(4, 2, 64, 16, 264), N.DBL_ERR_INVALID_ARGUMENT, b"aligned"),
           (N.RelayCache(1 << 31, 2, 64, 16, 256), N.DBL_ERR_UNSUPPORTED, b"32-bit")]
    z = (0, 0, 0, 0)

    def refused(rc, status, text):
        assert rc == status and text in L.dbl_last_error(), L.dbl_last_error()

    for fn in ("append", "read", "attention", "release", "fork", "reserve", "compact", "copy_pages"):
        call = getattr(L, "dbl_relay_cache_" + fn)
        more = {"append": (), "read": (), "attention": (None, 0), "release": (None, 0), "fork": (None, None, 0),
                "reserve": (None, 1, None, None, 0), "compact": (None, None, 0), "copy_pages": (None, None, 0)}[fn]
        refused(call(None, *more, None), N.DBL_ERR_INVALID_ARGUMENT, b"null")
        for c, status, text in bad:
            a = {"append": lambda: N.RelayCacheAppendArgs(c, 1, 1, 1, 0, N.DBL_F32),
                 "read": lambda: N.RelayCacheReadArgs(c, 1, 1, 1, 0, N.DBL_F32),
                 "attention": lambda: N.RelayCacheAttentionArgs(c, 1, 1, 2, 1, 0, 0, 0, N.DBL_F32),
                 "copy_pages": lambda: c}.get(fn, lambda: N.RelayCachePagesArgs(c, 1, 1, 0))()
            refused(call(ctypes.byref(a), *more, None), status, text)

    ap = lambda *x, **k: L.dbl_relay_cache_append(ctypes.byref(N.RelayCacheAppendArgs(good, *x, **k)), None)  # noqa: E731
    refused(ap(0, 1, 1, 0, N.DBL_F32, page_table=256), N.DBL_ERR_INVALID_ARGUMENT, b"n_seq")
    refused(ap(1, 1, 4, 2, N.DBL_F32, page_table=256), N.DBL_ERR_INVALID_ARGUMENT, b"stride")
    refused(ap(1, 1, 1, 0, N.DBL_F32), N.DBL_ERR_INVALID_ARGUMENT, b"page_table")
    refused(ap(1, 0, 1, 0, N.DBL_F32, page_table=256), N.DBL_ERR_INVALID_ARGUMENT, b"tokens")
    refused(ap(1, 1, 1, 0, 7, page_table=256), N.DBL_ERR_INVALID_ARGUMENT, b"dtype")
    refused(ap(1, 1, 1, 0, N.DBL_F32, page_table=256, k=256), N.DBL_ERR_INVALID_ARGUMENT, b"required")
    refused(ap(1, 1, 1, 0, N.DBL_F32, 256, 256, (128, 128, 64, 2), z, 256, 256), N.DBL_ERR_INVALID_ARGUMENT, b"innermost")
    rd = lambda *x, **k: L.dbl_relay_cache_read(ctypes.byref(N.RelayCacheReadArgs(good, *x, **k)), None)  # noqa: E731
    refused(rd(1, 1, 1, 0, N.DBL_F32, 256, 256, None, 256, 264), N.DBL_ERR_INVALID_ARGUMENT, b"aligned")
    refused(rd(1, -1, 1, 0, N.DBL_F32, 256, 256, None, 256, 256), N.DBL_ERR_INVALID_ARGUMENT, b"tokens")

    def at(ws=None, size=0, **k):
        f = dict(n_seq=1, queries=1, heads=2, table_width=1, dtype=N.DBL_F32, scale=1.0, q=256, page_table=256,
                 lengths=256, out=256)
        return L.dbl_relay_cache_attention(ctypes.byref(N.RelayCacheAttentionArgs(cache=good, **{**f, **k})), ws, size, None)

    refused(at(heads=3), N.DBL_ERR_INVALID_ARGUMENT, b"multiple of kv_heads")
    refused(at(queries=0), N.DBL_ERR_INVALID_ARGUMENT, b"queries")
    refused(at(dtype=9), N.DBL_ERR_INVALID_ARGUMENT, b"dtype")
    refused(at(out=None), N.DBL_ERR_INVALID_ARGUMENT, b"required")
    refused(at(prefix_len=17, prefix_pages=256, prefix_width=1), N.DBL_ERR_INVALID_ARGUMENT, b"prefix_pages")
    refused(at(prefix_len=-1), N.DBL_ERR_INVALID_ARGUMENT, b"prefix_len")
    refused(at(q_stride=(128, 128, 64, 3)), N.DBL_ERR_INVALID_ARGUMENT, b"innermost")
    refused(at(n_seq=1 << 20, queries=1 << 12), N.DBL_ERR_UNSUPPORTED, b"32-bit")

    def pg(fn, *more, **k):
        f = dict(n_seq=2, table_width=1, page_table=256, lengths=256, refs=256, page_table_out=256, lengths_out=256,
                 refs_out=256)
        return getattr(L, "dbl_relay_cache_" + fn)(ctypes.byref(N.RelayCachePagesArgs(cache=good, **{**f, **k})), *more, None)

    need = L.dbl_relay_cache_pages_workspace_bytes(4, 2)
    assert need > 0 and L.dbl_relay_cache_pages_workspace_bytes(0, 2) == 0
    refused(pg("release", None, 1), N.DBL_ERR_INVALID_ARGUMENT, b"list")
    refused(pg("release", 256, 1, lengths_out=None), N.DBL_ERR_INVALID_ARGUMENT, b"lengths_out")
    refused(pg("fork", 256, None, 1), N.DBL_ERR_INVALID_ARGUMENT, b"lists")
    refused(pg("fork", 256, 256, 1, refs=None), N.DBL_ERR_INVALID_ARGUMENT, b"required")
    refused(pg("reserve", None, 1, None, 256, need), N.DBL_ERR_INVALID_ARGUMENT, b"missing")
    refused(pg("reserve", None, -1, 256, 256, need), N.DBL_ERR_INVALID_ARGUMENT, b"tokens")
    refused(pg("reserve", None, 1, 256, 256, need - 1), N.DBL_ERR_WORKSPACE, b"workspace")
    refused(pg("reserve", None, 1, 256, 260, need), N.DBL_ERR_INVALID_ARGUMENT, b"aligned")
    refused(pg("compact", 256, None, need), N.DBL_ERR_WORKSPACE, b"workspace")
    refused(pg("compact", None, 256, need), N.DBL_ERR_INVALID_ARGUMENT, b"used")
    refused(L.dbl_relay_cache_copy_pages(ctypes.byref(good), None, None, 1, None), N.DBL_ERR_INVALID_ARGUMENT, b"lists")


def test_no_cpu_fallback_and_pool_shapes():
    pool = dbl.relay_cache_pool(2, 1, 64, 16, device="cpu")
    assert tuple(pool.shape) == (2, 1, 1, 1280) and pool.dtype == torch.uint8
    with pytest.raises(ValueError, match="head_dim"):
        dbl.relay_cache_pool(2, 1, 96, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        dbl.relay_cache_pool(2, 1, 64, 20, device="cpu")
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU fallback"):
        dbl.relay_cache_append(pool, table, lens, torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, 1, 64))
    with pytest.raises(ValueError, match="no CPU fallback"):
        dbl.relay_cache_attention(torch.zeros(1, 1, 64), pool, table, lens)


# ------------------------------------------------------------------------------------------ GPU helpers
def _i32(x, dev):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=dev)


def _ok():
    code = ctypes.c_int(0)
    assert N.lib().dbl_device_error(ctypes.byref(code)) == N.DBL_OK, code.value


def _device_code():
    code = ctypes.c_int(0)
    N.lib().dbl_device_error(ctypes.byref(code))
    return code.value


def _tables(rng, lens, page, extra=0, width=None):
    """A table of distinct random pages for sequences of `lens` tokens, and how many pages it names."""
    need = [-(-n // page) for n in lens]
    width = width or max(1, max(need))
    total = sum(need) + extra
    order = rng.permutation(total)
    table = np.full((len(lens), width), -1)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table, max(1, total), order[at:]


def _fill(dev, rng, lens, hkv, d, page, dtype=BF16, garbage=True, extra=0):
    """A pool holding random tokens; the values it holds by the model; bytes never written are 0xFF
    (NaN as scales)."""
    table, pages, _ = _tables(rng, lens, page, extra)
    pool = dbl.relay_cache_pool(pages, hkv, d, page, device=dev)
    if garbage:
        pool.fill_(255)
    t = max(1, max(lens))
    off = 2 * rng.standard_normal((1, 1, hkv, d))
    k = torch.as_tensor(rng.standard_normal((len(lens), t, hkv, d)) + off).to(dev, dtype)
    v = torch.as_tensor(rng.standard_normal((len(lens), t, hkv, d))).to(dev, dtype)
    tab = _i32(table, dev)
    got = dbl.relay_cache_append(pool, tab, _i32([0] * len(lens), dev), k, v, counts=_i32(lens, dev))
    assert got.tolist() == list(lens)
    kk = [M.values(k[i, :n].double().cpu().numpy()) for i, n in enumerate(lens)]
    vv = [M.values(v[i, :n].double().cpu().numpy()) for i, n in enumerate(lens)]
    return pool, tab, got, kk, vv


# ------------------------------------------------------------------------------------------ append and read
@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,page,h", [(64, 16, 3), (128, 16, 1), (128, 64, 2), (64, 48, 5)])
def test_append_bytes_and_read(cuda, native_lib, dtype, d, page, h):
    """Ragged prompts, then single tokens, then a run that starts inside a tile: every byte of the
    pages against the model (bf16 inputs: f32 arithmetic decides as 64 bits do, up to exponent gaps
    that this range of inputs does not have; f32 inputs are rounded to 12 bits for the same reason),
    bytes of tokens not written keep what was there."""
    rng = np.random.default_rng(page + d)
    lens = [0, 1, 16, 17, 33, 100]
    runs = [[0, 1, 16, 15, 31, 40], [0, 0, 0, 1, 1, 1], [0, 0, 0, 1, 1, 59]]
    table, pages, _ = _tables(rng, lens, page)
    tab = _i32(table, cuda)
    pool = dbl.relay_cache_pool(pages, h, d, page, device=cuda)
    pool.random_(0, 256, generator=torch.Generator(device=cuda).manual_seed(3))
    want = pool.cpu().numpy().copy()
    at = np.zeros(len(lens), int)
    dense = [[], []]
    for counts in runs:
        t = max(counts) + 2  # two tokens of padding
        x = [rng.standard_normal((len(lens), t, h, d)) * np.exp(rng.uniform(-3, 3, (len(lens), t, h, 1))) for _ in "kv"]
        x = [torch.as_tensor(a).to(F32) for a in x]
        x = [a.bfloat16() if dtype == BF16 else (a.view(torch.int32) & ~0xFFF).view(F32) for a in x]
        new = dbl.relay_cache_append(pool, tab, _i32(at, cuda), x[0].to(cuda), x[1].to(cuda), counts=_i32(counts, cuda))
        for i, c in enumerate(counts):
            for j in range(c):
                pos = at[i] + j
                for a in range(h):
                    tile = want[table[i, pos // page], a, pos % page // 16]
                    M.pack_token(tile, pos % 16, "k", x[0][i, j, a].double().numpy())
                    M.pack_token(tile, pos % 16, "v", x[1][i, j, a].double().numpy())
        dense[0].append([x[0][i, :c].double().numpy() for i, c in enumerate(counts)])
        dense[1].append([x[1][i, :c].double().numpy() for i, c in enumerate(counts)])
        at += counts
        assert new.tolist() == list(at)
    assert list(at) == lens
    assert (pool.cpu().numpy() == want).all()
    # read back, from inside and past the end
    start = [0, 0, 3, 5, 16, 33]
    for out in (F32, BF16):
        k, v = dbl.relay_cache_read(pool, tab, _i32(lens, cuda), start=_i32(start, cuda), tokens=70, dtype=out)
        for got, xs in ((k, dense[0]), (v, dense[1])):
            got = got.float().cpu()
            for i, n in enumerate(lens):
                e = np.zeros((70, h, d))
                whole = M.values(np.concatenate([r[i] for r in xs]).reshape(-1, h, d))
                part = whole[start[i]:start[i] + 70]
                e[:len(part)] = part
                e = torch.as_tensor(e).float()  # one rounding
                assert torch.equal(got[i], e.to(out).float()), (i, out)
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_strided_views_and_alignment(cuda, native_lib, dtype):
    """k and v as slices of one fused projection, transposed storage, and rows that do not start on 16 bytes."""
    rng = np.random.default_rng(5)
    n, t, h, d, page = 2, 19, 3, 64, 32
    table, pages, _ = _tables(rng, [t] * n, page)
    tab, zero = _i32(table, cuda), _i32([0] * n, cuda)
    x = torch.as_tensor(rng.standard_normal((n, t, 2 * h * d + 1))).to(cuda, dtype)
    views = [(x[..., :h * d].unflatten(-1, (h, d)), x[..., h * d:2 * h * d].unflatten(-1, (h, d))),
             (x[..., 1:h * d + 1].unflatten(-1, (h, d)), x[..., h * d + 1:].unflatten(-1, (h, d)))]
    y = torch.as_tensor(rng.standard_normal((2, h, n, t, d))).to(cuda, dtype).permute(0, 2, 3, 1, 4)
    views.append((y[0], y[1]))
    z = torch.as_tensor(rng.standard_normal((2, n, t, d, h))).to(cuda, dtype).transpose(3, 4)
    views.append((z[0], z[1]))  # the innermost stride is not 1
    for k, v in views:
        pools = [dbl.relay_cache_pool(pages, h, d, page, device=cuda) for _ in "ab"]
        dbl.relay_cache_append(pools[0], tab, zero, k, v)
        dbl.relay_cache_append(pools[1], tab, zero, k.contiguous(), v.contiguous())
        assert torch.equal(*pools)
        assert pools[0].any()
    _ok()


@gpu
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F32, 64)])
def test_append_few_tokens_inside_a_tile(cuda, native_lib, dtype, d):
    """Calls of 1 to 40 tokens that begin inside a tile, with k and v at the very end of their memory: no lane may
    read past the call's own tokens, and what is written is what one token at a time writes."""
    rng = np.random.default_rng(6)
    h, page = 5, 16
    for t in (1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 40):
        start = [0, 5, 15]
        table, pages, _ = _tables(rng, [s + t for s in start], page)
        tab = _i32(table, cuda)
        store = torch.empty((2, 3, t, h, d), device=cuda, dtype=dtype)  # v ends where the memory does
        store.copy_(torch.as_tensor(rng.standard_normal(store.shape)))
        pools = [dbl.relay_cache_pool(pages, h, d, page, device=cuda) for _ in "ab"]
        new = dbl.relay_cache_append(pools[0], tab, _i32(start, cuda), store[0], store[1])
        assert new.tolist() == [s + t for s in start]
        for i in range(t):
            dbl.relay_cache_append(pools[1], tab, _i32([s + i for s in start], cuda), store[0, :, i:i + 1], store[1, :, i:i + 1])
        assert torch.equal(*pools), t
    _ok()


@gpu
def test_append_special_values(cuda, native_lib):
    """Constants, a range below 2^-100, the largest values, and groups that hold an infinity or NaN: those
    become NaN, the other groups of the token are untouched."""
    d, h = 128, 1
    rng = np.random.default_rng(1)
    x = torch.as_tensor(rng.standard_normal((1, 9, h, d)), dtype=F32).bfloat16().float()
    x[0, 0, 0, :32] = 1.5
    x[0, 1, 0, :32] = -0.0
    x[0, 2, 0, :32] = torch.linspace(0, 1, 32).bfloat16().float() * 2.0 ** -110
    x[0, 3, 0, 5] = float("nan")
    x[0, 4, 0, 37] = float("inf")
    x[0, 5, 0, 70] = -float("inf")
    x[0, 6, 0, 100] = float("inf")
    x[0, 6, 0, 101] = -float("inf")
    x[0, 7, 0, :32] = torch.as_tensor([3.0e38, -3.0e38] * 16)  # the range leaves f32
    x[0, 8, 0, :32] = torch.as_tensor([1.5e38, -1.5e38] * 16)
    e = M.values(x.double().numpy())
    pool = dbl.relay_cache_pool(1, h, d, 16, device=cuda)
    tab = _i32([[0]], cuda)
    new = dbl.relay_cache_append(pool, tab, _i32([0], cuda), x.to(cuda), x.to(cuda))
    for got in dbl.relay_cache_read(pool, tab, new, tokens=9, dtype=F32):
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(e))
        ok = ~np.isnan(e)
        assert np.array_equal(got[ok], e[ok].astype(np.float32).astype(np.float64))
    nan = np.isnan(e).reshape(9, 4, 32)
    assert nan.all(-1).sum() == 5 and nan.any(-1).sum() == 5
    _ok()


# ------------------------------------------------------------------------------------------ attention
U32, UBF = 2.0 ** -23, 2.0 ** -7  # spacing of f32 (sums that may truncate) and of bf16


def _check_attention(got, want, dtype, d, keys):
    """Error bounds, element by element.  A score is a sum of d products in f32 (their partial sums and the
    groups' minima: 2 d roundings), p follows it by exp (2 units more); o adds the rounding of p to f16
    (2^-11; two parts, 2^-22, for f32), sums over the keys, and of the output."""
    o, mx, sm = (x.double().cpu().numpy() for x in got)
    eo, em, es, size, mass = want
    ds = (2 * d + 8) * U32 * mass + 4 * U32
    assert (np.abs(mx - em) <= ds + U32 * np.abs(em)).all()
    tail = np.sqrt(keys) * 4 * U32
    assert (np.abs(sm - es) <= es * (2 * ds + tail) + U32).all()
    dp = 2.0 ** -11 if dtype == BF16 else 2.0 ** -22
    tol = size * (2 * ds + tail + dp)[..., None] + np.abs(eo) * (UBF / 2 if dtype == BF16 else U32)
    assert np.isfinite(o).all()
    assert (np.abs(o - eo) <= tol + 1e-30).all(), float((np.abs(o - eo) / (tol + 1e-30)).max())


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hkv,group,tq,d,page,lens", [
    (1, 1, 1, 64, 16, [1]), (2, 1, 1, 128, 16, [37]), (3, 1, 1, 128, 64, [0, 1, 15, 16, 17, 63, 64, 65, 300]),
    (2, 4, 1, 64, 32, [5, 0, 200, 129]), (1, 7, 1, 128, 48, [400, 31]), (2, 8, 1, 128, 64, [513, 1]),
    (1, 16, 1, 64, 64, [100, 77]), (1, 40, 1, 128, 16, [90, 3]), (2, 1, 5, 128, 16, [5, 3, 0, 64, 130]),
    (1, 3, 9, 64, 64, [9, 200, 1]), (1, 2, 40, 128, 32, [40, 70, 1]), (1, 1, 1, 64, 128, [2500]),
    (1, 1, 1, 128, 64, [4097, 2])])
@pytest.mark.parametrize("prefix", [0, 1, 77])
def test_attention(cuda, native_lib, dtype, hkv, group, tq, d, page, lens, prefix):
    rng = np.random.default_rng(len(lens) + d + tq + prefix)
    rows = [prefix] + list(lens)  # the prefix is a sequence of its own
    pool, tab, held, kk, vv = _fill(cuda, rng, rows, hkv, d, page)
    q = torch.as_tensor(rng.standard_normal((len(lens), tq, hkv * group, d))).to(cuda, dtype)
    pre = (kk[0], vv[0]) if prefix else (None, None)
    want = M.attention(q.double().cpu().numpy(), kk[1:], vv[1:], lens, *pre)
    got = dbl.relay_cache_attention(q if tq > 1 else q[:, 0], pool, tab[1:], held[1:],
                                    prefix_pages=tab[0] if prefix else None, prefix_len=prefix)
    if tq == 1:
        got = [x[:, None] for x in got]
    _check_attention(got, want, dtype, d, max(lens) + prefix + 1)
    empty = np.array([[prefix == 0 and n - tq + t + 1 <= 0 for t in range(tq)] for n in lens])
    assert (got[0].float().cpu().numpy()[empty] == 0).all()
    assert (got[1].cpu().numpy()[empty] == 0).all() and (got[2].cpu().numpy()[empty] == 1).all()
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_many_sequences_share_a_prefix(cuda, native_lib, dtype):
    rng = np.random.default_rng(11)
    n, hkv, d, page, prefix = 37, 2, 128, 64, 700
    lens = [int(x) for x in rng.integers(0, 150, n)]
    pool, tab, held, kk, vv = _fill(cuda, rng, [prefix] + lens, hkv, d, page)
    q = torch.as_tensor(rng.standard_normal((n, hkv, d))).to(cuda, dtype)
    want = M.attention(q[:, None].double().cpu().numpy(), kk[1:], vv[1:], lens, kk[0], vv[0])
    got = dbl.relay_cache_attention(q, pool, tab[1:], held[1:], prefix_pages=tab[0], prefix_len=prefix)
    _check_attention([x[:, None] for x in got], want, dtype, d, 900)
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,hkv,group,tq,d,page,prefix", [(64, 2, 1, 1, 128, 64, 4200), (40, 4, 2, 3, 64, 48, 3300),
                                                          (5, 1, 1, 1, 64, 16, 104900), (33, 2, 9, 1, 128, 32, 8001)])
def test_attention_long_shared_prefix(cuda, native_lib, dtype, n, hkv, group, tq, d, page, prefix):
    """Prefixes with a launch of their own: sequences x kv heads x tokens of at least 2^19."""
    rng = np.random.default_rng(n)
    assert n * hkv * prefix >= 1 << 19
    lens = [int(x) for x in rng.integers(0, 200, n)]
    lens[0], lens[-1] = 0, tq
    pool, tab, held, kk, vv = _fill(cuda, rng, [prefix] + lens, hkv, d, page)
    q = torch.as_tensor(rng.standard_normal((n, tq, hkv * group, d))).to(cuda, dtype)
    want = M.attention(q.double().cpu().numpy(), kk[1:], vv[1:], lens, kk[0], vv[0])
    call = lambda: dbl.relay_cache_attention(q, pool, tab[1:], held[1:], prefix_pages=tab[0], prefix_len=prefix)  # noqa: E731
    got = call()
    _check_attention(got, want, dtype, d, prefix + 200)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got, call()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = call()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_scales_of_all_sizes(cuda, native_lib, dtype):
    """Queries and values far from 1 in size, rows of q that differ by many powers of two, tokens whose value
    scales differ, one all-zero query, constant value groups."""
    rng = np.random.default_rng(3)
    n, hkv, g, d, page, t = 2, 2, 3, 64, 16, 90
    table, pages, _ = _tables(rng, [t] * n, page)
    tab = _i32(table, cuda)
    k = rng.standard_normal((n, t, hkv, d)) * 1e-3
    v = rng.standard_normal((n, t, hkv, d)) * np.exp(rng.uniform(-8, 8, (n, t, 1, 1))) * 1e6
    v[0, 10:20, :, :32] = 7.0
    k, v = (torch.as_tensor(x).to(cuda, BF16) for x in (k, v))
    pool = dbl.relay_cache_pool(pages, hkv, d, page, device=cuda)
    held = dbl.relay_cache_append(pool, tab, _i32([0] * n, cuda), k, v)
    q = rng.standard_normal((n, hkv * g, d)) * 10.0 ** rng.integers(-6, 5, (n, hkv * g, 1))
    q[1, 2] = 0
    q = torch.as_tensor(q).to(cuda, dtype)
    kk, vv = ([M.values(x[i].double().cpu().numpy()) for i in range(n)] for x in (k, v))
    want = M.attention(q[:, None].double().cpu().numpy(), kk, vv, [t] * n)
    got = dbl.relay_cache_attention(q, pool, tab, held)
    _check_attention([x[:, None] for x in got], want, dtype, d, t)
    # every score below the type's smallest exponent range: the softmax is of differences
    q2 = q * 0 + 1e4
    want = M.attention(q2[:, None].double().cpu().numpy(), kk, vv, [t] * n, scale=-100.0)
    got = dbl.relay_cache_attention(q2, pool, tab, held, scale=-100.0)
    o, mx, _ = (x.double().cpu().numpy() for x in got)
    assert np.isfinite(o).all() and np.allclose(mx, want[1][:, 0], rtol=1e-4)
    _ok()


@gpu
def test_attention_nan_stays_where_it_is_read(cuda, native_lib):
    """A NaN key spoils its sequence's rows of that head only, a NaN value group its 32 channels only; a NaN
    query its own row only."""
    rng = np.random.default_rng(9)
    n, hkv, g, d, page, t = 3, 2, 2, 128, 16, 40
    table, pages, _ = _tables(rng, [t] * n, page)
    tab = _i32(table, cuda)
    k, v = (torch.as_tensor(rng.standard_normal((n, t, hkv, d)), dtype=F32) for _ in "kv")
    k[0, 33, 1, 70] = float("nan")
    v[1, 5, 0, 40] = float("inf")
    q = torch.as_tensor(rng.standard_normal((n, hkv * g, d)), dtype=F32)
    q[2, 3, 0] = float("nan")
    pool = dbl.relay_cache_pool(pages, hkv, d, page, device=cuda)
    held = dbl.relay_cache_append(pool, tab, _i32([0] * n, cuda), k.to(cuda), v.to(cuda))
    for dtype in (F32, BF16):
        o, mx, sm = dbl.relay_cache_attention(q.to(cuda, dtype), pool, tab, held)
        bad = torch.isnan(o).cpu().numpy()
        want = np.zeros_like(bad)
        want[0, 2:4] = True
        want[1, 0:2, 32:64] = True
        want[2, 3] = True
        assert np.array_equal(bad, want)
        assert np.array_equal(torch.isnan(sm).cpu().numpy(), want.all(-1))
    _ok()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tq,g,d,t,prefix", [(3, 1, 64, 2, 0), (4, 2, 128, 33, 0), (5, 1, 128, 130, 21), (3, 8, 64, 300, 0),
                                             (17, 1, 128, 16, 0)])
def test_attention_nan_of_later_tokens(cuda, native_lib, dtype, tq, g, d, t, prefix):
    """What a query does not see yet does not reach it: NaN keys and values of the last two drafted tokens leave the
    rows before them right, and the rows that see such a token get its NaN where they read it."""
    rng = np.random.default_rng(tq * t)
    lens, hkv = [t, t], 2
    pool, tab, held, kk, vv = _fill(cuda, rng, [prefix] + lens, hkv, d, 16)
    q = torch.as_tensor(rng.standard_normal((2, tq, hkv * g, d))).to(cuda, dtype)
    pre = (kk[0], vv[0]) if prefix else (None, None)
    want = M.attention(q.double().cpu().numpy(), kk[1:], vv[1:], lens, *pre)
    # the last two tokens once more: the last value of (0, head 1), the one before it, the last key of (1, head 0)
    k, v = (torch.as_tensor(rng.standard_normal((2, 2, hkv, d)), dtype=F32) for _ in "kv")
    v[0, 1, 1, 40] = float("inf")
    v[0, 0, 1, 3] = float("nan")
    k[1, 1, 0, 5] = float("nan")
    dbl.relay_cache_append(pool, tab[1:], held[1:] - 2, k.to(cuda), v.to(cuda))
    kw = dict(prefix_pages=tab[0], prefix_len=prefix) if prefix else {}
    got = dbl.relay_cache_attention(q, pool, tab[1:], held[1:], **kw)
    nan = torch.zeros_like(got[0], dtype=torch.bool)
    nan[0, -1, g:, 32:64] = True
    nan[0, -2:, g:, :32] = True
    nan[1, -1, :g] = True
    assert torch.equal(torch.isnan(got[0]), nan)
    none = torch.zeros_like(got[2], dtype=torch.bool)
    none[1, -1, :g] = True
    assert torch.equal(torch.isnan(got[2]), none)
    _check_attention([x[:, :-2] for x in got], [x[:, :-2] for x in want], dtype, d, t + prefix)
    _ok()


@gpu
def test_attention_repeats_streams_strides_and_graphs(cuda, native_lib):
    """The same bits from call to call, with one workspace, on a side stream, from a strided q, in a graph."""
    rng = np.random.default_rng(21)
    lens = [1000, 3, 0, 517]
    pool, tab, held, _, _ = _fill(cuda, rng, [300] + lens, 2, 128, 64)
    base = torch.as_tensor(rng.standard_normal((4, 3, 8, 128))).to(cuda, BF16)
    q = base[:, 1]  # a slice: rows of one sequence are contiguous, sequences are not
    call = lambda **kw: dbl.relay_cache_attention(q, pool, tab[1:], held[1:], prefix_pages=tab[0], prefix_len=300, **kw)  # noqa: E731
    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))
    assert all(torch.equal(a, b) for a, b in zip(first, dbl.relay_cache_attention(
        q.contiguous(), pool, tab[1:], held[1:], prefix_pages=tab[0], prefix_len=300)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, got))
    _ok()


@gpu
def test_offsets_past_32_bits(cuda, native_lib):
    """A pool of over 4 GB: pages at its end."""
    rng = np.random.default_rng(2)
    h, d, page = 16, 128, 64
    per = h * (page // 16) * 20 * d
    pages = (1 << 32) // per + 40
    pool = torch.empty((pages, h, page // 16, 20 * d), device=cuda, dtype=torch.uint8)
    tab = _i32([[pages - 1, 3, pages - 2]], cuda)
    k, v = (torch.as_tensor(rng.standard_normal((1, 150, h, d))).to(cuda, BF16) for _ in "kv")
    held = dbl.relay_cache_append(pool, tab, _i32([0], cuda), k, v)
    kk, vv = (M.values(x[0].double().cpu().numpy()) for x in (k, v))
    gk, gv = dbl.relay_cache_read(pool, tab, held, tokens=150, dtype=F32)
    assert np.array_equal(gk[0].double().cpu().numpy(), kk.astype(np.float32)) and np.array_equal(
        gv[0].double().cpu().numpy(), vv.astype(np.float32))
    q = torch.as_tensor(rng.standard_normal((1, h, d))).to(cuda, BF16)
    want = M.attention(q[:, None].double().cpu().numpy(), [kk], [vv], [150])
    _check_attention([x[:, None] for x in dbl.relay_cache_attention(q, pool, tab, held)], want, BF16, d, 150)
    dbl.relay_cache_copy_pages(pool, _i32([pages - 1], cuda), _i32([0], cuda))
    assert torch.equal(pool[0], pool[pages - 1])
    _ok()


@gpu
def test_missing_pages_are_recorded_and_left_out(cuda, native_lib):
    """Entries outside the pool (-1, too large) and tokens past the table: nothing outside the pool is touched, the
    tokens are left out, and the device error says so."""
    rng = np.random.default_rng(4)
    pool, tab, held, kk, vv = _fill(cuda, rng, [64, 64], 1, 64, 16, extra=1)
    _ok()
    bad = tab.clone()
    bad[0, 1], bad[1, 2] = -1, len(pool) + 5
    q = torch.as_tensor(rng.standard_normal((2, 1, 64))).to(cuda, F32)
    got = dbl.relay_cache_attention(q, pool, bad, held)
    assert _device_code() == 102
    keep = [np.r_[0:16, 32:64], np.r_[0:32, 48:64]]
    want = M.attention(q[:, None].double().cpu().numpy(), [x[i] for x, i in zip(kk, keep)],
                       [x[i] for x, i in zip(vv, keep)], [48, 48])
    _check_attention([x[:, None] for x in got], want, F32, 64, 64)
    k, _ = dbl.relay_cache_read(pool, bad, held, tokens=64, dtype=F32)
    assert _device_code() == 102 and not k[0, 16:32].any() and not k[1, 32:48].any() and k[0, 32:].any()
    before = pool.clone()
    x = torch.ones((2, 3, 1, 64), device=cuda)
    dbl.relay_cache_append(pool, bad, _i32([17, 63], cuda), x, x)
    assert _device_code() == 102
    changed = (pool != before).flatten(1).any(1).nonzero().flatten().tolist()
    assert changed == [int(tab[1, 3])]
    _ok()


def test_argument_checks(cuda):
    pool = dbl.relay_cache_pool(4, 2, 64, 16, device=cuda)
    tab, lens, refs = _i32([[0, 1]], cuda), _i32([3], cuda), _i32([1, 1, 0, 0], cuda)
    kv = torch.zeros((1, 1, 2, 64), device=cuda)
    with pytest.raises(ValueError, match="pool must be"):
        dbl.relay_cache_append(pool[:, :1], tab, lens, kv, kv)
    with pytest.raises(ValueError, match="k and v"):
        dbl.relay_cache_append(pool, tab, lens, kv[..., :32], kv[..., :32])
    with pytest.raises(ValueError, match="dtype of k"):
        dbl.relay_cache_append(pool, tab, lens, kv, kv.bfloat16())
    with pytest.raises(ValueError, match="lengths"):
        dbl.relay_cache_append(pool, tab, _i32([1, 2], cuda), kv, kv)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        dbl.relay_cache_attention(kv[:, 0].half(), pool, tab, lens)
    with pytest.raises(ValueError, match="page_table"):
        dbl.relay_cache_attention(kv[:, 0].expand(2, 2, 64), pool, tab, lens)
    with pytest.raises(ValueError, match="prefix_pages"):
        dbl.relay_cache_attention(kv[:, 0], pool, tab, lens, prefix_len=4)
    with pytest.raises(N.DblError, match="prefix_pages"):
        dbl.relay_cache_attention(kv[:, 0], pool, tab, lens, prefix_pages=_i32([0], cuda), prefix_len=17)
    with pytest.raises(N.DblError, match="multiple of kv_heads"):
        dbl.relay_cache_attention(torch.zeros((1, 3, 64), device=cuda), pool, tab, lens)
    with pytest.raises(ValueError, match="same length"):
        dbl.relay_cache_fork(pool, tab, lens, refs, _i32([0], cuda), _i32([0, 0], cuda))
    with pytest.raises(ValueError, match="out must be"):
        dbl.relay_cache_compact(pool, tab, refs, out=(tab.long(), refs))
    with pytest.raises(ValueError, match="list"):
        dbl.relay_cache_release(pool, tab, lens, refs, tab)


test_argument_checks = gpu(test_argument_checks)


# ------------------------------------------------------------------------------------------ pages
def _state(rng, rows, width, page, pages, live, longest):
    """A random consistent state: some sequences live, some forked from others, some reserved ahead."""
    m = M.Pages(np.full((rows, width), -1), np.zeros(rows, int), np.zeros(pages, int), page)
    free = list(rng.permutation(pages))
    for s in range(live):
        n = int(rng.integers(0, longest + 1))
        held = -(-n // page)
        ahead = int(rng.integers(0, 2))
        for w in range(min(width, held + ahead)):
            if not free:
                break
            m.table[s, w] = free.pop()
            m.refs[m.table[s, w]] = 1
        m.lengths[s] = min(n, int((m.table[s] >= 0).sum()) * page)
    return m


def _three(m, dev):
    return [_i32(x, dev) for x in (m.table, m.lengths, m.refs)]


def _same(got, m, what=3):
    want = [m.table, m.lengths, m.refs] if what == 3 else [m.table, m.refs]
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)


@gpu
@pytest.mark.parametrize("rows,width,page,pages,h,d", [(1, 1, 16, 1, 1, 64), (5, 4, 16, 30, 2, 64), (40, 9, 64, 260, 1, 128),
                                                       (300, 40, 32, 9000, 1, 64), (9, 3, 48, 8300, 1, 64)])
@pytest.mark.parametrize("inplace", [False, True])
def test_page_operations(cuda, native_lib, rows, width, page, pages, h, d, inplace):
    """Rounds of release, fork, reserve and compact on random states against the sequential model: the page table,
    lengths, reference counts, the number returned, and every byte of the pool."""
    rng = np.random.default_rng(rows * 7 + pages)
    m = _state(rng, rows, width, page, pages, max(1, rows // 2), width * page * 3 // 4)
    pool = torch.randint(0, 256, (pages, h, page // 16, 20 * d), device=cuda, dtype=torch.uint8)
    state = _three(m, cuda)
    for turn in range(4):
        gone = [int(s) for s in rng.permutation(rows)[:rng.integers(0, rows // 3 + 1)]]
        before = [t.clone() for t in state]
        keep = list(state)
        state = list(dbl.relay_cache_release(pool, *state, _i32(gone + gone[:1], cuda), out=state if inplace else None))
        m.release(gone)
        _same(state, m)
        assert inplace or all(torch.equal(a, b) for a, b in zip(before, keep))
        empty = [s for s in range(rows) if m.lengths[s] == 0 and (m.table[s] < 0).all()]
        full = [s for s in range(rows) if m.lengths[s] > 0]
        n = int(rng.integers(0, len(empty) + 1)) if full else 0
        children = [int(s) for s in rng.permutation(empty)[:n]]
        parents = [int(s) for s in rng.choice(full, n)] if n else []
        state = list(dbl.relay_cache_fork(pool, *state, _i32(parents, cuda), _i32(children, cuda),
                                          out=state if inplace else None))
        m.fork(parents, children)
        _same(state, m)
        counts = [int(rng.integers(0, 2 * page)) if rng.random() < 0.7 else 0 for _ in range(rows)]
        counts = [min(c, width * page - int(m.lengths[s])) for s, c in enumerate(counts)]
        old = pool.cpu().numpy().copy()
        table, refs, missing = dbl.relay_cache_reserve(pool, *state, _i32(counts, cuda),
                                                       out=(state[0], state[2]) if inplace else None)
        short = m.reserve(counts)
        assert missing.tolist() == [short]
        state = [table, state[1], refs]
        _same(state, m)
        assert np.array_equal(pool.cpu().numpy(), m.apply(old) if not short else old)
        old = pool.cpu().numpy().copy()
        table, refs, used = dbl.relay_cache_compact(pool, state[0], state[2], out=(state[0], state[2]) if inplace else None)
        assert used.tolist() == [m.compact()]
        state = [table, state[1], refs]
        _same(state, m)
        assert np.array_equal(pool.cpu().numpy(), m.apply(old))
    _ok()


@gpu
def test_reserve_copy_on_write_and_shortage(cuda, native_lib):
    page = 16
    m = M.Pages([[4, 2, -1], [-1] * 3, [-1] * 3, [-1] * 3], [20, 0, 0, 0], [0, 0, 1, 0, 1, 0], page)
    pool = torch.randint(0, 256, (6, 2, 1, 1280), device=cuda, dtype=torch.uint8)
    state = list(dbl.relay_cache_fork(pool, *_three(m, cuda), _i32([0, 0, 0], cuda), _i32([1, 2, 3], cuda)))
    m.fork([0, 0, 0], [1, 2, 3])
    _same(state, m)
    # all four holders of page 2 write: three copies, the last keeps it
    before = pool.clone()
    table, refs, missing = dbl.relay_cache_reserve(pool, *state, 1)
    assert missing.tolist() == [0] and table.tolist() == [[4, 0, -1], [4, 1, -1], [4, 3, -1], [4, 2, -1]]
    assert refs.tolist() == [1, 1, 1, 1, 4, 0]
    assert all(torch.equal(pool[p], before[2]) for p in (0, 1, 3)) and torch.equal(pool[5], before[5])
    # 13 tokens each need three copies and four more pages: 7 of 4 free, and nothing changes
    before = pool.clone()
    t2, r2, missing = dbl.relay_cache_reserve(pool, *state, 13)
    assert missing.tolist() == [3] and torch.equal(t2, state[0]) and torch.equal(r2, state[2]) and torch.equal(pool, before)
    # only two of the four write: both copy, the others keep it
    t3, r3, missing = dbl.relay_cache_reserve(pool, *state, _i32([1, 0, 1, 0], cuda))
    assert missing.tolist() == [0] and t3.tolist() == [[4, 0, -1], [4, 2, -1], [4, 1, -1], [4, 2, -1]]
    assert r3.tolist() == [1, 1, 2, 0, 4, 0]
    _ok()
    # a table without room for the tokens is recorded
    dbl.relay_cache_reserve(pool, *state, 40)
    assert _device_code() == 102


@gpu
def test_a_serving_loop(cuda, native_lib):
    """Prompt, fork, decode with copy on write, release, compact: the attention of every step against the model on
    each sequence's own history, in one CUDA stream without a host synchronisation between the calls."""
    rng = np.random.default_rng(8)
    hkv, g, d, page, rows, width, pages, prefix = 2, 2, 64, 16, 5, 8, 64, 21
    pool = dbl.relay_cache_pool(pages, hkv, d, page, device=cuda)
    pool.fill_(255)
    table = torch.full((rows + 1, width), -1, device=cuda, dtype=torch.int32)
    lengths, refs = torch.zeros(rows + 1, device=cuda, dtype=torch.int32), torch.zeros(pages, device=cuda, dtype=torch.int32)
    history = [[[], []] for _ in range(rows + 1)]

    def write(counts):
        nonlocal table, lengths, refs
        t = max(counts)
        table, refs, missing = dbl.relay_cache_reserve(pool, table, lengths, refs, _i32(counts, cuda))
        k, v = (torch.as_tensor(rng.standard_normal((rows + 1, t, hkv, d))).to(cuda, BF16) for _ in "kv")
        lengths = dbl.relay_cache_append(pool, table, lengths, k, v, counts=_i32(counts, cuda))
        for i, c in enumerate(counts):
            for at, x in ((0, k), (1, v)):
                history[i][at] = history[i][at] + [M.values(y) for y in x[i, :c].double().cpu().numpy()]
        assert missing.tolist() == [0]

    def attend():
        q = torch.as_tensor(rng.standard_normal((rows, hkv * g, d))).to(cuda, BF16)
        lens = lengths.tolist()
        as_array = lambda x: np.asarray(x).reshape(-1, hkv, d)  # noqa: E731
        want = M.attention(q[:, None].double().cpu().numpy(), [as_array(history[i][0]) for i in range(rows)],
                           [as_array(history[i][1]) for i in range(rows)], lens[:rows], as_array(history[rows][0]),
                           as_array(history[rows][1]))
        got = dbl.relay_cache_attention(q, pool, table[:rows], lengths[:rows], prefix_pages=table[rows], prefix_len=prefix)
        _check_attention([x[:, None] for x in got], want, BF16, d, 200)

    write([19, 0, 33, 0, 0, prefix])  # two prompts and the shared prefix (the last row)
    attend()
    table, lengths, refs = dbl.relay_cache_fork(pool, table, lengths, refs, _i32([0, 0, 2], cuda), _i32([1, 3, 4], cuda))
    for a, b in ((0, 1), (0, 3), (2, 4)):
        history[b] = [list(x) for x in history[a]]
    attend()
    for step in range(18):
        write([1, 1, 1, 1, 1, 0])
        attend()
        if step == 9:
            table, lengths, refs = dbl.relay_cache_release(pool, table, lengths, refs, _i32([0, 2], cuda))
            history[0], history[2] = [[], []], [[], []]
            table, refs, used = dbl.relay_cache_compact(pool, table, refs)
            assert used.tolist() == [int((refs > 0).sum())] and not refs[used.item():].any()
            attend()
    assert refs.sum() == (table >= 0).sum()
    _ok()


@gpu
def test_the_example(cuda, native_lib, capsys):
    """The serving example, small: its last step against relay_merge_decode on the cache's values, which it reads back
    rounded to bf16 (2^-9 of a value; rounding of both outputs to bf16, 2^-9 each, norm-wise below 1e-2)."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("serving", os.path.join(ROOT, "examples", "relay_cache_serving.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    assert m.main(["--sequences", "5", "--prefix", "77", "--prompt", "30", "--steps", "40"]) < 1e-2
    assert "pages in use" in capsys.readouterr().out
    _ok()


@gpu
def test_states_and_lists_of_other_types(cuda, native_lib):
    """int64 tables, lengths and lists, and strided ones, are converted; the arguments stay as they were."""
    pool = dbl.relay_cache_pool(8, 1, 64, 16, device=cuda)
    big = torch.full((4, 6), -1, device=cuda, dtype=torch.int64)
    table, lengths, refs = big[::2, ::2], torch.tensor([0, 0], device=cuda), torch.zeros(8, device=cuda, dtype=torch.int64)
    table, refs2, missing = dbl.relay_cache_reserve(pool, table, lengths, refs, torch.tensor([20, 3], device=cuda))
    assert missing.dtype == torch.int32 and missing.tolist() == [0]
    assert table.tolist() == [[0, 1, -1], [2, -1, -1]] and refs2.tolist() == [1, 1, 1, 0, 0, 0, 0, 0]
    assert (big == -1).all() and not refs.any()
    kv = torch.randn(2, 20, 1, 64, device=cuda)
    lengths = dbl.relay_cache_append(pool, table.long(), lengths, kv, kv, counts=torch.tensor([20, 3], device=cuda))
    assert lengths.tolist() == [20, 3]
    o, _, _ = dbl.relay_cache_attention(kv[:, 0], pool, table.long(), lengths.long())
    assert torch.equal(o, dbl.relay_cache_attention(kv[:, 0], pool, table, lengths)[0])
    table, refs2, used = dbl.relay_cache_compact(pool, table.long(), refs2.long())
    assert used.tolist() == [3] and table.tolist() == [[0, 1, -1], [2, -1, -1]]
    table, lengths, refs2 = dbl.relay_cache_release(pool, table, lengths, refs2, torch.tensor([1], device=cuda))
    assert lengths.tolist() == [20, 0] and refs2.tolist() == [1, 1, 0, 0, 0, 0, 0, 0]
    dbl.relay_cache_release(pool, table, lengths, refs2, torch.zeros(0, device=cuda, dtype=torch.int32))  # an empty list
    _ok()
