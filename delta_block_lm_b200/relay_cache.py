"""The relay cache in 4 bits, over torch CUDA tensors: keys and values that grow by tokens, in pages
that sequences share, copy and give back, and the attention that reads them.

It serves where ``relay_merge_decode`` does, at 5 bits a value (codes and their group's scale and
minimum) instead of 16, and without padding every sequence to one capacity.  The reference has no
counterpart: its relay attention keeps dense keys and values.

The state is four tensors that the caller owns:

    pool        uint8 [pages, kv_heads, page_size / 16, 20 head_dim] (``relay_cache_pool``)
    page_table  int32 [sequences, width]: each sequence's pages in order, -1 where it has none
    lengths     int32 [sequences]: tokens held; lowering one drops a sequence's last tokens
    refs        int32 [pages]: how many entries of the page table hold a page (0: free)

The pool is written in place; calls that change the page table, lengths or refs return new tensors
(``out=`` takes them to tensors of the caller, the arguments themselves included).  Nothing here
waits for the device, so a serving loop can be captured into a CUDA graph.  A token whose page does
not exist is left out and recorded for ``dbl_device_error`` (code 102).

    relay_cache_reserve    pages for the next tokens, copy on write    relay_cache_fork     share a sequence's pages
    relay_cache_append     write tokens                                relay_cache_release  give pages back
    relay_cache_attention  attention of the newest tokens              relay_cache_compact  pages in use to the front
    relay_cache_read       tokens back as values                       relay_cache_copy_pages
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading
from typing import Optional

import torch

from . import _native as N
from .kernels import _dtype_code, _ptr, _require_cuda

TILE = 16  # tokens of one tile: page sizes are multiples of it


def _packer(args):
    """Packs the fields of an argument structure, one after another, into its bytes: a fifth of the time that
    building the ctypes structure takes."""
    codes = {ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f", ctypes.c_void_p: "P"}

    def of(t):
        if issubclass(t, ctypes.Structure):
            return "".join(of(f) for _, f in t._fields_)
        return f"{t._length_}{codes[t._type_]}" if issubclass(t, ctypes.Array) else codes[t]

    packed = struct.Struct("@" + of(args) + "0q")
    assert packed.size == ctypes.sizeof(args), args
    return packed.pack


_APPEND, _READ = _packer(N.RelayCacheAppendArgs), _packer(N.RelayCacheReadArgs)
_ATTENTION, _PAGES = _packer(N.RelayCacheAttentionArgs), _packer(N.RelayCachePagesArgs)


class _Here:
    """The context of a call whose device is the current one already."""

    def __enter__(self):
        return None

    def __exit__(self, *_):
        return None


_here = _Here()

# A decode step makes several of these calls, and the host path is most of a small one's time: the short ways
# to the current device and stream, and the library's functions looked up once.


def _device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """The index of the CUDA device that the tensors share."""
    d = first.get_device()
    for t in others:
        if t is not None and t.get_device() != d:
            d = -1
    if d < 0:
        _require_cuda(first, *others)  # says what is wrong
    return d


def _on(d: int):
    return _here if d == torch._C._cuda_getDevice() else torch.cuda.device(d)


_stream = torch._C._cuda_getCurrentRawStream
_functions: dict = {}


def _library(name: str):
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = getattr(N.lib(), "dbl_relay_cache_" + name)
    return f


def _call(name: str, *args) -> None:
    status = _library(name)(*args)
    if status:
        N.check(status)


def relay_cache_pool(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, *, device="cuda") -> torch.Tensor:
    """An empty pool (zeroed) of ``pages`` pages of ``page_size`` tokens (a multiple of 16)."""
    if head_dim not in (64, 128):
        raise ValueError(f"relay cache: head_dim must be 64 or 128, got {head_dim}")
    if page_size <= 0 or page_size % TILE:
        raise ValueError(f"relay cache: page_size must be a multiple of {TILE}, got {page_size}")
    return torch.zeros((pages, kv_heads, page_size // TILE, 20 * head_dim), device=device, dtype=torch.uint8)


def _cache(pool: torch.Tensor) -> tuple:
    """The fields of dbl_relay_cache: pages, kv heads, head width, page size, address."""
    shape = pool.shape
    if pool.dtype != torch.uint8 or len(shape) != 4 or not pool.is_contiguous() or shape[3] not in (1280, 2560):
        raise ValueError("relay cache: pool must be a contiguous uint8 [pages, kv_heads, page_size / 16, 20 head_dim]"
                         f" with head_dim 64 or 128, got {pool.dtype} {list(shape)}")
    p, h, t, b = shape
    return p, h, b // 20, t * TILE, pool.data_ptr()


def _ints(name: str, t: Optional[torch.Tensor], shape: tuple) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"relay cache: {name} must be {list(shape)}, got {list(t.shape)}")
    if t.dtype != torch.int32 or not t.is_contiguous():
        t = t.to(torch.int32).contiguous()
    return t


def _at(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _list(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 1:
        raise ValueError(f"relay cache: {name} must be a list (one dimension), got {list(t.shape)}")
    return _ints(name, t, tuple(t.shape))


def relay_cache_append(pool, page_table, lengths, k, v, *, counts=None, out=None) -> torch.Tensor:
    """Writes the tokens k, v [N, T, kv_heads, D] (f32 or bf16; any strides with unit innermost) after
    the ``lengths`` [N] tokens that each sequence holds, and returns the new lengths.  ``counts`` [N]:
    how many of the T tokens are real (ragged prompts).  The pages must have been reserved."""
    dev = _device(pool, page_table, lengths, k, v, counts, out)
    c = _cache(pool)
    shape = k.shape
    if len(shape) != 4 or shape[2:] != c[1:3] or shape != v.shape:
        raise ValueError(f"relay cache append: k and v must be [N,T,{c[1]},{c[2]}], got {list(k.shape)} and "
                         f"{list(v.shape)}")
    n, t = shape[:2]
    if v.dtype != k.dtype:
        raise ValueError("relay cache append: v must have the dtype of k")
    if page_table.dim() != 2 or page_table.shape[0] != n:
        raise ValueError(f"relay cache append: page_table must be [{n},width], got {list(page_table.shape)}")
    page_table = _ints("page_table", page_table, page_table.shape)
    lengths, counts = _ints("lengths", lengths, (n,)), _ints("counts", counts, (n,))
    if t == 0 or n == 0:
        return lengths.clone() if out is None else out.copy_(lengths)
    if k.stride(3) != 1:
        k = k.contiguous()
    if v.stride(3) != 1:
        v = v.contiguous()
    with _on(dev):
        new = torch.empty_like(lengths)
        a = _APPEND(*c, n, t, page_table.shape[1], 0, _dtype_code(k), k.data_ptr(), v.data_ptr(), *k.stride(), *v.stride(),
                    page_table.data_ptr(), lengths.data_ptr(), _at(counts), new.data_ptr())
        _call("append", a, _stream(dev))
        return new if out is None else out.copy_(new)


def relay_cache_read(pool, page_table, lengths, *, start=None, tokens: int, dtype=torch.bfloat16):
    """Tokens start[n] .. start[n] + tokens - 1 of every sequence as the values that the cache holds:
    (k, v) [N, tokens, kv_heads, D] in ``dtype`` (f32 or bf16); zeros at and past ``lengths``."""
    dev = _device(pool, page_table, lengths, start)
    c = _cache(pool)
    if page_table.dim() != 2:
        raise ValueError(f"relay cache read: page_table must be [N,width], got {list(page_table.shape)}")
    n = page_table.shape[0]
    page_table = _ints("page_table", page_table, page_table.shape)
    lengths, start = _ints("lengths", lengths, (n,)), _ints("start", start, (n,))
    with _on(dev):
        k = pool.new_empty((n, tokens, c[1], c[2]), dtype=dtype)
        v = torch.empty_like(k)
        a = _READ(*c, n, tokens, page_table.shape[1], 0, _dtype_code(k), page_table.data_ptr(), lengths.data_ptr(),
                  _at(start), k.data_ptr(), v.data_ptr())
        if k.numel():
            _call("read", a, _stream(dev))
    return k, v


_workspaces = threading.local()  # .kept: (what for, device, stream) -> a workspace kept from call to call


def _workspace(what: str, need: int, dev: int, stream: int) -> torch.Tensor:
    """A workspace whose counters (the attention's) are zero.  The calls of one thread on one stream follow
    one another, so each thread keeps one a stream; launches of two threads may interleave between the
    two launches of a call.  A graph that is being captured gets its own (it may be replayed beside other
    calls)."""
    capturing = torch._C._cuda_isCurrentStreamCapturing()
    try:
        kept = _workspaces.kept
    except AttributeError:
        kept = _workspaces.kept = {}
    ws = None if capturing else kept.get((what, dev, stream))
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, device=torch.device("cuda", dev), dtype=torch.uint8)
        ws[:N.RELAY_CACHE_COUNTER_BYTES].zero_()
        if not capturing:
            kept[what, dev, stream] = ws
    return ws


def relay_cache_attention(q, pool, page_table, lengths, *, prefix_pages=None, prefix_len: int = 0,
                          scale: Optional[float] = None, out=None, workspace: Optional[torch.Tensor] = None):
    """Attention of each sequence's newest tokens over [shared prefix ; own tokens].

    q [N, heads, D], or [N, Tq, heads, D] for the last Tq tokens of each sequence, causal among
    themselves; f32 or bf16, heads a multiple of the pool's kv heads.  ``lengths`` counts the queries'
    own tokens (append first).  ``prefix_pages`` [width] names the pages of ``prefix_len`` tokens that
    every sequence sees before its own.  ``workspace``: a uint8 tensor whose first
    ``RELAY_CACHE_COUNTER_BYTES`` bytes are zero before its first use, and that no other thread uses
    meanwhile (by default each thread keeps one a stream, until it ends).  Returns (o, row_max, row_sum) as
    ``relay_merge_decode``; a row without keys gives o = 0 and (0, 1)."""
    dev = _device(q, pool, page_table, lengths, prefix_pages, out, workspace)
    c = _cache(pool)
    shape = q.shape
    if len(shape) == 3:
        n, heads, d = shape
        tq, rows, steps = 1, (n, heads), (heads, 1)
    elif len(shape) == 4:
        n, tq, heads, d = shape
        rows, steps = (n, tq, heads), (tq * heads, heads, 1)
    else:
        d = 0
    if d != c[2]:
        raise ValueError(f"relay cache attention: q must be [N,heads,{c[2]}] or [N,Tq,heads,{c[2]}], got {list(shape)}")
    table_shape = page_table.shape
    if len(table_shape) != 2 or table_shape[0] != n:
        raise ValueError(f"relay cache attention: page_table must be [{n},width], got {list(table_shape)}")
    page_table = _ints("page_table", page_table, table_shape)
    lengths = _ints("lengths", lengths, (n,))
    prefix_at = prefix_width = 0
    if prefix_len:
        if prefix_pages is None or prefix_pages.dim() != 1:
            raise ValueError("relay cache attention: prefix_pages must be a list of pages")
        prefix_pages = _list("prefix_pages", prefix_pages)
        prefix_at, prefix_width = prefix_pages.data_ptr(), prefix_pages.shape[0]
    strides = q.stride()
    if strides[-1] != 1:
        q = q.contiguous()
        strides = q.stride()
    if len(shape) == 3:
        strides = (strides[0], 0, strides[1], 1)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    with _on(dev):
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
        elif out.shape != shape or out.dtype != q.dtype or not out.is_contiguous():
            raise ValueError("relay cache attention: out must be contiguous with the shape and dtype of q")
        device = q.device
        row_max = torch.empty_strided(rows, steps, device=device, dtype=torch.float32)
        row_sum = torch.empty_strided(rows, steps, device=device, dtype=torch.float32)
        a = _ATTENTION(*c, n, tq, heads, table_shape[1], 0, prefix_len, prefix_width, _dtype_code(q), scale, q.data_ptr(),
                       *strides, page_table.data_ptr(), lengths.data_ptr(), prefix_at, out.data_ptr(), row_max.data_ptr(),
                       row_sum.data_ptr())
        if q.numel():
            stream = _stream(dev)
            if workspace is None:
                workspace = _workspace("attention", _library("attention_workspace_bytes")(a), dev, stream)
            _call("attention", a, workspace.data_ptr(), workspace.numel(), stream)
    return out, row_max, row_sum


def _pages(pool, page_table, lengths, refs, out, lists, new_lengths=True):
    """(device, arguments, outputs, tensors to keep) of a page operation; lengths None: it has none."""
    dev = _device(pool, page_table, lengths, refs, *lists, *(out or ()))
    c = _cache(pool)
    if page_table.dim() != 2:
        raise ValueError(f"relay cache: page_table must be [sequences,width], got {list(page_table.shape)}")
    s, w = page_table.shape
    page_table, refs = _ints("page_table", page_table, (s, w)), _ints("refs", refs, c[:1])
    lengths = _ints("lengths", lengths, (s,))
    new_lengths = new_lengths and lengths is not None
    given = (page_table, lengths, refs) if new_lengths else (page_table, refs)
    if out is None:
        after = tuple([torch.empty_like(t) for t in given])
    else:
        after = tuple(out)
        if len(after) != len(given):
            raise ValueError(f"relay cache: out must be {len(given)} tensors")
        for t, o in zip(given, after):
            if o.shape != t.shape or o.dtype != torch.int32 or not o.is_contiguous():
                raise ValueError("relay cache: out must be contiguous int32 tensors shaped like the state")
    a = _PAGES(*c, s, w, 0, page_table.data_ptr(), _at(lengths), refs.data_ptr(), after[0].data_ptr(),
               after[1].data_ptr() if new_lengths else 0, after[-1].data_ptr())
    return dev, a, after, (page_table, lengths, refs)


def _scratch(pages, sequences, dev, stream):
    return _workspace("pages", _library("pages_workspace_bytes")(pages, sequences), dev, stream)


def relay_cache_release(pool, page_table, lengths, refs, sequences, *, out=None):
    """Gives back the pages of ``sequences`` (a list of row numbers).  Returns (page_table, lengths, refs)."""
    sequences = _list("sequences", sequences)
    dev, a, after, _keep = _pages(pool, page_table, lengths, refs, out, (sequences,))
    with _on(dev):
        _call("release", a, sequences.data_ptr(), sequences.numel(), _stream(dev))
    return after


def relay_cache_fork(pool, page_table, lengths, refs, parents, children, *, out=None):
    """children[i] (named once and no parent itself) continues from parents[i], sharing its pages; the
    pages that it held are given back.  Returns (page_table, lengths, refs)."""
    parents, children = _list("parents", parents), _list("children", children)
    if parents.shape != children.shape:
        raise ValueError("relay cache fork: parents and children must have the same length")
    dev, a, after, _keep = _pages(pool, page_table, lengths, refs, out, (parents, children))
    with _on(dev):
        _call("fork", a, parents.data_ptr(), children.data_ptr(), parents.numel(), _stream(dev))
    return after


def relay_cache_reserve(pool, page_table, lengths, refs, tokens, *, out=None):
    """Pages for the next ``tokens`` (a number, or a list of one for each sequence) tokens of every
    sequence.  Every page that they are written to and that others hold too is replaced before (with the
    tokens that it holds below ``lengths``), so lowering a length drops a sequence's last tokens and no one
    else's.  Returns (page_table, refs, missing): ``missing`` [1] is 0, or how many pages the pool lacks, and
    then nothing changes.  ``out``: (page_table, refs)."""
    counts = None
    if isinstance(tokens, torch.Tensor):
        counts, tokens = _ints("tokens", tokens, tuple(lengths.shape)), 0
    dev, a, after, _keep = _pages(pool, page_table, lengths, refs, out, () if counts is None else (counts,), False)
    with _on(dev):
        missing, stream = refs.new_empty(1, dtype=torch.int32), _stream(dev)
        ws = _scratch(pool.shape[0], page_table.shape[0], dev, stream)
        _call("reserve", a, _ptr(counts), tokens, missing.data_ptr(), ws.data_ptr(), ws.numel(), stream)
    return after[0], after[1], missing


def relay_cache_compact(pool, page_table, refs, *, out=None):
    """Moves the pages in use to the front of the pool (in place) and renames them in the page table.
    Returns (page_table, refs, used): pages 0 .. used - 1 are in use, the others free.  A shared
    prefix's pages follow if they are a row of the page table."""
    dev, a, after, _keep = _pages(pool, page_table, None, refs, out, ())
    with _on(dev):
        used, stream = refs.new_empty(1, dtype=torch.int32), _stream(dev)
        ws = _scratch(pool.shape[0], page_table.shape[0], dev, stream)
        _call("compact", a, used.data_ptr(), ws.data_ptr(), ws.numel(), stream)
    return after[0], after[1], used


def relay_cache_copy_pages(pool, src, dst) -> None:
    """Copies page src[i] to page dst[i] (no page is both, none is written twice)."""
    src, dst = _list("src", src), _list("dst", dst)
    dev = _device(pool, src, dst)
    if src.shape != dst.shape:
        raise ValueError("relay cache copy: src and dst must have the same length")
    c = N.RelayCache(*_cache(pool))
    with _on(dev):
        _call("copy_pages", ctypes.byref(c), _ptr(src), _ptr(dst), src.numel(), _stream(dev))
