"""The operators of the 4-bit relay cache: what is measured, and their plain forms.

A cache pool is a uint8 tensor [pages, kv_heads, page_size / 16, 20 D] (D = 64 or 128 channels a head).  The last
dimension is one tile of 16 tokens, G = D / 32 groups of channels:

  offset   bytes  content
  0        8 D    key codes    [16 tokens][4 parts t][G groups j][8 codes i]           channel 32 j + 8 t + i
  8 D      2 D    key groups   [16 tokens][G]                                          (scale, minimum), bf16 each
  10 D     8 D    value codes  [2 halves][8 parts g][8 tokens][G groups j][4 codes i]  channel 32 j + 4 g + i
  18 D     2 D    value groups [16 tokens][G]                                          (scale, minimum), bf16 each

two codes a byte, the lower one in the lower half, and value = minimum + scale * code.  For the 32 values x of a
group: minimum = min(x) rounded down to bf16, scale = (max(x) - minimum) / 15 rounded up to bf16, code = the smallest
c of 0 .. 15 with x - minimum <= (c + 1/2) scale.  A range below 2^-100 has scale 0 and codes 0; a range that is not
finite makes the group NaN.

The page table [sequences, width] names each sequence's pages in order (-1: none), `lengths` its tokens and `refs`
[pages] how many page-table entries hold a page.
"""
import random

import torch

own = False

TILE, GROUP = 16, 32
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the first tokens of one small conversation: nothing but latency
        _attention("token_first", "bf16", 1, 1, 4, 4, 64, 16, 0, 37, 37),
        # the relay benchmark's decode step (64 sequences, prefix 4096, 1024 own tokens, 16 heads of 128), cache in 4 bits
        _attention("token_relay", "bf16", 64, 1, 16, 16, 128, 64, 4096, 1024, 1024),
        # a batch of conversations of all lengths, 8 query heads to a cache head
        _attention("token_grouped_ragged", "bf16", 48, 1, 32, 4, 128, 32, 0, 1, 8191),
        # one long document: the long-context benchmark's 131072 tokens
        _attention("token_long", "bf16", 1, 1, 16, 16, 128, 64, 0, 131072, 131072),
        # f32 activations, odd numbers of everything, an empty sequence among them, a prefix that ends inside a page
        _attention("token_f32_odd", "f32", 7, 1, 6, 2, 64, 16, 1001, 0, 3001),
        # six drafted tokens a sequence checked at once (causal among themselves)
        _attention("draft_check", "bf16", 16, 6, 16, 8, 128, 32, 77, 6, 4099),
        # prompts written into the cache: the prefill benchmark's 8 x 4096 tokens, 16 heads of 128
        _append("fill_prompts", "bf16", 8, 4096, 16, 128, 64, 0, 0, False),
        # one decode step of 256 sequences (the decode benchmark's), each at its own length
        _append("fill_token", "bf16", 256, 1, 16, 128, 64, 1, 1000, False),
        # ragged prompts in f32 that continue inside a page
        _append("fill_f32_ragged", "f32", 5, 777, 3, 64, 16, 0, 100, True),
        # the page work of one step: 16 prompts, 240 continuations dropped and forked again, one new token each
        _step("pages_step", 16, 240, 16, 128, 64, 500, 2000, 1),
        # the same for a handful of short sequences
        _step("pages_step_small", 2, 6, 4, 64, 16, 20, 60, 1),
        # a pool of 4096 pages, half of them in use, scattered by sequences that left
        _compact("pages_compact", 4096, 64, 0.5, 16, 128, 64),
    ]


def _attention(name, dtype, n, tq, hq, hkv, d, page, prefix, lo, hi):
    return {"name": name, "kind": "attention", "dtype": dtype, "n": n, "tq": tq, "hq": hq, "hkv": hkv, "d": d,
            "page": page, "prefix": prefix, "lo": lo, "hi": hi}


def _append(name, dtype, n, t, hkv, d, page, lo, hi, ragged):
    return {"name": name, "kind": "append", "dtype": dtype, "n": n, "t": t, "hkv": hkv, "d": d, "page": page,
            "lo": lo, "hi": hi, "ragged": ragged}


def _step(name, live, forks, hkv, d, page, lo, hi, tokens):
    return {"name": name, "kind": "step", "live": live, "forks": forks, "hkv": hkv, "d": d, "page": page, "lo": lo,
            "hi": hi, "tokens": tokens}


def _compact(name, pages, rows, used, hkv, d, page):
    return {"name": name, "kind": "compact", "pages": pages, "rows": rows, "used": used, "hkv": hkv, "d": d,
            "page": page}


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["attention", "attention", "attention", "append", "step", "compact"])
    d, page = rng.choice([64, 128]), rng.choice([16, 32, 64, 128])
    if kind == "attention":
        group = rng.choice([1, 1, 2, 4, 7, 8])
        hkv, n = rng.choice([1, 2, 3, 4, 8, 16]), log(1, 64)
        tq = rng.choice([1, 1, 1, 2, 5, 9])
        prefix = rng.choice([0, 0, log(1, 4096)])
        most = min(131072, 2000000 // (n * hkv))  # tokens of all sequences and heads: the longest case's
        most = min(most, 20_000_000_000 // (4 * d * n * tq * hkv * group) - prefix)
        if most < 16:
            tq, prefix, most = 1, 0, 16
        hi = log(16, most)
        lo = rng.choice([0, tq, hi])
        case = _attention("", rng.choice(["bf16", "bf16", "f32"]), n, tq, hkv * group, hkv, d, page, prefix,
                          min(lo, hi), hi)
    elif kind == "append":
        n, hkv = log(1, 256), rng.choice([1, 3, 4, 8, 16])
        t = rng.choice([1, log(1, max(1, 500000 // (n * hkv)))])
        lo = log(1, 500) - 1
        case = _append("", rng.choice(["bf16", "f32"]), n, t, hkv, d, page, lo, lo + log(1, 500), rng.random() < 0.5)
    elif kind == "step":
        live = log(1, 32)
        lo = log(1, 500)
        case = _step("", live, log(1, 224), rng.choice([1, 4, 16]), d, page, lo, lo + log(1, 1000),
                     rng.choice([1, 1, 4, 33]))
    else:
        case = _compact("", log(64, 4096), log(1, 64), rng.choice([0.2, 0.5, 0.8]), rng.choice([1, 4, 16]), d,
                        rng.choice([16, 32, 64]))
    del case["name"]
    return case


def _lengths(n, lo, hi):
    """n lengths spread over lo .. hi, the first of them lo (one alone: hi)."""
    return [hi] if n == 1 else [lo + int((i * 0.6180339887498949) % 1.0 * (hi - lo + 1)) for i in range(n)]


def _ceil(a, b):
    return -(-a // b)


def _layout(case):
    """The page numbers of a pool that sequences have left: {rows, width, table (a list), refs (a list)}."""
    rng = random.Random(case["pages"])
    pages, rows = case["pages"], case["rows"]
    used = sorted(rng.sample(range(pages), max(1, int(pages * case["used"]))))
    rng.shuffle(used)
    shared, rest = used[:max(1, len(used) // 16)], used[max(1, len(used) // 16):]  # a prompt that every row has
    each = _ceil(len(rest), rows)
    width = len(shared) + each + 1
    table, refs = [], [0] * pages
    for r in range(rows):
        mine = shared + rest[r * each:(r + 1) * each]
        for p in mine:
            refs[p] += 1
        table.append(mine + [-1] * (width - len(mine)))
    return {"width": width, "table": table, "refs": refs}


def work(case):
    kind = case["kind"]
    tile = 20 * case["d"]
    token = case["hkv"] * tile // TILE  # bytes of one token in the cache
    if kind == "attention":
        lens, size = _lengths(case["n"], case["lo"], case["hi"]), DTYPES[case["dtype"]].itemsize
        rows = case["n"] * case["tq"] * case["hq"]
        keys = sum(sum(max(0, n - case["tq"] + 1 + i) for i in range(case["tq"])) for n in lens)
        keys += case["prefix"] * case["n"] * case["tq"]
        return {"bytes": (sum(lens) + case["prefix"]) * token + rows * (2 * case["d"] * size + 8) + 4 * case["n"]
                + 4 * sum(_ceil(n, case["page"]) for n in lens),
                "flops": 4 * case["d"] * case["hq"] * keys}
    if kind == "append":
        size = DTYPES[case["dtype"]].itemsize
        tokens = sum(_counts(case))
        dense = case["hkv"] * case["d"] * 2 * size
        out = case["n"] * case["t"] * dense
        return {"bytes": tokens * (dense + 2 * token) + out, "flops": tokens * case["hkv"] * case["d"] * 2 * 8}
    if kind == "step":
        lens = _lengths(case["live"], case["lo"], case["hi"])
        moved = sum(_ceil(lens[i % case["live"]] % case["page"], TILE) for i in range(case["forks"]))
        rows = case["live"] + case["forks"]
        return {"bytes": 2 * moved * case["hkv"] * tile + 12 * rows * _ceil(case["hi"] + case["tokens"], case["page"]),
                "flops": 0}
    at = _layout(case)
    count = sum(r > 0 for r in at["refs"])
    moved = sum(r > 0 for r in at["refs"][count:])
    return {"bytes": 2 * moved * case["hkv"] * (case["page"] // TILE) * tile
            + 8 * (case["rows"] * at["width"] + case["pages"]), "flops": 0}


def _counts(case):
    return _lengths(case["n"], 1, case["t"]) if case["ragged"] else [case["t"]] * case["n"]


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _dense(case, pages, seed, count=None):
    """Keys and values [pages, hkv, page, d] as a model makes them: keys have an offset of their own in each channel."""
    g = _generator(seed + 1)
    offset = 2 * _randn(g, 1, case["hkv"], 1, case["d"])
    shape = (count or pages, case["hkv"], case["page"], case["d"])
    for _ in range(_ceil(pages, shape[0])):
        yield (_randn(g, *shape) + offset).bfloat16(), _randn(g, *shape).bfloat16()


def _pages_at_once(case, pages):
    return max(1, min(pages, (1 << 26) // (case["hkv"] * case["page"] * case["d"])))


def _tables(lens, page, width, g, first=0):
    """A page table over the pages first .. first + sum of pages - 1, in random order, and how many they are."""
    need = _ints([_ceil(n, page) for n in lens]).long()
    total = sum(_ceil(n, page) for n in lens)
    order = torch.randperm(total, generator=g, device="cuda") + first
    at = torch.arange(width, device="cuda") + (need.cumsum(0) - need)[:, None]
    table = torch.where(torch.arange(width, device="cuda") < need[:, None],
                        order[at.clamp(max=max(0, total - 1))] if total else at, torch.full_like(at, -1))
    return table.to(torch.int32), total


def prepare(case, seed):
    g = _generator(seed)
    kind, page, d = case["kind"], case["page"], case["d"]
    tiles = page // TILE
    state = {"case": case}
    if kind == "attention":
        lens = _lengths(case["n"], case["lo"], case["hi"])
        first = _ceil(case["prefix"], page)
        state["prefix_pages"] = torch.randperm(first, generator=g, device="cuda").to(torch.int32)
        state["table"], total = _tables(lens, page, max(1, _ceil(case["hi"], page)), g, first)
        state["lengths"] = _ints(lens)
        pages = max(1, first + total)
        state["pool"] = torch.empty((pages, case["hkv"], tiles, 20 * d), dtype=torch.uint8, device="cuda")
        step = _pages_at_once(case, pages)
        for at, (k, v) in zip(range(0, pages, step), _dense(case, pages, seed, step)):
            state["pool"][at:at + step] = _pack(k, v)[:pages - at]
        heads = (case["n"], case["hq"], d) if case["tq"] == 1 else (case["n"], case["tq"], case["hq"], d)
        state["q"] = _randn(g, *heads).to(DTYPES[case["dtype"]])
    elif kind == "append":
        lens, counts = _lengths(case["n"], case["lo"], case["hi"]), _counts(case)
        ends = [a + b for a, b in zip(lens, counts)]
        state["table"], total = _tables(ends, page, _ceil(max(ends), page), g)
        state["lengths"], state["counts"] = _ints(lens), _ints(counts) if case["ragged"] else None
        state["pool"] = torch.zeros((total, case["hkv"], tiles, 20 * d), dtype=torch.uint8, device="cuda")
        shape = (case["n"], case["t"], case["hkv"], d)
        state["k"] = (_randn(g, *shape) + 2 * _randn(g, 1, 1, case["hkv"], d)).to(DTYPES[case["dtype"]])
        state["v"] = _randn(g, *shape).to(DTYPES[case["dtype"]])
    elif kind == "step":
        live, forks = case["live"], case["forks"]
        lens = _lengths(live, case["lo"], case["hi"])
        lens += [lens[i % live] for i in range(forks)]
        width = _ceil(case["hi"] + case["tokens"], page) + 1
        state["table"], total = _tables(lens, page, width, g)
        extra = forks + (live + forks) * _ceil(case["tokens"], page)
        order = torch.randperm(total + extra, generator=g, device="cuda").to(torch.int32)
        state["table"] = torch.where(state["table"] >= 0, order[state["table"].clamp(min=0).long()], -1)
        state["lengths"] = _ints(lens)
        state["refs"] = torch.zeros(total + extra, dtype=torch.int32, device="cuda")
        state["refs"][order[:total].long()] = 1
        state["parents"] = _ints([i % live for i in range(forks)])
        state["children"] = _ints([live + i for i in range(forks)])
        state["pool"] = torch.randint(0, 256, (total + extra, case["hkv"], tiles, 20 * d), generator=g, device="cuda",
                                      dtype=torch.uint8)
    else:
        at = _layout(case)
        state["table"], state["refs"] = _ints(at["table"]), _ints(at["refs"])
        state["pool"] = torch.randint(0, 256, (case["pages"], case["hkv"], tiles, 20 * d), generator=g, device="cuda",
                                      dtype=torch.uint8)
    return state


# ------------------------------------------------------------------------------------------------ running
def run(state):
    return _OWN[state["case"]["kind"]](state) if own else _PLAIN[state["case"]["kind"]](state)


def _own_attention(s):
    import delta_block_lm_b200 as dbl
    return dbl.relay_cache_attention(s["q"], s["pool"], s["table"], s["lengths"], prefix_pages=s["prefix_pages"],
                                     prefix_len=s["case"]["prefix"])


def _own_append(s):
    import delta_block_lm_b200 as dbl
    lengths = dbl.relay_cache_append(s["pool"], s["table"], s["lengths"], s["k"], s["v"], counts=s["counts"])
    k, v = dbl.relay_cache_read(s["pool"], s["table"], lengths, start=s["lengths"], tokens=s["case"]["t"],
                                dtype=DTYPES[s["case"]["dtype"]])
    return lengths, k, v


def _own_step(s):
    import delta_block_lm_b200 as dbl
    table, lengths, refs = dbl.relay_cache_release(s["pool"], s["table"], s["lengths"], s["refs"], s["children"])
    table, lengths, refs = dbl.relay_cache_fork(s["pool"], table, lengths, refs, s["parents"], s["children"])
    table, refs, short = dbl.relay_cache_reserve(s["pool"], table, lengths, refs, s["case"]["tokens"])
    return table, lengths, refs, short, s["pool"]


def _own_compact(s):
    import delta_block_lm_b200 as dbl
    table, refs, used = dbl.relay_cache_compact(s["pool"], s["table"], s["refs"])
    return table, refs, used, s["pool"]


_OWN = {"attention": _own_attention, "append": _own_append, "step": _own_step, "compact": _own_compact}


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(x):
    """(scale, minimum, code) of the groups of x [..., D], in 32 bits; scale and minimum are bf16 values."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low = x.amin(-1).view(torch.int32)
    low = (torch.where(low < 0, low + 0xFFFF, low) & -0x10000).view(torch.float32)  # down to bf16
    span = x.amax(-1) - low
    scale = span / torch.full_like(span, 15)  # by a tensor: a number would be multiplied by its rounded reciprocal
    scale = ((scale.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32)  # up to bf16
    scale = torch.where(span < 2.0 ** -100, 0.0, scale)
    bad = ~torch.isfinite(span)
    scale, low = torch.where(bad, torch.nan, scale), torch.where(bad, torch.nan, low)
    above, step = x - low[..., None], scale[..., None]
    code = torch.ceil(above / step - 0.5)
    code = code + (above > (code + 0.5) * step).float() - (above <= (code - 0.5) * step).float()
    return scale, low, torch.where(step > 0, code.clamp(0, 15), 0.0)


def _pack(k, v):
    """Tiles [P, H, page / 16, 20 D] (uint8) of k, v [P, H, page, D]."""
    p, h, page, d = k.shape
    tiles = (p, h, page // TILE)
    parts = []
    for x, key in ((k, True), (v, False)):
        scale, low, code = _quantise(x)
        code = code.to(torch.uint8)
        if key:
            code = code.reshape(*tiles, TILE, d // 32, 4, 8).transpose(-3, -2)
        else:
            code = code.reshape(*tiles, 2, 8, d // 32, 8, 4).permute(0, 1, 2, 3, 6, 4, 5, 7)
        code = code.reshape(*tiles, 8 * d, 2)
        parts += [code[..., 0] | code[..., 1] << 4,
                  torch.stack([scale, low], -1).bfloat16().reshape(*tiles, d).view(torch.uint8)]
    return torch.cat(parts, -1)


def _unpack(tiles):
    """Keys and values [..., tokens, D] in f32 of tiles [..., page / 16, 20 D]."""
    lead, d = tiles.shape[:-2], tiles.shape[-1] // 20
    out = []
    for key, part in ((True, tiles[..., :10 * d]), (False, tiles[..., 10 * d:])):
        code = torch.stack([part[..., :8 * d] & 15, part[..., :8 * d] >> 4], -1)
        if key:
            code = code.reshape(*tiles.shape[:-1], TILE, 4, d // 32, 8).transpose(-3, -2)
        else:
            code = code.reshape(*tiles.shape[:-1], 2, 8, 8, d // 32, 4).movedim(-4, -2)
        group = part[..., 8 * d:].contiguous().view(torch.bfloat16).reshape(*tiles.shape[:-1], TILE, d // 32, 1, 2)
        code = code.reshape(*tiles.shape[:-1], TILE, d // 32, GROUP).float()
        out.append((group[..., 1].float() + group[..., 0].float() * code).reshape(*lead, -1, d))
    return out


def _gather(pool, table):
    """Keys and values [..., H, width * page, D] in f32 of the pages that a table [..., width] names."""
    pages = pool[table.clamp(min=0).long()]
    k, v = _unpack(pages)  # [..., width, H, page, D]
    return tuple(x.movedim(-3, -4).flatten(-3, -2) for x in (k, v))


def _plain_attention(s):
    case, q = s["case"], s["q"].float()
    n, tq, hkv, d = case["n"], case["tq"], case["hkv"], case["d"]
    group = case["hq"] // hkv
    rows = q.reshape(n, tq, hkv, group, d).transpose(1, 2).reshape(n, hkv, tq * group, d) * d ** -0.5
    k, v = _gather(s["pool"], s["table"])
    limit = s["lengths"][:, None] - tq + 1 + torch.arange(tq, device=q.device)
    seen = torch.arange(k.shape[2], device=q.device) < limit.repeat_interleave(group, 1)[:, None, :, None]
    live = (torch.arange(k.shape[2], device=q.device) < s["lengths"][:, None])[:, None, :, None]
    k, v = torch.where(live, k, 0.0), torch.where(live, v, 0.0)
    scores = torch.where(seen, rows @ k.transpose(-1, -2), -torch.inf)
    top = scores.amax(-1)
    if case["prefix"]:
        pk, pv = (x[:, :case["prefix"]] for x in _gather(s["pool"], s["prefix_pages"]))
        before = rows @ pk.transpose(-1, -2)
        top = torch.maximum(top, before.amax(-1))
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = torch.exp(scores - top[..., None])
    total, acc = p.sum(-1), p @ v
    if case["prefix"]:
        p = torch.exp(before - top[..., None])
        total, acc = total + p.sum(-1), acc + p @ pv
    total = torch.where(total == 0, 1.0, total)
    o = (acc / total[..., None]).unflatten(2, (tq, group)).transpose(1, 2).reshape(s["q"].shape)
    top, total = (x.unflatten(2, (tq, group)).transpose(1, 2).reshape(s["q"].shape[:-1]) for x in (top, total))
    return o.to(s["q"].dtype), top, total


def _plain_append(s):
    dtype, t = DTYPES[s["case"]["dtype"]], s["case"]["t"]
    counts = s["counts"] if s["counts"] is not None else torch.full_like(s["lengths"], t)
    real = (torch.arange(t, device="cuda") < counts[:, None])[..., None, None]
    values = []
    for x in (s["k"], s["v"]):
        scale, low, code = _quantise(x)
        values.append(torch.where(real, (low[..., None] + scale[..., None] * code).flatten(-2), 0.0).to(dtype))
    return s["lengths"] + counts, values[0], values[1]


def _plain_step(s):
    page, tokens, pool = s["case"]["page"], s["case"]["tokens"], s["pool"]
    table, lengths, refs = s["table"].clone(), s["lengths"].clone(), s["refs"].clone()
    parents, children = s["parents"].long(), s["children"].long()
    slot = torch.arange(table.shape[1], device="cuda")

    def count(rows, add):  # refs of the pages in `rows`, -1 left out
        one = torch.where(rows >= 0, add, 0).to(torch.int32).flatten()
        refs.index_add_(0, rows.clamp(min=0).long().flatten(), one)

    # release
    count(table[children], -1)
    table[children], lengths[children] = -1, 0
    # fork
    rows = torch.where(slot * page < lengths[parents][:, None], table[parents], -1)
    table[children], lengths[children] = rows, lengths[parents]
    count(rows, 1)
    # reserve: the page that the next token falls in is copied where others hold it too, the last of its holders keeps it
    full = (lengths + page - 1) // page
    ends = (lengths + tokens + page - 1) // page
    at = (lengths // page).clamp(max=table.shape[1] - 1).long()
    here = table.gather(1, at[:, None])[:, 0]
    asks = (lengths % page > 0) & (here >= 0)
    key = torch.where(asks, here, 0).long()
    row = torch.arange(len(lengths), device="cuda", dtype=torch.int32)
    asked = torch.zeros_like(refs).index_add_(0, key, asks.to(torch.int32))
    last = torch.full_like(refs, -1).scatter_reduce_(0, key, torch.where(asks, row, -1), "amax")
    cow = asks & (refs[key] > 1) & ~((asked[key] == refs[key]) & (last[key] == row))
    fresh = (slot >= full[:, None]) & (slot < ends[:, None]) & (table < 0)
    wants = fresh | (cow[:, None] & (slot == at[:, None]))  # in the order of sequences, then slots
    rank = wants.flatten().cumsum(0).view_as(wants) - 1
    free = refs == 0
    place = torch.where(free, free.cumsum(0) - 1, len(refs))
    first = torch.zeros(len(refs) + 1, dtype=torch.int32, device="cuda")
    first.scatter_(0, place, torch.arange(len(refs), device="cuda", dtype=torch.int32))
    short = (wants.sum() - free.sum()).clamp(min=0).to(torch.int32)
    got = first[rank.clamp(0, len(refs) - 1)]
    ok = short == 0
    new = torch.where(wants & ok, got, table)
    refs.index_add_(0, key, torch.where(cow & ok, -1, 0).to(torch.int32))
    refs.index_add_(0, got.flatten().long(), (wants & ok).flatten().to(torch.int32))
    # the tiles of the copied pages that hold tokens
    to = torch.where(cow & ok, new.gather(1, at[:, None])[:, 0], here).clamp(min=0).long()
    tile = torch.arange(pool.shape[2], device="cuda")
    held = (cow & ok)[:, None] & (tile * TILE < (lengths % page)[:, None])
    which = held[:, None, :, None].expand(-1, pool.shape[1], -1, pool.shape[3])
    index = ((to[:, None, None, None] * pool.shape[1] + torch.arange(pool.shape[1], device="cuda")[:, None, None])
             * pool.shape[2] + tile[:, None]) * pool.shape[3] + torch.arange(pool.shape[3], device="cuda")
    pool.view(-1)[index[which]] = pool[key][which]
    return new, lengths, refs, short.reshape(1), pool


def _plain_compact(s):
    pool, refs, table = s["pool"], s["refs"], s["table"]
    used = (refs > 0).sum()
    number = torch.arange(len(refs), device="cuda")
    holes = torch.nonzero((refs == 0) & (number < used))[:, 0]
    movers = torch.nonzero((refs > 0) & (number >= used))[:, 0]
    pool[holes] = pool[movers]
    to = number.clone()
    to[movers] = holes
    new = torch.zeros_like(refs).index_put_((to[refs > 0],), refs[refs > 0])
    moved = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table)
    return moved, new, used.to(torch.int32).reshape(1), pool


_PLAIN = {"attention": _plain_attention, "append": _plain_append, "step": _plain_step, "compact": _plain_compact}


# ------------------------------------------------------------------------------------------------ 64 bits
def _values64(x):
    """What the cache keeps of x [..., D], from the definition in 64 bits."""
    x = x.double().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)

    def to_bf16(y, up):
        near = y.bfloat16()
        over = near.double() < y if up else near.double() > y
        bits = near.view(torch.int16)
        away = (bits >= 0) if up else (bits < 0)  # the next value in that direction is further from zero
        return torch.where(over, torch.where(away, bits + 1, bits - 1), bits).view(torch.bfloat16).double()

    low = to_bf16(low, False)
    step = to_bf16((high - low) / 15, True)
    code = torch.floor((x - low) / step + 0.5)
    code = torch.where((code - 0.5) * step == x - low, code - 1, code).clamp(0, 15)
    return torch.where(high - low < 2.0 ** -100, low.expand_as(x), low + step * code).flatten(-2)


def exact(case, seed):
    if case["kind"] == "append":
        s = prepare(case, seed)
        counts = _counts(case)
        k, v = _values64(s["k"]), _values64(s["v"])
        for i, c in enumerate(counts):
            k[i, c:], v[i, c:] = 0, 0
        return None, k, v
    if case["kind"] != "attention":
        return None
    s = prepare(case, seed)
    n, tq, hkv, d = case["n"], case["tq"], case["hkv"], case["d"]
    pages, step = len(s["pool"]), _pages_at_once(case, len(s["pool"]))
    dense = [torch.cat(x)[:pages] for x in zip(*((a, b) for a, b in _dense(case, pages, seed, step)))]
    q = s["q"].double().reshape(n, tq, case["hq"], d)
    out = torch.zeros_like(q)
    top, total = torch.zeros(q.shape[:3], dtype=torch.float64, device="cuda"), torch.ones(q.shape[:3], dtype=torch.float64, device="cuda")
    lens = _lengths(n, case["lo"], case["hi"])
    group = case["hq"] // hkv
    first = [_values64(x[s["prefix_pages"].long()].transpose(0, 1).reshape(hkv, -1, d)[:, :case["prefix"]]) for x in dense]
    for i, length in enumerate(lens):
        mine = s["table"][i, :_ceil(length, case["page"])].long()
        k, v = (torch.cat([p, _values64(x[mine].transpose(0, 1).reshape(hkv, -1, d)[:, :length])], 1)
                for p, x in zip(first, dense))
        for j in range(tq):
            end = case["prefix"] + max(0, length - tq + 1 + j)
            if end == 0:
                continue
            scores = (q[i, j].reshape(hkv, group, d) @ k[:, :end].transpose(1, 2)) * d ** -0.5
            m = scores.amax(-1, keepdim=True)
            p = torch.exp(scores - m)
            out[i, j] = ((p @ v[:, :end]) / p.sum(-1, keepdim=True)).reshape(-1, d)
            top[i, j], total[i, j] = m.flatten(), p.sum(-1).flatten()
    shape = s["q"].shape
    return out.reshape(shape), top.reshape(shape[:-1]), total.reshape(shape[:-1])
