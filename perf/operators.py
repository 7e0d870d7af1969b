"""Cases of the paged key/value cache operators and their plain forms.

The cache (``KvCache``): page ``table[s][p // ps]`` holds position ``p`` of
sequence ``s``; a page holds a tile of ``ps`` rows for every (layer, K or V, kv
head). A bf16 tile is ``[ps][128]``. A 4-bit tile is ``ps`` rows of 64 code
bytes, then ``ps`` rows of four bf16 scales, one for each 32 dims; 32-bit word
``4 t + g`` of a row's codes holds dims ``32 g + 8 t ..`` (lowest nibble first,
code = value + 8).

Operators: ``attend`` (attention over the cache with an optional sliding window
and first positions that stay visible, one or many rows for each sequence, bf16
or 4-bit pages), ``append`` / ``read`` (4-bit rows stored and loaded),
``fork``, ``free``, ``compact`` and ``resize`` of pages.
"""
import math
import random

import numpy as np
import torch

own = False  # False: the plain forms below; True: the framework's operators

HEAD_DIM = 128
DEVICE = "cuda:0"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _attend(name, seqs, past, rows, kv_heads, group, layers, bits, dtype, window, sinks, page=32,
            mix=0):
    return {"name": name, "op": "attend", "seqs": seqs, "past_min": past[0], "past_max": past[1],
            "rows_min": rows[0], "rows_max": rows[1], "kv_heads": kv_heads, "group": group,
            "layers": layers, "bits": bits, "dtype": dtype, "window": window, "sinks": sinks,
            "page": page, "mix": mix}


def listed():
    return [
        # One stream's decode step a minute into a long reading: the latency case.
        _attend("window step, 1 stream", 1, (700, 700), (1, 1), 8, 2, 28, 16, "f32", 256, 9),
        # A batch of 16 requests in lockstep, each minutes long, fp32 activations.
        _attend("window step, 16 streams", 16, (900, 2047), (1, 1), 8, 2, 4, 16, "f32", 1024, 9),
        # Many very long streams with a wide window: the cache read from HBM.
        _attend("window step, 32 long", 32, (12000, 16383), (1, 1), 8, 2, 1, 16, "bf16", 4096, 4),
        # A prompt of 256 text ids (and its 9 role rows) prefilled under a narrow window.
        _attend("window prompt, 265 rows", 1, (0, 0), (265, 265), 8, 2, 28, 16, "f32", 128, 9),
        # Two long ragged prompts prefilled together.
        _attend("window prompts, long", 2, (0, 2000), (2500, 4096), 8, 2, 1, 16, "bf16", 2048, 16,
                mix=3),
        # One stream's decode step over a 4-bit cache.
        _attend("4-bit step, 1 stream", 1, (512, 512), (1, 1), 8, 2, 28, 4, "f32", 0, 0),
        # 64 streams of ten minutes and more over a 4-bit cache: the bandwidth case.
        _attend("4-bit step, 64 streams", 64, (7000, 8191), (1, 1), 8, 2, 1, 4, "bf16", 0, 0),
        # A chunk of new text rows on sequences that already hold a long past, 4-bit pages.
        _attend("4-bit chunk, 4 sequences", 4, (1000, 4000), (100, 512), 8, 2, 2, 4, "bf16", 0, 0,
                mix=5),
        # The rows of 16 prompts quantised into 4-bit pages and read back.
        {"name": "4-bit store and load", "op": "store", "seqs": 16, "past_min": 0, "past_max": 100,
         "rows_min": 150, "rows_max": 265, "kv_heads": 8, "layers": 4, "dtype": "f32", "page": 32,
         "mix": 1},
        # One 265-position prompt forked into 15 more takes (28 layers: 3.7 MB pages).
        {"name": "fork, 15 takes", "op": "fork", "sources": 1, "takes": 15, "len_min": 265,
         "len_max": 265, "kv_heads": 8, "layers": 28, "page": 32, "spare": 40, "mix": 0},
        # A small batch turning over: half leaves, the pages close up, new ones join.
        {"name": "turnover, 8 sequences", "op": "turnover", "seqs": 8, "len_min": 40,
         "len_max": 200, "kv_heads": 8, "layers": 4, "page": 16, "spare": 9, "mix": 2},
        # A serving batch of 64 turning over.
        {"name": "turnover, 64 sequences", "op": "turnover", "seqs": 64, "len_min": 500,
         "len_max": 1500, "kv_heads": 8, "layers": 4, "page": 32, "spare": 100, "mix": 4},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["step", "step", "step", "rows", "rows", "store", "fork", "turnover"])
        mix = rng.randrange(1 << 20)
        kv = rng.choice([1, 2, 4, 8])
        page = rng.choice([16, 32, 64])
        bits, dtype = rng.choice([16, 4]), rng.choice(["f32", "bf16"])
        window = rng.choice([0, _log(rng, 1, 4096)])
        sinks = rng.choice([0, _log(rng, 1, 64)]) if window else 0
        if kind in ("step", "rows"):
            n = _log(rng, 1, 64) if kind == "step" else _log(rng, 1, 8)
            top = _log(rng, 1, 16384)
            rows = 1 if kind == "step" else _log(rng, 2, 4096)
            c = _attend("", n, (top // rng.choice([1, 2, 8]), top),
                        (rows if kind == "step" else max(1, rows // 2), rows), kv,
                        rng.choice([1, 2, 4]), rng.choice([1, 2, 7]), bits, dtype, window, sinks,
                        page, mix)
            keys = c["seqs"] * (c["past_max"] + c["rows_max"])
            if keys * kv > 64 * 8192 * 8 or c["layers"] * keys * kv * 512 > 3e8:
                continue
            if c["seqs"] * c["rows_max"] * kv * c["group"] * (c["past_max"] + c["rows_max"]) > 8e8:
                continue
        elif kind == "store":
            c = {"op": "store", "seqs": _log(rng, 1, 64), "past_min": 0,
                 "past_max": rng.randrange(200), "rows_min": 1, "rows_max": _log(rng, 1, 2000),
                 "kv_heads": kv, "layers": rng.choice([1, 3, 6]), "dtype": dtype, "page": page,
                 "mix": mix}
            if c["seqs"] * c["rows_max"] * kv > 16 * 265 * 8:
                continue
        elif kind == "fork":
            c = {"op": "fork", "sources": rng.choice([1, 1, 2, 3]), "takes": _log(rng, 1, 15),
                 "len_min": 0, "len_max": _log(rng, 1, 2048), "kv_heads": kv,
                 "layers": _log(rng, 1, 28), "page": page, "spare": rng.randrange(50), "mix": mix}
        else:
            top = _log(rng, 1, 1500)
            c = {"op": "turnover", "seqs": 2 * _log(rng, 1, 32), "len_min": top // 4,
                 "len_max": top, "kv_heads": kv, "layers": rng.choice([1, 2, 4]), "page": page,
                 "spare": rng.randrange(60), "mix": mix}
        if c["op"] in ("fork", "turnover"):
            if _pages(c) * _page_bytes(c, 16) > 1.2e9 or work(c)["bytes"] < 1:
                continue
        c.pop("name", None)
        return c


# ---------------------------------------------------------------------------
# sizes
# ---------------------------------------------------------------------------
def _page_bytes(case, bits):
    return case["layers"] * 2 * case["kv_heads"] * case["page"] * (256 if bits == 16 else 72)


def _between(case, lo, hi, n, salt):
    r = random.Random(case["mix"] * 7919 + salt)
    return [r.randint(lo, hi) for _ in range(n)]


def _rows_of(case):
    return _between(case, case["rows_min"], case["rows_max"], case["seqs"], 1)


def _lengths(case):
    """Positions of each sequence after the call's rows."""
    if case["op"] in ("attend", "store"):
        past = _between(case, case["past_min"], case["past_max"], case["seqs"], 2)
        return [p + r for p, r in zip(past, _rows_of(case))]
    if case["op"] == "fork":
        return _between(case, case["len_min"], case["len_max"], case["sources"], 3)
    return _between(case, case["len_min"], case["len_max"], case["seqs"], 4)


def _need(case, lengths):
    return [-(-n // case["page"]) for n in lengths]


def _pages(case):
    used = sum(_need(case, _lengths(case)))
    if case["op"] == "fork":  # one tail page for each take
        return used + case["sources"] * case["takes"] + case["spare"]
    return used + case.get("spare", 5)


def _visible(pos, window, sinks):
    """How many keys the row at `pos` sees."""
    if window == 0 or pos < window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    lens = _lengths(case)
    if case["op"] == "attend":
        size = 4 if case["dtype"] == "f32" else 2
        heads = case["kv_heads"] * case["group"]
        row = 256 if case["bits"] == 16 else 72
        rows = _rows_of(case)
        pairs, keys = 0, 0
        for n, r in zip(lens, rows):
            pairs += sum(_visible(p, case["window"], case["sinks"]) for p in range(n - r, n))
            first = max(0, n - r - case["window"] + 1) if case["window"] else 0
            keys += n - first + min(case["sinks"], first)
        moved = sum(rows) * heads * HEAD_DIM * size * 2 + keys * case["kv_heads"] * 2 * row
        return {"bytes": moved, "flops": 4 * HEAD_DIM * heads * pairs}
    if case["op"] == "store":
        n = sum(_rows_of(case)) * case["kv_heads"] * 2
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * (2 * HEAD_DIM * size + 2 * 72), "flops": 0}
    if case["op"] == "fork":
        copies = sum(case["takes"] for n in lens if n % case["page"])
        return {"bytes": 2 * copies * _page_bytes(case, 16) + 4 * _pages(case), "flops": 0}
    half = case["seqs"] // 2
    need = _need(case, lens)
    front, back = sum(need[:half]), sum(need[half:])
    # in the turnover's steady state each compaction moves the other half down,
    # as far as that half does not overlap the place it goes to
    moved = min(front, back) * 2
    return {"bytes": 2 * moved * _page_bytes(case, 16) + 4 * _pages(case), "flops": 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _bf16_nearest(x):
    """x (float64, >= 0) rounded once to the nearest bf16 value, ties to even:
    the 52 mantissa bits are cut to 7."""
    bits = x.view(torch.int64)
    bits = (bits + ((1 << 44) - 1) + ((bits >> 45) & 1)) >> 45 << 45
    return bits.view(torch.float64)


def _quantise(x):
    """[..., 128] -> (n [..., 4, 32] in -7..7, scale [..., 4]), both rounded once
    from the exact quotients (float64: values next to a border)."""
    x = x.double().reshape(*x.shape[:-1], 4, 32)
    # a tensor of sevens: division by a Python number multiplies by its reciprocal
    top = x.abs().amax(-1)
    s = _bf16_nearest(top / torch.full_like(top, 7.0))
    n = torch.where(s[..., None] > 0, torch.round(x / s.clamp_min(1e-300)[..., None]), 0.0)
    return n.clamp(-7, 7), s


def _pack(x):
    """Rows [..., 128] as (code bytes [..., 64], scale bytes [..., 8])."""
    n, s = _quantise(x)
    u = (n + 8).to(torch.uint8).reshape(*x.shape[:-1], 4, 4, 4, 2)  # [g][t][byte][nibble]
    b = u[..., 0] | (u[..., 1] << 4)
    codes = b.transpose(-3, -2).reshape(*x.shape[:-1], 64)
    return codes, s.to(torch.bfloat16).view(torch.uint8)


def _unpack(codes, scales):
    """Code bytes [..., 64] and bf16 scales [..., 4] as float32 rows [..., 128]."""
    b = codes.reshape(*codes.shape[:-1], 4, 4, 4).transpose(-3, -2)  # [g][t][byte]
    n = torch.stack((b & 15, b >> 4), -1).reshape(*codes.shape[:-1], 4, 32).float() - 8.0
    return (n * scales.float()[..., None]).reshape(*codes.shape[:-1], HEAD_DIM)


def _package():
    from __graft_entry__ import load_package

    return load_package()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    kv, ps, layers = case["kv_heads"], case["page"], case["layers"]
    bits = case.get("bits", 4 if case["op"] == "store" else 16)
    lens, pages = _lengths(case), _pages(case)
    need = _need(case, lens)
    seqs = case["sources"] * (1 + case["takes"]) if case["op"] == "fork" else case["seqs"]
    width = max(1, max(need))
    # pages in use, in shuffled order; a shared or free page is one no table names
    order = torch.randperm(pages, generator=g, device=DEVICE, dtype=torch.int32)
    table = torch.full((seqs, width), -1, dtype=torch.int32, device=DEVICE)
    slot = torch.tensor([i * width + j for i, n in enumerate(need) for j in range(n)],
                        dtype=torch.int64, device=DEVICE)
    table.view(-1)[slot] = order[: slot.numel()]
    refs = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    refs[order[: slot.numel()].long()] = 1
    lengths = torch.tensor(lens + [0] * (seqs - len(lens)), dtype=torch.int32, device=DEVICE)

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=dtype)

    if bits == 16:
        pool = normal(pages, layers, 2, kv, ps, HEAD_DIM, dtype=torch.bfloat16)
    else:
        x = normal(pages, layers, 2, kv, ps, HEAD_DIM, dtype=torch.bfloat16)
        pool = torch.empty(pages, layers, 2, kv, ps * 72, dtype=torch.uint8, device=DEVICE)
        for l in range(layers):
            codes, scales = _pack(x[:, l])
            pool[:, l, ..., : ps * 64] = codes.flatten(-2)
            pool[:, l, ..., ps * 64:] = scales.flatten(-2)
        del x
    st = {"case": case, "pool": pool, "table": table, "lengths": lengths, "refs": refs,
          "layer": layers // 2, "seqs": seqs}
    if case["op"] in ("attend", "store"):
        rows = _rows_of(case)
        total, st["max_rows"] = sum(rows), max(rows)
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        st["row_start"] = None
        if case["op"] == "store" or case["rows_max"] > 1:
            st["row_start"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
        if case["op"] == "attend":
            st["q"] = normal(total, kv * case["group"], HEAD_DIM, dtype=_dtype(case))
            st["max_length"] = max(lens)
        else:
            st["k"] = normal(total, kv, HEAD_DIM, dtype=_dtype(case))
            st["v"] = normal(total, kv, HEAD_DIM, dtype=_dtype(case))
    elif case["op"] == "fork":
        t = case["takes"]
        st["src"] = [i for i in range(case["sources"]) for _ in range(t)]
        st["dst"] = [case["sources"] + i for i in range(case["sources"] * t)]
    else:
        half = case["seqs"] // 2
        st["halves"] = [(list(range(half)), lens[:half]),
                        (list(range(half, case["seqs"])), lens[half:])]
    if own:  # the cache object that a program keeps over these buffers
        st["cache"] = _package().KvCache(pool, table, lengths, refs, layers=layers, kv_heads=kv,
                                         page_size=ps, kv_bits=bits)
    else:    # index lists on the device, made once
        as_index = lambda v: torch.tensor(v, dtype=torch.int64, device=DEVICE)  # noqa: E731
        if case["op"] == "fork":
            st["src"], st["dst"] = as_index(st["src"]), as_index(st["dst"])
        elif case["op"] == "turnover":
            st["halves"] = [(as_index(s), as_index(n)) for s, n in st["halves"]]
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    case = st["case"]
    if own:
        c = st["cache"]
        if case["op"] == "attend":
            return c.attend(st["layer"], st["q"], window=case["window"], sinks=case["sinks"],
                            row_start=st["row_start"], max_rows=st["max_rows"],
                            max_length=st["max_length"])
        if case["op"] == "store":
            c.append(st["layer"], st["k"], st["v"], row_start=st["row_start"],
                     max_rows=st["max_rows"])
            return c.read(st["layer"], st["k"].shape[0], dtype=st["k"].dtype,
                          row_start=st["row_start"], max_rows=st["max_rows"])
        if case["op"] == "fork":
            c.fork(st["src"], st["dst"])
        else:
            for seqs, lens in st["halves"]:
                c.free(seqs)
                c.compact()
                c.resize(seqs, lens)
        return st["table"], st["lengths"], st["refs"], st["pool"]
    if case["op"] == "attend":
        return _plain_attend(st)
    if case["op"] == "store":
        return _plain_store(st)
    if case["op"] == "fork":
        _plain_free(st, st["dst"])
        _plain_fork(st)
    else:
        (a, la), (b, lb) = st["halves"]
        _plain_free(st, a)
        _plain_compact(st)
        _plain_grow(st, a, la)
        _plain_free(st, b)
        _plain_compact(st)
        _plain_grow(st, b, lb)
    return st["table"], st["lengths"], st["refs"], st["pool"]


def _row_places(st, total):
    """Group and position of every row."""
    n = st["case"]["seqs"]
    row = torch.arange(total, device=DEVICE)
    if st["row_start"] is None:
        return row, st["lengths"].long() - 1
    start = st["row_start"].long()
    group = torch.searchsorted(start[1:], row, right=True)
    return group, st["lengths"].long()[:n][group] - start[group + 1] + row


def _plain_attend(st):
    case, q, pool = st["case"], st["q"], st["pool"]
    kv, g, ps, n = case["kv_heads"], case["group"], case["page"], case["seqs"]
    group, pos = _row_places(st, q.shape[0])
    tiles = pool[st["table"].clamp_min(0).long(), st["layer"]]  # [n, width, 2, kv, ...]
    if case["bits"] == 16:
        dense = tiles.float()
    else:
        codes = tiles[..., : ps * 64].unflatten(-1, (ps, 64))
        scales = tiles[..., ps * 64:].contiguous().view(torch.bfloat16).unflatten(-1, (ps, 4))
        dense = _unpack(codes, scales)
    dense = dense.permute(2, 0, 3, 1, 4, 5).reshape(2, n, kv, -1, HEAD_DIM)
    k, v = dense[0], dense[1]
    width = st["max_rows"]
    slot = torch.zeros_like(group)  # the row's place in its group
    if st["row_start"] is not None:
        slot = torch.arange(q.shape[0], device=DEVICE) - st["row_start"].long()[group]
    qp = torch.zeros(n, width, kv * g, HEAD_DIM, device=DEVICE)
    qp[group, slot] = q.float()
    qp = qp.reshape(n, width, kv, g, HEAD_DIM).transpose(1, 2).reshape(n, kv, width * g, HEAD_DIM)
    s = (qp @ k.transpose(-1, -2)) * (1.0 / math.sqrt(HEAD_DIM))
    at = torch.full((n, width), -1, device=DEVICE)
    at[group, slot] = pos
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = key <= at[..., None]
    if case["window"]:
        seen &= (at[..., None] - key < case["window"]) | (key < case["sinks"])
    seen = seen.repeat_interleave(g, 1)[:, None]  # [n, 1, width * g, keys]
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    out = out.reshape(n, kv, width, g, HEAD_DIM).transpose(1, 2).reshape(n, width, kv * g, HEAD_DIM)
    return out[group, slot].to(q.dtype)


def _plain_store(st):
    case, pool = st["case"], st["pool"]
    ps = case["page"]
    group, pos = _row_places(st, st["k"].shape[0])
    page = st["table"][group, pos // ps].long()
    row = (pos % ps)[:, None]
    tiles = pool[:, st["layer"]]  # [pages, 2, kv, ps * 72]
    codes = tiles[..., : ps * 64].unflatten(-1, (ps, 64))
    scales = tiles[..., ps * 64:].unflatten(-1, (ps, 8))
    head = torch.arange(case["kv_heads"], device=DEVICE)
    at = page[:, None], head, row
    ck, sk = _pack(st["k"])
    cv, sv = _pack(st["v"])
    codes[:, 0][at], scales[:, 0][at] = ck, sk
    codes[:, 1][at], scales[:, 1][at] = cv, sv
    k = _unpack(codes[:, 0][at], scales[:, 0][at].view(torch.bfloat16))
    v = _unpack(codes[:, 1][at], scales[:, 1][at].view(torch.bfloat16))
    return k.to(st["k"].dtype), v.to(st["k"].dtype)


def _plain_free(st, seqs):
    rows = st["table"][seqs].long()
    held = rows >= 0
    st["refs"].index_add_(0, rows.clamp_min(0).view(-1), -held.view(-1).to(torch.int32))
    st["table"][seqs] = -1
    st["lengths"][seqs] = 0


def _plain_take(st, wanted):
    """A free page for every true entry of `wanted`, lowest pages first."""
    free = torch.argsort((st["refs"] > 0).to(torch.int32), stable=True)
    place = wanted.view(-1).to(torch.int64).cumsum(0) - 1
    page = free[place.clamp(0, free.numel() - 1)].view(wanted.shape)
    st["refs"].index_add_(0, page.view(-1), wanted.view(-1).to(torch.int32))
    return page.to(torch.int32)


def _plain_fork(st):
    ps, src, dst = st["case"]["page"], st["src"], st["dst"]
    table, lengths, pool = st["table"], st["lengths"], st["pool"]
    n = lengths[src].long()
    full = n // ps
    logical = torch.arange(table.shape[1], device=DEVICE)
    rows = torch.where(logical < full[:, None], table[src], -1)
    shared = rows >= 0
    st["refs"].index_add_(0, rows.clamp_min(0).long().view(-1), shared.view(-1).to(torch.int32))
    partial = (logical == full[:, None]) & (n % ps > 0)[:, None]
    page = _plain_take(st, partial)
    has = torch.nonzero(partial.any(1)).view(-1)
    pool[page[partial].long()] = pool[table[src[has], full[has]].long()]
    table[dst] = torch.where(partial, page, rows)
    lengths[dst] = lengths[src]


def _plain_compact(st):
    refs, table, pool = st["refs"], st["table"], st["pool"]
    live = refs > 0
    page = torch.arange(refs.numel(), device=DEVICE)
    low = page < live.sum()
    src, dst = torch.nonzero(live & ~low).view(-1), torch.nonzero(~live & low).view(-1)
    pool[dst] = pool[src]
    refs[dst] = refs[src]
    refs[src] = 0
    page[src] = dst
    table.copy_(torch.where(table >= 0, page[table.clamp_min(0).long()].to(torch.int32), -1))


def _plain_grow(st, seqs, lens):
    logical = torch.arange(st["table"].shape[1], device=DEVICE)
    wanted = logical < (-(-lens // st["case"]["page"]))[:, None]
    page = _plain_take(st, wanted)
    st["table"][seqs] = torch.where(wanted, page, -1)
    st["lengths"][seqs] = lens.to(torch.int32)


# ---------------------------------------------------------------------------
# the operators' definitions in 64 bits, row by row
# ---------------------------------------------------------------------------
def _exact_tile(tile, ps):
    word = tile[: ps * 64].reshape(ps, 16, 4).long()
    word = word[..., 0] + (word[..., 1] << 8) + (word[..., 2] << 16) + (word[..., 3] << 24)
    out = torch.zeros(ps, HEAD_DIM, dtype=torch.float64, device=tile.device)
    scale = tile[ps * 64:].reshape(ps, 4, 2).contiguous().view(torch.bfloat16)[..., 0].double()
    for d in range(HEAD_DIM):
        w = (d % 32) // 8 * 4 + d // 32
        out[:, d] = ((word[:, w] >> (4 * (d % 8))) % 16 - 8).double() * scale[:, d // 32]
    return out


def _exact_attend(st):
    case, q = st["case"], st["q"].double()
    kv, g, ps = case["kv_heads"], case["group"], case["page"]
    out = torch.zeros_like(q)
    table, row = st["table"].tolist(), 0
    lens, rows = _lengths(case), _rows_of(case)
    if case["bits"] == 4:  # one tile at a time is slow: all pages of a head as one tall tile
        flat = st["pool"][:, st["layer"]]
        codes = flat[..., : ps * 64].transpose(0, 1).transpose(1, 2)
        scales = flat[..., ps * 64:].transpose(0, 1).transpose(1, 2)
    for i in range(case["seqs"]):
        n, r = lens[i], rows[i]
        mine = torch.tensor(table[i][: -(-n // ps)], device=DEVICE, dtype=torch.int64)
        pos = torch.arange(n - r, n, device=DEVICE)[:, None]
        key = torch.arange(n, device=DEVICE)[None]
        hidden = key > pos
        if case["window"]:
            hidden = hidden | ((key >= case["sinks"]) & (key <= pos - case["window"]))
        for h in range(kv):
            dense = []
            for which in (0, 1):
                if case["bits"] == 16:
                    t = st["pool"][mine, st["layer"], which, h].double().reshape(-1, HEAD_DIM)
                else:
                    tall = torch.cat((codes[which, h][mine].reshape(-1),
                                      scales[which, h][mine].reshape(-1)))
                    t = _exact_tile(tall, mine.numel() * ps)
                dense.append(t[:n])
            for j in range(g):
                s = q[row: row + r, h * g + j] @ dense[0].T / HEAD_DIM ** 0.5
                w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                out[row: row + r, h * g + j] = w @ dense[1]
        row += r
    return out


def _exact_store(st):
    def value(t):
        x = t.double().cpu().numpy().reshape(-1, 32)
        m, e = np.frexp(np.abs(x).max(1, keepdims=True) / 7.0)  # m in [0.5, 1)
        s = np.ldexp(np.rint(np.ldexp(m, 8)), e - 8)  # eight significant bits
        n = np.clip(np.rint(np.divide(x, s, out=np.zeros_like(x), where=s > 0)), -7, 7)
        return torch.from_numpy((n * s).reshape(t.shape)).to(DEVICE)

    return tuple(value(st[w]) for w in ("k", "v"))


def exact(case, seed):
    if case["op"] not in ("attend", "store"):
        return None  # tables, counts and copied pages: nothing is computed in floating point
    st = prepare(case, seed)
    return _exact_attend(st) if case["op"] == "attend" else _exact_store(st)
