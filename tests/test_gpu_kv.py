"""Paged key / value caches on the GPU against oracle.kv in 64 bits.

Bound of an attention output (derived, per row): a score is a 128-term dot
product in fp32. Each product and each of its additions is off by at most a
rounding (tensor cores may cut instead of round: 2^-23), so the score is off by
e = (128 + 16) * 2^-23 * scale * max_c sum_d |q_d k_cd|, the 16 for the scaling,
a split of q into 16-bit parts and the exponent's argument. Softmax weights
are then off by a factor within exp(+-2 e), and the weighted sum of n values by
another (n + 64) * 2^-23, the 64 for the exponentials, the normalisation and
the merging of partial results. bf16 outputs add half a step, 2^-8 of the value
at most, and 2^-11 of the largest value for weights rounded once to fp16: a
weight is off by at most 2^-11 of itself, so the weighted mean by 2^-11 max |v|
(below fp16's normal range by 2^-25 at most each, beside a sum of at least 1: the
2^-23 above per value covers it):
  |out - exact| <= max_c |v_c| * (expm1(2 e) + (n + 64) * 2^-23 [+ 2^-11])
                   [+ 2^-8 * |exact|].
"""
import numpy as np
import pytest
import torch

from oracle import kv as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


class Filled:
    """A cache whose sequences have the given lengths, pages in shuffled order,
    random rows; unused rows and pages hold NaN scales / NaN values."""

    def __init__(self, pkg, lens, *, kv=2, ps=32, bits=16, layers=2, seed=0, spare=3, width=None,
                 pages=None):
        rng = np.random.default_rng(seed)
        need = [-(-n // ps) for n in lens]
        self.ps, self.bits, self.kv, self.layers, self.lens = ps, bits, kv, layers, list(lens)
        pages = sum(need) + spare if pages is None else pages
        width = max(1, max(need)) if width is None else width
        order = rng.permutation(pages)
        table = np.full((len(lens), width), -1, np.int32)
        refs = np.zeros(pages, np.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at: at + n]
            refs[order[at: at + n]] = 1
            at += n
        row = 256 if bits == 16 else 72
        pool = np.zeros((pages, layers, 2, kv, ps * row), np.uint8)
        if bits == 16:
            v = pool.view(np.uint16).reshape(pages, layers, 2, kv, ps, 128)
            x = torch.from_numpy(rng.standard_normal(v.shape, dtype=np.float32)).to(BF16)
            v[:] = x.view(torch.int16).numpy().view(np.uint16)
        else:
            pool[..., : ps * 64] = rng.integers(0, 256, pool[..., : ps * 64].shape)
            s = torch.from_numpy(rng.uniform(0.02, 0.4, (pages, layers, 2, kv, ps * 4)).astype(
                np.float32)).to(BF16).view(torch.int16).numpy()
            pool[..., ps * 64:] = s.view(np.uint8)
        # what no sequence holds: NaN
        used = np.zeros((pages, ps), bool)
        for s, n in enumerate(lens):
            for p in range(n):
                used[table[s, p // ps], p % ps] = True
        nan = np.array([0x7fc0], np.uint16)
        for page, r in np.argwhere(~used):
            if bits == 16:
                pool.view(np.uint16).reshape(pages, layers, 2, kv, ps, 128)[page, :, :, :, r] = nan
            else:
                pool[page, :, :, :, ps * 64 + r * 8: ps * 64 + (r + 1) * 8] = np.tile(
                    nan.view(np.uint8), 4)
        self.host = pool
        self.table = table
        t = lambda a: torch.from_numpy(a.copy()).to(DEV)  # noqa: E731
        self.cache = pkg.KvCache(t(pool.reshape(-1)), t(table), t(np.array(lens, np.int32)),
                                 t(refs), layers=layers, kv_heads=kv, page_size=ps, kv_bits=bits)

    def dense(self, layer, seq, n=None):
        """(K, V) [n][kv][128] float64, and which positions have a page."""
        return dense_of(self.host, self.table[seq], self.lens[seq] if n is None else n, layer,
                        self.ps, self.bits)


def dense_of(pool, row, n, layer, ps, bits):
    kv = pool.shape[3]
    p = np.arange(n)
    page, r = row[p // ps] if n else np.zeros(0, int), p % ps
    held = (page >= 0) & (page < pool.shape[0])
    tile = pool[np.where(held, page, 0), layer]  # [n][2][kv][bytes]
    if bits == 16:
        u = tile.view(np.uint16).reshape(n, 2, kv, ps, 128)[p, :, :, r].astype(np.uint32) << 16
        out = u.view(np.float32).astype(np.float64)
    else:
        code = tile[..., : ps * 64].reshape(n, 2, kv, ps, 64)[p, :, :, r]
        s = tile[..., ps * 64:].copy().view(np.uint16).reshape(n, 2, kv, ps, 4)[p, :, :, r]
        s = (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
        out = np.zeros((n, 2, kv, 128))
        for d in range(128):
            b, sh = O.code_place(d)
            out[..., d] = (((code[..., b] >> sh) & 15).astype(np.int64) - 8) * s[..., d // 32]
    out[~held] = 0.0
    return out[:, 0], out[:, 1], held


def check_rows(got, q, groups, filled, layer, window, sinks, scale=128 ** -0.5, dense=None):
    """groups: (sequence, length, first row, end row)."""
    got64, q64 = got.double().cpu().numpy(), q.double().cpu().numpy()
    heads = q64.shape[1]
    for seq, n, r0, r1 in groups:
        k, v, held = dense(seq, n) if dense else filled.dense(layer, seq, n)
        g = heads // k.shape[1]
        for r in range(r0, r1):
            pos = n - (r1 - r)
            if pos < 0:
                assert not got64[r].any()
                continue
            want = O.attend(q64[r], k, v, held, pos, window, sinks, scale)
            at = [c for c in range(pos + 1) if held[c] and O.sees(pos, c, window, sinks)]
            if not at:
                assert not got64[r].any()
                continue
            mag = np.stack([(np.abs(k[at, h // g]) @ np.abs(q64[r, h])).max() for h in range(heads)])
            big = np.stack([np.abs(v[at, h // g]).max() for h in range(heads)])
            e = 144 * 2.0 ** -23 * abs(scale) * mag
            tol = big * (np.expm1(2 * e) + (len(at) + 64) * 2.0 ** -23)
            if got.dtype == BF16:
                tol = tol[:, None] + 2.0 ** -11 * big[:, None] + 2.0 ** -8 * np.abs(want)
            else:
                tol = tol[:, None]
            bad = np.abs(got64[r] - want) > tol
            assert not bad.any(), (seq, n, r, pos, np.argwhere(bad)[:4].tolist(),
                                   np.abs(got64[r] - want).max(), tol.max())


def rand_q(rows, heads, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, heads, 128, generator=g).to(dtype).to(DEV)


# ---- attention, one row per sequence
SPANS = [(0, 0), (1, 0), (1, 1), (16, 0), (20, 5), (33, 40), (70, 3), (1000, 4)]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window,sinks", SPANS)
def test_step_spans(pkg, bits, dtype, window, sinks):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 129, 257]
    f = Filled(pkg, lens, bits=bits, seed=window + sinks)
    q = rand_q(len(lens), 4, dtype)
    out = f.cache.attend(1, q, window=window, sinks=sinks)
    check_rows(out, q, [(s, n, s, s + 1) for s, n in enumerate(lens)], f, 1, window, sinks)
    f.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kv,group", [(1, 1), (1, 3), (2, 2), (3, 1), (2, 4), (1, 5), (1, 8), (8, 2)])
@pytest.mark.parametrize("ps", [16, 32, 256])
def test_step_heads_and_pages(pkg, bits, dtype, kv, group, ps):
    lens = [70, 0, 5, 300]
    f = Filled(pkg, lens, kv=kv, ps=ps, bits=bits, layers=3, seed=kv * 10 + group)
    q = rand_q(3, kv * group, dtype)
    seqs = torch.tensor([3, 0, 3], dtype=torch.int32, device=DEV)  # a sequence may be named twice
    out = f.cache.attend(2, q, window=90, sinks=2, seqs=seqs, scale=0.2)
    check_rows(out, q, [(3, 300, 0, 1), (0, 70, 1, 2), (3, 300, 2, 3)], f, 2, 90, 2, 0.2)
    f.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [2000, 5003])
def test_step_long(pkg, bits, dtype, n):
    f = Filled(pkg, [n], bits=bits, layers=1, kv=1, seed=n)
    q = rand_q(1, 2, dtype)
    for hint in (0, n, 10):  # the hints never change what is computed
        out = f.cache.attend(0, q, max_length=hint)
        check_rows(out, q, [(0, n, 0, 1)], f, 0, 0, 0)
    out = f.cache.attend(0, q, window=1500, sinks=33)
    check_rows(out, q, [(0, n, 0, 1)], f, 0, 1500, 33)


# ---- attention, many rows per sequence
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kv,group", [(2, 1), (1, 2), (1, 4), (1, 3), (1, 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 3), (130, 70)])
def test_rows_ragged(pkg, bits, dtype, kv, group, window, sinks):
    lens = [90, 0, 200, 33, 7, 150]
    counts = [90, 0, 130, 1, 9, 0]  # the whole prompt, none, a chunk, one row, more rows than positions
    f = Filled(pkg, lens, kv=kv, bits=bits, seed=kv + group)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = rand_q(int(starts[-1]) + 4, kv * group, dtype)
    out = torch.full_like(q, 7.0)
    got = f.cache.attend(1, q, window=window, sinks=sinks, out=out,
                         row_start=torch.from_numpy(starts).to(DEV))
    assert got is out
    assert (out[int(starts[-1]):] == 7.0).all()  # rows behind the last group
    groups = [(s, n, int(starts[s]), int(starts[s + 1])) for s, n in enumerate(lens)]
    check_rows(out, q, groups, f, 1, window, sinks)
    f.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 8, 17, 64, 65, 129])
def test_rows_counts(pkg, bits, dtype, rows):
    f = Filled(pkg, [rows + 37, rows], kv=1, bits=bits, layers=1, seed=rows)
    q = rand_q(2 * rows, 2, dtype)
    starts = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=DEV)
    outs = []
    for hint in (0, rows):
        outs.append(f.cache.attend(0, q, row_start=starts, max_rows=hint, max_length=rows + 37))
        check_rows(outs[-1], q, [(0, rows + 37, 0, rows), (1, rows, rows, 2 * rows)], f, 0, 0, 0)
    # a hint that is too small costs time, not rows
    out = f.cache.attend(0, q, row_start=starts, max_rows=1, max_length=1)
    check_rows(out, q, [(0, rows + 37, 0, rows), (1, rows, rows, 2 * rows)], f, 0, 0, 0)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1),
                                          (2 ** 31 - 90, 7), (3, 2 ** 31 - 1)])
def test_spans_at_the_ends_of_their_type(pkg, bits, rows, window, sinks):
    f = Filled(pkg, [150], kv=1, bits=bits, layers=1, seed=3)
    starts = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    for dtype in (F32, BF16):
        q = rand_q(rows, 2, dtype)
        out = f.cache.attend(0, q, row_start=starts, window=window, sinks=sinks)
        check_rows(out, q, [(0, 150, 0, rows)], f, 0, window, sinks)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_groups_of_unknown_rows(pkg, bits, dtype):
    rng = np.random.default_rng(7)
    rows = rng.integers(0, 20, 300)
    rows[11] = 700  # far more tiles than its share
    lens = rows + rng.integers(0, 30, 300)
    f = Filled(pkg, lens.tolist(), kv=1, ps=16, bits=bits, layers=1, seed=2)
    starts = np.concatenate([[0], np.cumsum(rows)])
    q = rand_q(int(starts[-1]), 2, dtype)
    out = f.cache.attend(0, q, row_start=torch.tensor(starts, dtype=torch.int32, device=DEV), window=50,
                         sinks=2)
    check_rows(out, q, [(s, n, starts[s], starts[s + 1]) for s, n in enumerate(lens)], f, 0, 50, 2)
    f.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_chunks(pkg, bits):
    """Rows of two sequences captured once; replays follow lengths and rows."""
    f = Filled(pkg, [900, 300], kv=1, bits=bits, layers=1, width=64, seed=5)
    starts = torch.tensor([0, 30, 60], dtype=torch.int32, device=DEV)
    q, out = rand_q(60, 2, BF16), torch.zeros(60, 2, 128, dtype=BF16, device=DEV)
    f.cache.attend(0, q, row_start=starts, window=400, sinks=3, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        f.cache.attend(0, q, row_start=starts, window=400, sinks=3, out=out)
    for n0, n1, r0 in ((900, 300, 30), (700, 20, 11), (31, 299, 50)):
        f.cache.lengths.copy_(torch.tensor([n0, n1], dtype=torch.int32))
        starts.copy_(torch.tensor([0, r0, 60], dtype=torch.int32))
        q.copy_(rand_q(60, 2, BF16, n0))
        g.replay()
        check_rows(out, q, [(0, n0, 0, r0), (1, n1, r0, 60)], f, 0, 400, 3)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("group", [7, 130])
def test_more_heads_than_a_tile_has_rows(pkg, bits, dtype, group):
    f = Filled(pkg, [70, 40], kv=1, bits=bits, layers=1, seed=group)
    for rows in (1, 19):
        q = rand_q(2 * rows, group, dtype)
        starts = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=DEV)
        out = f.cache.attend(0, q, row_start=starts, window=30, sinks=2)
        check_rows(out, q, [(0, 70, 0, rows), (1, 40, rows, 2 * rows)], f, 0, 30, 2)


# few tiles over long caches: CTAs share the positions of a tile, some of them none
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens,rows,kv", [([3001], [40], 1), ([700, 2500, 64, 9], [17, 64, 64, 9], 1),
                                          ([1500, 40], [300, 40], 2), ([1030], [20], 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (900, 3), (33, 200)])
def test_few_rows_over_long_caches(pkg, bits, dtype, lens, rows, kv, window, sinks):
    f = Filled(pkg, lens, kv=kv, bits=bits, width=128, seed=sum(lens), layers=1)
    starts = np.concatenate([[0], np.cumsum(rows)])
    q = rand_q(int(starts[-1]), 2 * kv, dtype)
    kw = dict(row_start=torch.tensor(starts, dtype=torch.int32, device=DEV), max_rows=max(rows),
              window=window, sinks=sinks)
    out = f.cache.attend(0, q, **kw)
    assert torch.equal(out, f.cache.attend(0, q, **kw))
    check_rows(out, q, [(s, n, starts[s], starts[s + 1]) for s, n in enumerate(lens)], f, 0, window,
               sinks)
    # told of fewer rows, CTAs take more tiles in turn; told of the lengths, fewer share one
    for more in (dict(max_rows=9), dict(max_length=max(lens))):
        check_rows(f.cache.attend(0, q, **{**kw, **more}), q,
                   [(s, n, starts[s], starts[s + 1]) for s, n in enumerate(lens)], f, 0, window, sinks)
    f.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_tiles_agree_on_odd_values(pkg, bits, dtype):
    """A NaN that some rows of a tile see and others do not, in one CTA's share."""
    n, rows, window, sinks = 2000, 40, 1200, 5
    f = Filled(pkg, [n], kv=1, bits=bits, layers=1, seed=8, width=128)
    p = n - rows - window + 21  # seen by rows 0 to 20
    pool = f.host.copy()
    page, r = f.table[0, p // 32], p % 32
    if bits == 16:
        pool.view(np.uint16).reshape(-1, 1, 2, 1, 32, 128)[page, 0, 1, 0, r, 5] = 0x7fc0
    else:
        pool[page, 0, 1, 0, 32 * 64 + r * 8: 32 * 64 + r * 8 + 2] = np.array([0x7fc0], np.uint16).view(np.uint8)
    f.cache.pool.copy_(torch.from_numpy(pool.reshape(-1)))
    q = rand_q(rows, 2, dtype)
    starts = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    out = f.cache.attend(0, q, window=window, sinks=sinks, row_start=starts)
    hit = torch.isnan(out)
    assert hit[:21, :, 5].all() and not hit[21:].any() and not hit[..., 64:].any()


def test_rows_wide_window_long(pkg):
    n, r = 1100, 300
    for bits in (16, 4):
        f = Filled(pkg, [n], kv=1, bits=bits, layers=1, seed=bits)
        q = rand_q(r, 2, BF16)
        starts = torch.tensor([0, r], dtype=torch.int32, device=DEV)
        for window, sinks in ((0, 0), (500, 20)):
            out = f.cache.attend(0, q, window=window, sinks=sinks, row_start=starts)
            check_rows(out, q, [(0, n, 0, r)], f, 0, window, sinks)


# ---- what lies in masked places, and what is missing
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rows", [1, 40])
def test_masked_places_do_not_reach_the_output(pkg, bits, rows):
    """NaN and infinities behind the window, past the row and in free pages."""
    n = 200
    f = Filled(pkg, [n], kv=1, bits=bits, layers=1, seed=9)
    window, sinks = 30, 4
    first = n - rows - window + 1  # nothing in [sinks, first) is seen by any of the rows
    pool = f.host.copy()
    for p in range(sinks, first):
        page, r = f.table[0, p // 32], p % 32
        if bits == 16:
            bad = [0x7f80, 0xff80, 0x7fc0, 0xff7f][p % 4]  # inf, -inf, NaN, the lowest value
            pool.view(np.uint16).reshape(-1, 1, 2, 1, 32, 128)[page, :, :, :, r] = bad
        else:
            pool[page, ..., 32 * 64 + r * 8: 32 * 64 + r * 8 + 8] = np.array(
                [0x7f80, 0xff80, 0x7fc0, 0x7f7f], np.uint16).view(np.uint8)
    f.cache.pool.copy_(torch.from_numpy(pool.reshape(-1)))
    for dtype in (F32, BF16):
        q = rand_q(rows, 2, dtype)
        starts = torch.tensor([0, rows], dtype=torch.int32, device=DEV) if rows > 1 else None
        out = f.cache.attend(0, q, window=window, sinks=sinks, row_start=starts)
        assert torch.isfinite(out).all()
        check_rows(out, q, [(0, n, 0, rows)], f, 0, window, sinks)


@pytest.mark.parametrize("bits", [16, 4])
def test_values_seen_propagate(pkg, bits):
    f = Filled(pkg, [50, 50], kv=1, bits=bits, layers=1, seed=4)
    pool = f.host.copy()
    page = f.table[0, 0]
    if bits == 16:
        pool.view(np.uint16).reshape(-1, 1, 2, 1, 32, 128)[page, 0, 1, 0, 3, 5] = 0x7fc0
    else:
        pool[page, 0, 1, 0, 32 * 64 + 3 * 8: 32 * 64 + 3 * 8 + 2] = np.array([0x7fc0], np.uint16).view(np.uint8)
    f.cache.pool.copy_(torch.from_numpy(pool.reshape(-1)))
    for rows in (1, 20):
        q = rand_q(2 * rows, 2, F32)
        starts = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=DEV)
        out = f.cache.attend(0, q, row_start=starts)
        hit = torch.isnan(out[:rows])
        assert hit[..., 5].all() and not torch.isnan(out[rows:]).any()
        assert not hit[..., 64:].any()  # other dims (other groups of 32) stay


@pytest.mark.parametrize("bits", [16, 4])
def test_missing_pages_are_not_seen(pkg, bits):
    f = Filled(pkg, [200, 40], kv=2, bits=bits, seed=6)
    f.table[0, 1] = f.table[0, 3] = -1
    f.table[1, :] = -1
    f.cache.page_table.copy_(torch.from_numpy(f.table))
    for rows in (1, 70):
        q = rand_q(rows + 1, 4, F32)
        starts = torch.tensor([0, rows, rows + 1], dtype=torch.int32, device=DEV)
        out = f.cache.attend(1, q, row_start=starts)
        check_rows(out, q, [(0, 200, 0, rows), (1, 40, rows, rows + 1)], f, 1, 0, 0)
        # a window that only covers missing pages
        out = f.cache.attend(1, q[:1].contiguous(), window=1,
                             seqs=torch.tensor([1], dtype=torch.int32, device=DEV))
        assert not out.any()
    f.cache.check()


@pytest.mark.parametrize("bits", [16, 4])
def test_bad_device_values_are_skipped_and_reported(pkg, bits):
    """Indices out of range in device arrays: recorded, nothing read or
    written through them (the bounds are checked in the kernels)."""
    f = Filled(pkg, [64, 64, 64], kv=1, bits=bits, layers=1, seed=2)
    c = f.cache
    q = rand_q(3, 2, F32)

    def broken(bad_table=None, bad_len=None, seqs=None):
        t, n = f.table.copy(), np.array(f.lens, np.int32)
        if bad_table is not None:
            t[1, 0] = bad_table
        if bad_len is not None:
            n[1] = bad_len
        c.page_table.copy_(torch.from_numpy(t))
        c.lengths.copy_(torch.from_numpy(n))
        s = torch.tensor(seqs, dtype=torch.int32, device=DEV) if seqs else None
        out = c.attend(0, q, seqs=s)
        with pytest.raises(pkg.CudaError, match="out of range"):
            c.check()
        c.check()  # cleared
        c.page_table.copy_(torch.from_numpy(f.table))
        c.lengths.copy_(torch.from_numpy(np.array(f.lens, np.int32)))
        check_rows(out, q, [(0, 64, 0, 1), (2, 64, 2, 3)], f, 0, 0, 0)
        return out

    for page in (f.host.shape[0], 1 << 30, -2, -(1 << 31)):
        out = broken(bad_table=page)
        g = f.table.copy()
        f.table[1, 0] = -1  # as if it had no page
        check_rows(out, q, [(1, 64, 1, 2)], f, 0, 0, 0)
        f.table = g
    for n in (65, 1 << 30, -1):
        assert not broken(bad_len=n)[1].any()
    for s in (3, -1, 1 << 30):
        assert not broken(seqs=[0, s, 2])[1].any()
    # appends through them touch nothing
    before = c.pool.clone()
    c.page_table[1, 1] = f.host.shape[0] + 5
    k = rand_q(1, 1, F32)
    c.append(0, k, k, seqs=torch.tensor([1], dtype=torch.int32, device=DEV))
    c.append(0, k, k, seqs=torch.tensor([9], dtype=torch.int32, device=DEV))
    c.lengths[2] = 0
    c.append(0, k, k, seqs=torch.tensor([2], dtype=torch.int32, device=DEV))
    assert torch.equal(c.pool, before)
    with pytest.raises(pkg.CudaError):
        c.check()


def test_row_start_out_of_order(pkg):
    f = Filled(pkg, [64, 64], kv=1, layers=1)
    q = rand_q(6, 2, F32)
    for starts in ([0, 9, 4], [5, 3, 6], [-4, 2, 100], [3, 3, 3]):
        out = torch.zeros_like(q)
        f.cache.attend(0, q, out=out, row_start=torch.tensor(starts, dtype=torch.int32, device=DEV))
        assert torch.isfinite(out).all()
    try:
        f.cache.check()
    except pkg.CudaError:
        pass


# ---- strides, addresses, streams, graphs, sizes
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [1, 50])
def test_strides_and_alignment(pkg, dtype, rows):
    f = Filled(pkg, [rows + 60], kv=2, bits=4, seed=3)
    starts = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    q = rand_q(rows, 4, dtype)
    want = f.cache.attend(1, q, row_start=starts)
    fused = torch.zeros(rows, 10, 128, dtype=dtype, device=DEV)  # q | k | v of one projection
    fused[:, 2:6] = q
    odd = torch.zeros(rows * 4 * 129 + 1, dtype=dtype, device=DEV)[1:].view(rows, 4, 129)[..., :128]
    odd.copy_(q)
    head_major = q.transpose(0, 1).contiguous().transpose(0, 1)
    for other in (fused[:, 2:6], odd, head_major):
        out = torch.zeros(rows * 4 * 131 + 1, dtype=dtype, device=DEV)[1:].view(rows, 4, 131)
        f.cache.attend(1, other, row_start=starts, out=out[..., :128])
        assert torch.equal(out[..., :128], want) and not out[..., 128:].any()
    # one row broadcast to many (stride 0)
    wide = q[:1].expand(rows, 4, 128)
    assert torch.equal(f.cache.attend(1, wide, row_start=starts),
                       f.cache.attend(1, wide.contiguous(), row_start=starts))


def test_python_refusals(pkg):
    f = Filled(pkg, [40, 40], kv=2)
    c = f.cache
    q = rand_q(2, 4, F32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    bad = pkg.InvalidInput
    for call in (
        lambda: c.attend(0, q.half()), lambda: c.attend(0, q[..., :64]), lambda: c.attend(0, q[0]),
        lambda: c.attend(0, q.cpu()), lambda: c.attend(0, q[:, :3].contiguous()),
        lambda: c.attend(5, q), lambda: c.attend(2 ** 32, q), lambda: c.attend(0, q, window=-1),
        lambda: c.attend(0, q, out=q.to(BF16)), lambda: c.attend(0, q, seqs=i32([0])),
        lambda: c.attend(0, q, seqs=i32([0, 1]).long()), lambda: c.attend(0, q, row_start=i32([])),
        lambda: c.attend(0, q, seqs=i32([0, 1]).cpu()), lambda: c.attend(0, rand_q(3, 4, F32)),
        lambda: c.attend(0, q, window=2 ** 33), lambda: c.append(0, q[:, :2], q[:, :1]),
        lambda: c.append(0, q, q), lambda: c.append(0, q[:, :2], q[:, :2].to(BF16)),
        lambda: c.read(0, -1), lambda: c.read(0, 1, dtype=torch.float16),
        lambda: c.free([2]), lambda: c.free([0, 0]), lambda: c.free([2 ** 40]),
        lambda: c.fork([0], [0]), lambda: c.resize([0], [1, 2]), lambda: c.free([0.5]),
        lambda: c.evict([0], 0),
    ):
        with pytest.raises(bad):
            call()
    with pytest.raises(bad, match="bytes"):
        pkg.KvCache(c.pool[:-1], c.page_table, c.lengths, c.refs, layers=2, kv_heads=2)
    with pytest.raises(bad, match="aligned"):
        c2 = pkg.KvCache(torch.zeros(c.pool.numel() + 8, dtype=torch.uint8, device=DEV)[8:],
                         c.page_table, c.lengths, c.refs, layers=2, kv_heads=2)
        c2.attend(0, q)
    # empty calls
    assert c.attend(0, q[:0]).shape == (0, 4, 128)
    c.append(0, q[:0, :2], q[:0, :2])
    assert c.read(0, 0)[0].shape == (0, 2, 128)
    c.free([])
    c.resize([], [])
    c.fork([], [])
    c.check()


def test_other_streams(pkg):
    f = Filled(pkg, [300, 200], kv=2, bits=4, seed=8)
    q = rand_q(2, 4, F32)
    want = f.cache.attend(1, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:  # reads of one cache on several streams at once
            with torch.cuda.stream(s):
                outs.append(f.cache.attend(1, q))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_two_threads(pkg):
    import threading

    f = Filled(pkg, [300, 200], kv=2, bits=16, seed=8)
    qs = [rand_q(2, 4, F32, s) for s in range(4)]
    want = [f.cache.attend(1, q, window=50 + i) for i, q in enumerate(qs)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                o = f.cache.attend(1, qs[i], window=50 + i)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(o, want[i]):
                    bad.append(i)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_steps(pkg, bits):
    """append + attend captured once; replays follow the lengths, tables and
    rows on the device."""
    lens = [20, 50]
    f = Filled(pkg, lens, kv=2, bits=bits, layers=1, width=6, spare=20, seed=5)
    c = f.cache
    c.resize([0, 1], [100, 100])
    k, v, q = rand_q(2, 2, F32, 1), rand_q(2, 2, F32, 2), rand_q(2, 4, F32, 3)
    out = torch.zeros_like(q)
    c.append(0, k, v)  # warm-up
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.append(0, k, v)
        c.attend(0, q, window=40, sinks=3, out=out)
    f.host = c.pool.cpu().numpy().reshape(f.host.shape)
    f.table = c.page_table.cpu().numpy()
    for step in range(6):
        n = [21 + step, 51 + 2 * step]
        c.lengths.copy_(torch.tensor(n, dtype=torch.int32))
        for t, s in ((k, 10), (v, 20), (q, 30)):
            t.copy_(rand_q(t.shape[0], t.shape[1], F32, s + step))
        g.replay()
        torch.cuda.synchronize()
        f.host = c.pool.cpu().numpy().reshape(f.host.shape)
        check_rows(out, q, [(0, n[0], 0, 1), (1, n[1], 1, 2)], f, 0, 40, 3)
        kk, vv, _ = f.dense(0, 0, n[0])
        want = k[0].cpu().numpy().astype(np.float64)
        if bits == 4:
            want = O.quantise_fast(want)
        else:
            want = k[0].to(BF16).double().cpu().numpy()
        assert np.array_equal(kk[n[0] - 1], want)
    c.check()


FIRST_IN_A_GRAPH = """
import torch
from __graft_entry__ import load_package
pkg = load_package()
cs = [pkg.KvCache.allocate(2, 4096, layers=1, kv_heads=1, kv_bits=b) for b in (16, 4)]
for c in cs:
    c.resize([0, 1], [700, 90])
    c.pool.zero_()
torch.cuda.synchronize()
out = []
g = torch.cuda.CUDAGraph()
starts = torch.tensor([0, 40, 80], dtype=torch.int32, device="cuda")
qs = [torch.randn(80, 2, 128, device="cuda").to(t) for t in (torch.float32, torch.bfloat16)]
with torch.cuda.graph(g):  # no kernel of these has run in this process
    for c in cs:
        for q in qs:
            out += [c.attend(0, q, row_start=starts), c.attend(0, q[:2].contiguous())]
g.replay()
torch.cuda.synchronize()
assert all(not t.any() for t in out)
for c in cs:
    c.check()
print("fine")
"""


def test_first_calls_may_be_captured(pkg):
    import subprocess
    import sys
    from pathlib import Path

    r = subprocess.run([sys.executable, "-c", FIRST_IN_A_GRAPH], capture_output=True, text=True,
                       timeout=300, cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_repeats_are_bitwise_equal(pkg):
    f = Filled(pkg, [3000, 1000], kv=2, bits=4, layers=1, seed=1)
    for rows in (1, 300):
        q = rand_q(2 * rows, 4, F32)
        starts = torch.tensor([0, rows, 2 * rows], dtype=torch.int32, device=DEV)
        a = [f.cache.attend(0, q, row_start=starts) for _ in range(4)]
        assert all(torch.equal(a[0], x) for x in a[1:])


@pytest.mark.parametrize("bits", [16, 4])
def test_offsets_past_32_bits(pkg, bits):
    """Pages beyond 4 GiB of pool."""
    layers, kv, ps = 28, 8, 64
    page = layers * 2 * kv * ps * (256 if bits == 16 else 72)
    pages = (9 << 30) // page
    n = 150
    c = pkg.KvCache.allocate(2, 256, layers=layers, kv_heads=kv, pages=pages, page_size=ps,
                             kv_bits=bits)
    assert c.pool_bytes > 1 << 33
    top = torch.tensor([[pages - 1, pages - 3, pages - 2, -1], [0, 1, 2, -1]], dtype=torch.int32)
    c.page_table.copy_(top)
    c.lengths.fill_(n)
    c.refs[[pages - 1, pages - 2, pages - 3, 0, 1, 2]] = 1
    k, v = rand_q(n, kv, F32, 1), rand_q(n, kv, F32, 2)
    starts = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    high = torch.tensor([0], dtype=torch.int32, device=DEV)
    for layer in (0, 27):
        c.append(layer, k, v, row_start=starts, seqs=high)
        c.append(layer, k, v, row_start=starts, seqs=high + 1)
        a = c.read(layer, n, row_start=starts, seqs=high)
        b = c.read(layer, n, row_start=starts, seqs=high + 1)
        want = k.to(BF16).float() if bits == 16 else torch.from_numpy(
            O.quantise_fast(k.cpu().numpy())).float().to(DEV)
        assert torch.equal(a[0], want) and torch.equal(b[0], want) and torch.equal(a[1], b[1])
        for rows in (1, 40):
            q = rand_q(rows, 16, BF16)
            st = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
            x = c.attend(layer, q, row_start=st, seqs=high)
            assert torch.equal(x, c.attend(layer, q, row_start=st, seqs=high + 1))
    # compaction brings them down
    want = c.attend(27, q, row_start=st, seqs=high)
    c.free([1])
    c.compact()
    assert c.page_table[0].tolist() == [2, 0, 1, -1]
    assert torch.equal(c.attend(27, q, row_start=st, seqs=high), want)
    c.check()


# ---- storing and loading rows
def test_quantise_is_exact(pkg):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((64, 128)).astype(np.float32)
    x[0] = 0.0
    x[1, :32] = np.arange(32) * 0.25           # halves of the step: ties
    x[1, 31] = 7.0
    x[2, :32] = np.linspace(-3, 3, 32)
    x[2, 31] = 7.0 * 1.00390625                # amax / 7 on a bf16 midpoint
    x[3, :32] = np.linspace(-3, 3, 32)
    x[3, 31] = np.nextafter(np.float32(7.0 * 1.00390625), np.float32(0))
    x[4, :32] *= np.float32(1e-38)
    x[5, :32] *= np.float32(3e37)
    x[6, :32] = np.float32(1e-45) * np.arange(32)
    x[7, 5], x[7, 40], x[7, 70] = np.nan, np.inf, -np.inf
    x[8, :32] = 2.0 ** -130 * np.arange(32)
    x[9] = -np.abs(x[9])
    for i in range(10, 40):                    # ties of n at random scales
        s = np.float32(float(torch.tensor(float(rng.uniform(0.1, 2))).to(BF16)))
        x[i, :32] = (rng.integers(-7, 7, 32) + 0.5) * s
        x[i, 0] = 7 * s
    c = pkg.KvCache.allocate(1, 64, layers=1, kv_heads=1, kv_bits=4)
    c.resize([0], [64])
    t = torch.from_numpy(x).to(DEV)[:, None]
    starts = torch.tensor([0, 64], dtype=torch.int32, device=DEV)
    c.append(0, t, t.flip(0).contiguous(), row_start=starts)
    k, v = c.read(0, 64, row_start=starts)
    assert torch.equal(torch.nan_to_num(k, 9e9), torch.nan_to_num(v.flip(0), 9e9))
    got = k[:, 0].cpu().numpy().astype(np.float64)
    pool = c.pool.cpu().numpy().reshape(-1, 1, 2, 1, 32 * 72)
    for i in range(64):
        n, s = O.quantise_row(x[i])
        want = n * np.repeat(s, 32)
        assert np.array_equal(got[i], want.astype(np.float32), equal_nan=True), i
        page = int(c.page_table[0, i // 32])
        code = pool[page, 0, 0, 0, (i % 32) * 64: (i % 32 + 1) * 64]
        for d in range(128):
            b, sh = O.code_place(d)
            assert (code[b] >> sh) & 15 == n[d] + 8
    c.check()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_read_ragged(pkg, bits, dtype):
    lens, counts = [40, 0, 70, 33], [40, 0, 5, 1]
    f = Filled(pkg, lens, kv=3, bits=bits, layers=2, seed=11)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=DEV)
    total = sum(counts)
    fused = rand_q(total + 3, 8, dtype)
    k, v = fused[:, 1:4], fused[:, 5:8]
    before = f.cache.pool.clone()
    f.cache.append(1, k, v, row_start=starts)
    a, b = f.cache.read(1, total + 3, dtype=dtype, row_start=starts)
    for got, src in ((a, k), (b, v)):
        x = src[:total].double().cpu().numpy()
        want = O.quantise_fast(x) if bits == 4 else src[:total].to(BF16).double().cpu().numpy()
        assert torch.equal(got[:total], torch.from_numpy(want).to(dtype).to(DEV))
    # nothing but those rows of that layer changed
    page = f.cache.pool_bytes // f.host.shape[0]
    now, was = (p.cpu().numpy().reshape(f.host.shape) for p in (f.cache.pool, before))
    assert page == now[0].size and np.array_equal(now[:, 0], was[:, 0])
    row = 256 if bits == 16 else 64
    written = set()
    for s, (n, r) in enumerate(zip(lens, counts)):
        written |= {(int(f.table[s, p // 32]), p % 32) for p in range(n - r, n)}
    for pg in range(now.shape[0]):
        for r in range(32):
            same = np.array_equal(now[pg, 1, :, :, r * row: (r + 1) * row],
                                  was[pg, 1, :, :, r * row: (r + 1) * row])
            assert same == ((pg, r) not in written)
    f.cache.check()


def test_append_names_a_sequence_twice(pkg):
    f = Filled(pkg, [33, 5], kv=1, bits=4, layers=1)
    k = rand_q(3, 1, F32)
    seqs = torch.tensor([0, 1, 0], dtype=torch.int32, device=DEV)
    for _ in range(5):
        f.cache.append(0, k, k, seqs=seqs)
    a, _ = f.cache.read(0, 2)
    want = O.quantise_fast(k.cpu().numpy())
    assert np.array_equal(a[0].cpu().numpy(), want[2]) and np.array_equal(a[1].cpu().numpy(), want[1])


def test_read_without_pages(pkg):
    f = Filled(pkg, [64], kv=1, bits=16, layers=1)
    f.cache.page_table[0, 0] = -1
    starts = torch.tensor([0, 70], dtype=torch.int32, device=DEV)  # six rows before position 0
    k, v = f.cache.read(0, 70, row_start=starts)
    assert not k[:38].any() and not v[:38].any() and k[38:].any(-1).all()
    f.cache.check()


# ---- pages
def pattern(c, pages):
    """Fills page p of the pool with 16-byte units that name it."""
    per = c.pool_bytes // pages // 16
    ids = torch.arange(pages, device=DEV, dtype=torch.int32)
    unit = torch.arange(per, device=DEV, dtype=torch.int32)
    x = torch.stack((ids[:, None].expand(pages, per), unit.expand(pages, per),
                     ids[:, None] * 7 + unit, ids[:, None] ^ unit), -1).contiguous()
    c.pool[: c.pool_bytes].copy_(x.view(torch.uint8).reshape(-1))


def page_ids(c, pages):
    """Which pattern each page holds (whole, or the test fails)."""
    per = c.pool_bytes // pages // 16
    x = c.pool[: c.pool_bytes].view(torch.int32).reshape(pages, per, 4)
    ids, unit = x[:, 0, 0].clone(), torch.arange(per, device=DEV, dtype=torch.int32)
    want = torch.stack((ids[:, None].expand(pages, per), unit.expand(pages, per),
                        ids[:, None] * 7 + unit, ids[:, None] ^ unit), -1)
    assert torch.equal(x, want)
    return ids.tolist()


def same_state(c, o):
    assert c.page_table.tolist() == o.table
    assert c.lengths.tolist() == o.lengths
    assert c.refs.tolist() == o.refs
    assert page_ids(c, len(o.refs)) == o.data


@pytest.mark.parametrize("seed", range(12))
def test_page_calls_follow_the_oracle(pkg, seed):
    rng = np.random.default_rng(seed)
    seqs, width = int(rng.integers(2, 12)), int(rng.integers(1, 40))
    ps = int(rng.choice([16, 32, 64]))
    pages = int(rng.integers(2, seqs * width + 3))
    bits = int(rng.choice([16, 4]))
    c = pkg.KvCache.allocate(seqs, width * ps, layers=int(rng.integers(1, 4)),
                             kv_heads=int(rng.integers(1, 4)), pages=pages, page_size=ps,
                             kv_bits=bits)
    o = O.Cache(pages, seqs, width, ps)
    pattern(c, pages)
    o.data = list(range(pages))
    failures = 0
    for step in range(40):
        s = rng.permutation(seqs)[: rng.integers(1, seqs + 1)].tolist()
        kind = int(rng.integers(0, 6))
        ok = True
        if kind in (0, 1):
            n = [int(rng.integers(0, width * ps + 1)) for _ in s]
            c.resize(s, n)
            ok = o.resize(s, n)
        elif kind == 2 and len(s) > 1:
            src = [int(rng.choice(s[: len(s) // 2])) for _ in s[len(s) // 2:]]
            c.fork(src, s[len(s) // 2:])
            ok = o.fork(src, s[len(s) // 2:])
        elif kind == 3:
            c.free(s)
            o.free(s)
        elif kind == 4:
            w, k = int(rng.integers(1, 3 * ps)), int(rng.integers(0, 2 * ps))
            c.evict(s, w, k)
            o.evict(s, w, k)
        else:
            c.compact()
            o.compact()
        if ok:
            c.check()
        else:
            failures += 1
            with pytest.raises(pkg.InvalidInput, match="free pages") as e:
                c.check()
            assert e.value.code == pkg.engine.ERR_CACHE_FULL
        same_state(c, o)


def test_page_calls_many_pages(pkg):
    """More pages than one pass of the block scans, more sequences than warps."""
    pages, seqs, width, ps = 5000, 300, 40, 16
    rng = np.random.default_rng(1)
    c = pkg.KvCache.allocate(seqs, width * ps, layers=1, kv_heads=1, pages=pages, page_size=ps,
                             kv_bits=4)
    o = O.Cache(pages, seqs, width, ps)
    pattern(c, pages)
    o.data = list(range(pages))
    everyone = list(range(seqs))
    for step in range(3):
        n = [int(x) for x in rng.integers(0, 260, seqs)]
        c.resize(everyone, n)
        assert o.resize(everyone, n)
        same_state(c, o)
        gone = rng.permutation(seqs)[:100].tolist()
        c.free(gone)
        o.free(gone)
        src = [s for s in everyone if s not in gone][:50]
        c.fork(src, gone[:50])
        assert o.fork(src, gone[:50])
        same_state(c, o)
        c.compact()
        o.compact()
        same_state(c, o)
    c.check()


def test_shared_tail_is_copied_before_growth(pkg):
    """A sequence cut back into a shared page and grown again."""
    c = pkg.KvCache.allocate(3, 128, layers=1, kv_heads=1, page_size=32, kv_bits=16)
    o = O.Cache(12, 3, 4, 32)
    pattern(c, 12)
    o.data = list(range(12))
    for call in (("resize", [0], [96]), ("fork", [0, 0], [1, 2]), ("resize", [1, 2], [40, 50]),
                 ("resize", [1, 2], [60, 51]), ("resize", [0], [10]), ("resize", [0, 1], [12, 64])):
        getattr(c, call[0])(*call[1:])
        assert getattr(o, call[0])(*call[1:])
        same_state(c, o)
    c.check()


def test_page_calls_in_a_graph(pkg):
    c = pkg.KvCache.allocate(4, 64, layers=1, kv_heads=1, page_size=16)
    o = O.Cache(16, 4, 4, 16)
    pattern(c, 16)
    o.data = list(range(16))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    calls = [("resize", [0, 1], [40, 20]), ("fork", [0], [2]), ("free", [0]), ("compact",),
             ("resize", [3], [64])]
    with torch.cuda.graph(g):
        for name, *a in calls:
            getattr(c, name)(*a)
    assert c.lengths.tolist() == [0, 0, 0, 0]
    for _ in range(3):
        g.replay()
        for name, *a in calls:
            getattr(o, name)(*a)
        same_state(c, o)
    c.check()


# ---- a run of them together
@pytest.mark.parametrize("bits", [16, 4])
def test_a_serving_run(pkg, bits):
    """A prompt is stored, forked into takes that each go on with rows of their
    own under a window, pages behind it are given back, one take ends, the
    pages are compacted, another starts from the prompt; every output against
    the rows each take has seen."""
    window, sinks, layers, kv, heads = 40, 5, 2, 2, 4
    c = pkg.KvCache.allocate(4, 256, layers=layers, kv_heads=kv, pages=14, page_size=16,
                             kv_bits=bits)
    rng = np.random.default_rng(bits)
    rows = {s: [] for s in range(4)}  # per sequence: [layers][2][kv][128] of every position

    def held(x):
        x = np.asarray(x, np.float64)
        return O.quantise_fast(x) if bits == 4 else torch.from_numpy(x).to(BF16).double().numpy()

    def step(seqs, counts):
        c.resize(seqs, [len(rows[s]) + n for s, n in zip(seqs, counts)])
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        new = rng.standard_normal((int(starts[-1]), layers, 2, kv, 128)).astype(np.float32)
        st, sq = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (starts, seqs))
        t = torch.from_numpy(new).to(DEV)
        for i, s in enumerate(seqs):
            rows[s] = rows[s] + list(held(new[starts[i]: starts[i + 1]]))
        for l in range(layers):
            c.append(l, t[:, l, 0], t[:, l, 1], row_start=st, seqs=sq)
            q = rand_q(int(starts[-1]), heads, F32, int(rng.integers(1 << 20)))
            out = c.attend(l, q, window=window, sinks=sinks, row_start=st, seqs=sq)

            def dense(s, n):
                a = np.stack([r[l] for r in rows[s]])
                return a[:, 0], a[:, 1], np.ones(n, bool)

            check_rows(out, q, [(s, len(rows[s]), int(starts[i]), int(starts[i + 1]))
                                for i, s in enumerate(seqs)], None, l, window, sinks, dense=dense)

    step([0], [37])
    c.fork([0, 0], [1, 2])
    rows[1], rows[2] = list(rows[0]), list(rows[0])
    for n in range(12):
        step([0, 1, 2], [1 + n % 3, 2, 1])
        c.evict([0, 1, 2], window, sinks)
    step([1], [50])
    c.evict([1], window, sinks)
    c.free([0])
    c.compact()
    rows[0] = []
    c.check()
    used = int((c.refs > 0).sum())
    assert (c.refs[:used] > 0).all() and int(c.page_table.max()) == used - 1
    step([2, 1], [3, 1])
    c.fork([2], [3])
    rows[3] = list(rows[2])
    step([3, 2], [20, 1])
    step([0], [30])
    c.check()
