"""Paged key / value caches without a GPU: what the C entry points refuse, the
index arithmetic of the layout, and the oracle's own consistency."""
import ctypes as C
import random
import subprocess
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest

from oracle import kv as O

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "qwen3-tts-hip_b200" / "csrc"

# Addresses that are never followed: every call here is refused, or has no
# rows, before anything reaches a device.
P = 1 << 20


@pytest.fixture(scope="module")
def kv(pkg):
    return pkg.kv


def cache(kv, **over):
    f = dict(pool=P, page_table=P, lengths=P, refs=P, work=P, device=0, pages=8, seqs=4,
             max_pages=3, layers=2, kv_heads=2, page_size=32, bits=16)
    f.update(over)
    return kv._Cache(*[f[n] for n, _ in kv._Cache._fields_])


def rows(kv, **over):
    f = dict(seqs=None, row_start=None, groups=0, rows=0, max_rows=0, max_length=0)
    f.update(over)
    order = ("seqs", "row_start", "groups", "rows", "max_rows", "max_length")
    return kv._ROWS.pack(*[f[n] or 0 for n in order])


def attend(pkg, kv, c=None, r=None, layer=0, q=P, out=P, dtype=0, heads=2, scale=0.1, window=0,
           sinks=0, stride=128):
    return pkg.lib().qtts_kv_attend(
        C.byref(c) if c is not None else None, layer, r, q,
        2 * stride, stride, out, 2 * stride, stride, dtype, heads, scale, window, sinks, None)


def refused(pkg, status, words):
    assert status == pkg.engine.ERR_INVALID_INPUT
    assert words in pkg.lib().qtts_last_error().decode()


@pytest.mark.parametrize("over,words", [
    ({"pages": 0}, "pages"), ({"seqs": -1}, "seqs"), ({"max_pages": 0}, "max_pages"),
    ({"layers": 0}, "layers"), ({"kv_heads": 0}, "kv_heads"), ({"kv_heads": 2000}, "kv_heads"),
    ({"bits": 8}, "bits"), ({"page_size": 24}, "page_size"), ({"page_size": 8}, "page_size"),
    ({"page_size": 512}, "page_size"), ({"max_pages": 1 << 30}, "exceeds"),
    ({"pages": (1 << 28) + 1}, "pages"), ({"pool": None}, "pool"), ({"pool": P + 8}, "aligned"),
    ({"page_table": None}, "page_table"), ({"lengths": None}, "lengths"), ({"work": None}, "work"),
])
def test_bad_caches_are_refused(pkg, kv, over, words):
    refused(pkg, attend(pkg, kv, cache(kv, **over), rows(kv)), words)


def test_sizes(pkg, kv):
    a, b = C.c_size_t(), C.c_size_t()
    for bits, row in ((16, 256), (4, 72)):
        c = cache(kv, bits=bits, pool=None, page_table=None, lengths=None, refs=None, work=None)
        assert pkg.lib().qtts_kv_sizes(C.byref(c), C.byref(a), C.byref(b)) == 0
        assert a.value == 8 * 2 * 2 * 2 * 32 * row
        assert b.value >= 3 * 8
    refused(pkg, pkg.lib().qtts_kv_sizes(None, C.byref(a), C.byref(b)), "cache")


@pytest.mark.parametrize("over,words", [
    ({"groups": -1}, "negative"), ({"rows": 2, "groups": 1}, "row_start"),
    ({"groups": 5, "rows": 5}, "exceeds"), ({"max_rows": -1}, "negative"),
    ({"max_length": -1}, "negative"),
])
def test_bad_rows_are_refused(pkg, kv, over, words):
    refused(pkg, attend(pkg, kv, cache(kv), rows(kv, **over)), words)
    refused(pkg, attend(pkg, kv, cache(kv)), "rows")


@pytest.mark.parametrize("over,words", [
    ({"layer": 2}, "layer"), ({"layer": -1}, "layer"), ({"heads": 3}, "q_heads"),
    ({"heads": 0}, "q_heads"), ({"scale": float("nan")}, "scale"),
    ({"scale": float("inf")}, "scale"), ({"window": -1}, "window"), ({"sinks": -1}, "sinks"),
    ({"dtype": 2}, "dtype"), ({"q": None}, "q"), ({"out": None}, "out"), ({"q": P + 2}, "aligned"),
    ({"stride": 1 << 41}, "stride"), ({"q": P, "out": P}, "overlap"),
])
def test_bad_attend_arguments_are_refused(pkg, kv, over, words):
    refused(pkg, attend(pkg, kv, cache(kv), rows(kv, groups=1, rows=1), **over), words)


def test_append_and_read_refusals(pkg, kv):
    L = pkg.lib()
    for f in (L.qtts_kv_append, L.qtts_kv_read):
        r, c = rows(kv, groups=1, rows=1), cache(kv)
        a = [C.byref(c), 0, r, P, 256, 128, P, 256, 128, 0, None]
        for i, bad, words in ((1, 2, "layer"), (3, None, "k"), (6, None, "v"), (9, 7, "dtype"),
                              (6, P + 1, "aligned")):
            refused(pkg, f(*[bad if j == i else x for j, x in enumerate(a)]), words)
        # no rows: nothing to do, nothing refused
        r = rows(kv)
        assert f(C.byref(c), 0, r, None, 0, 0, None, 0, 0, 0, None) == 0


def ints(*v):
    return (C.c_int32 * max(1, len(v)))(*v)


def test_page_call_refusals(pkg, kv):
    L = pkg.lib()
    c = cache(kv)
    big = ints(*[0] * 1025)
    refused(pkg, L.qtts_kv_free(C.byref(c), ints(4), 1, None), "outside")
    refused(pkg, L.qtts_kv_free(C.byref(c), ints(-1), 1, None), "outside")
    refused(pkg, L.qtts_kv_free(C.byref(c), ints(1, 1), 2, None), "twice")
    refused(pkg, L.qtts_kv_free(C.byref(c), None, 1, None), "null")
    refused(pkg, L.qtts_kv_free(C.byref(c), big, 1025, None), "1024")
    refused(pkg, L.qtts_kv_resize(C.byref(c), ints(0, 0), ints(1, 2), 2, None), "twice")
    refused(pkg, L.qtts_kv_resize(C.byref(c), ints(0), ints(97), 1, None), "positions")
    refused(pkg, L.qtts_kv_resize(C.byref(c), ints(0), ints(-1), 1, None), "positions")
    refused(pkg, L.qtts_kv_resize(C.byref(c), ints(0), None, 1, None), "null")
    refused(pkg, L.qtts_kv_fork(C.byref(c), ints(0, 1), ints(1, 2), 2, None), "destination")
    refused(pkg, L.qtts_kv_fork(C.byref(c), ints(0, 0), ints(1, 1), 2, None), "twice")
    refused(pkg, L.qtts_kv_fork(C.byref(c), ints(9), ints(1), 1, None), "outside")
    refused(pkg, L.qtts_kv_evict(C.byref(c), ints(0), 1, 0, 0, None), "window")
    refused(pkg, L.qtts_kv_evict(C.byref(c), ints(0), 1, 4, -1, None), "sinks")
    none = cache(kv, refs=None)
    for status in (L.qtts_kv_compact(C.byref(none), None),
                   L.qtts_kv_free(C.byref(none), ints(0), 1, None)):
        refused(pkg, status, "refs")
    for f in (L.qtts_kv_free, ):
        assert f(C.byref(c), None, 0, None) == 0
    assert L.qtts_kv_resize(C.byref(c), None, None, 0, None) == 0
    assert L.qtts_kv_fork(C.byref(c), None, None, 0, None) == 0


def test_python_class_refuses_host_tensors(pkg):
    import torch

    t = torch.zeros(4, 3, dtype=torch.int32)
    with pytest.raises(pkg.InvalidInput, match="CUDA"):
        pkg.KvCache(torch.zeros(16, dtype=torch.uint8), t, t[:, 0].contiguous(),
                    torch.zeros(8, dtype=torch.int32), layers=1, kv_heads=1)
    with pytest.raises(pkg.InvalidInput, match="int32"):
        pkg.KvCache(torch.zeros(16, dtype=torch.uint8), t.long(), t[:, 0].contiguous(),
                    torch.zeros(8, dtype=torch.int32), layers=1, kv_heads=1)
    with pytest.raises(pkg.InvalidInput, match="positive"):
        pkg.KvCache.allocate(0, 10, layers=1, kv_heads=1)
    with pytest.raises(pkg.InvalidInput, match="page_size"):
        pkg.KvCache.allocate(1, 10, layers=1, kv_heads=1, page_size=5)


def test_structs_match_the_rust_binding():
    from test_rust_binding import _c_struct_fields, _rust_struct_fields

    for name in ("qtts_kv_cache", "qtts_kv_rows", "qtts_cache_options"):
        assert _c_struct_fields(name) == _rust_struct_fields(name), name


# ---- the layout's arithmetic, compiled for the host
PROBE = r"""
#include <cstdio>
#include <cstdlib>
#include <initializer_list>
#include "kv_layout.h"
using namespace qtts;
int main(int argc, char** argv) {
  KvGeom g{atoi(argv[1]), 1, atoi(argv[2]), atoi(argv[3]), atoi(argv[4]), atoi(argv[5]), atoi(argv[6])};
  printf("%lld %lld %lld\n", kv_page_bytes(g), kv_tile_bytes(g), kv_capacity(g));
  const int ps = 1 << g.shift;
  // every tile of the first and last page, in order and without gaps or overlap
  for (int page : {0, g.pages - 1}) {
    long long at = page * kv_page_bytes(g);
    for (int l = 0; l < g.layers; ++l)
      for (int w = 0; w < 2; ++w)
        for (int h = 0; h < g.kv_heads; ++h) {
          if (kv_tile_at(g, page, l, w, h) != at) return 1;
          at += kv_tile_bytes(g);
        }
    if (at != (page + 1LL) * kv_page_bytes(g)) return 2;
  }
  // a row's bytes stay inside its tile
  for (int r = 0; r < ps; ++r) {
    const int bytes = g.bits == 16 ? 256 : 64;
    if (kv_row_at(g, r) != r * bytes) return 3;
    if (kv_row_at(g, r) + bytes > kv_tile_bytes(g)) return 4;
    if (g.bits == 4 && (kv_scale_at(g, r) < ps * 64 || kv_scale_at(g, r) + 8 > kv_tile_bytes(g)))
      return 5;
  }
  for (int d = 0; d < 128; d += 8) printf("%d ", kv_code_word_at(d));
  printf("\n");
  for (int pos : {0, 1, 5, 40, 41, 100})
    for (int window : {0, 1, 7, 41})
      for (int sinks : {0, 1, 9, 64}) {
        const KvSpan s = kv_span(pos, window, sinks);
        for (int k = 0; k <= pos + 2; ++k) {
          const bool in = k < s.sink_end || (k >= s.first && k <= pos);
          if (in != kv_sees(pos, k, window, sinks)) return 6;
        }
        if (s.sink_end > s.first || s.sink_end < 0 || s.first < 0) return 7;
      }
  for (int j = 0; j < 6; ++j)
    for (int len : {0, 1, 40, 70, 96})
      for (int window : {1, 8, 33})
        for (int sinks : {0, 1, 17}) {
          bool seen = false;  // by any row at or after the newest position
          for (int p = len > 0 ? len - 1 : 0; p < len + 200; ++p)
            for (int k = j * ps; k < (j + 1) * ps; ++k) seen |= k < len && kv_sees(p, k, window, sinks);
          if (kv_page_behind(j, g.shift, len, window, sinks) && seen) return 8;
        }
  return 0;
}
"""


@pytest.mark.parametrize("bits", [16, 4])
def test_layout_arithmetic(tmp_path, bits):
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    rng = random.Random(bits)
    for pages, layers, heads, shift in [(1, 1, 1, 4), (200000, 28, 8, 5)] + [
            (rng.randint(1, 1 << 20), rng.randint(1, 40), rng.randint(1, 16), rng.randint(4, 8))
            for _ in range(20)]:
        p = subprocess.run([str(exe), *map(str, (pages, 7, layers, heads, shift, bits))],
                           capture_output=True, text=True)
        assert p.returncode == 0, (p.returncode, pages, layers, heads, shift)
        page, tile, cap = map(int, p.stdout.split()[:3])
        row = 256 if bits == 16 else 72
        assert tile == row << shift and page == layers * 2 * heads * tile and cap == 7 << shift
        words = list(map(int, p.stdout.split()[3:]))
        assert words == [O.code_place(d)[0] for d in range(0, 128, 8)]


# ---- the oracle
def test_oracle_rounding():
    assert [O.nearest_even(Fraction(k, 2)) for k in range(6)] == [0, 0, 1, 2, 2, 2]
    rng = np.random.default_rng(0)
    import torch

    for x in np.concatenate([rng.standard_normal(200) ** 2, [1e-40, 3e-41, 2.0 ** -133, 0.0]]):
        x = np.float32(x)
        want = float(torch.tensor(x).to(torch.bfloat16))
        assert O.bf16_of(Fraction(float(x))) == want


def test_oracle_quantise_forms_agree():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 128)).astype(np.float32)
    # exact ties: amax = 7 * mid and halves of the step
    x[0, :32] = np.arange(32) * 0.25
    x[0, 31] = 7.0 * 1.00390625
    x[1, :] = 0.0
    fast = O.quantise_fast(x)
    for i in range(len(x)):
        n, s = O.quantise_row(x[i])
        assert np.array_equal(n * np.repeat(s, 32), fast[i])
        assert np.abs(n).max() <= 7


def test_oracle_pages_stay_consistent():
    rng = random.Random(3)
    for _ in range(30):
        c = O.Cache(rng.randint(3, 30), 5, 6, 16)
        c.data = list(range(len(c.data)))
        for _ in range(40):
            s = rng.sample(range(5), rng.randint(1, 3))
            k = rng.randrange(5)
            if k == 0:
                c.resize(s, [rng.randint(0, 96) for _ in s])
            elif k == 1 and len(s) > 1:
                c.fork([s[0]] * (len(s) - 1), s[1:])
            elif k == 2:
                c.free(s)
            elif k == 3:
                c.evict(s, rng.randint(1, 40), rng.randint(0, 20))
            else:
                c.compact()
            named = [p for r in c.table for p in r if p >= 0]
            assert [named.count(p) for p in range(len(c.refs))] == c.refs


def test_engine_cache_options(pkg, tmp_path):
    from qwen3_tts_hip_b200.engine import _CacheOptions

    o = _CacheOptions()
    pkg.lib().qtts_cache_options_default(C.byref(o))
    assert (o.max_cache_steps, o.kv_bits, o.window, o.sinks) == (512, 16, 0, 0)
    e = pkg.EngineOptions()
    assert (e.max_cache_steps, e.kv_bits, e.kv_window, e.kv_sinks) == (512, 16, 0, 0)
    for args, words in (((0, 128, 8), "kv_bits"), ((0, 128, 4, -1), "window"),
                        ((0, 128, 4, 8, -1), "sinks"), ((0, 128, 4, 0, 3), "sinks need"),
                        ((0, 0, 4), "max_cache_steps")):
        with pytest.raises(pkg.InvalidInput, match=words):
            pkg.HipTtsEngine.load_with_options(tmp_path, pkg.EngineOptions(*args))
    h = C.c_void_p()
    refused(pkg, pkg.lib().qtts_engine_load_with_cache(b"/tmp", 0, None, C.byref(h)), "cache")
