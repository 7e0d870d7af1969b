// Index arithmetic of the paged key / value caches, shared by the kernels and
// by host code (it compiles with a plain C++ compiler).
//
// A sequence's position p lives in logical page p / ps (ps = page size, a
// power of two from 16 to 256), row p % ps; the page table names the physical
// page. A physical page holds one tile of ps rows for every (layer, K or V,
// kv head), in that order.
//   16 bits: ps rows of 128 bf16.
//   4 bits:  ps rows of 64 code bytes, then ps rows of four bf16 scales, one
//            per group of 32 dims. Code n + 8 (n in -7..7) stands for n * scale.
//            32-bit word 4 t + g of a row's codes holds dims 32 g + 8 t .. + 7,
//            lowest nibble first, so that the lane t of a quad of lanes finds
//            its eight dims of each of the four groups in one 16-byte load.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define QTTS_HD __host__ __device__ __forceinline__
#else
#define QTTS_HD inline
#endif

namespace qtts {

constexpr int kKvDim = 128;           // head dim of every cache
constexpr int kKvGroup = 32;          // dims that share a scale (4 bits)
constexpr int kKvGroups = kKvDim / kKvGroup;
constexpr int kKvCodeBytes = kKvDim / 2;
constexpr int kKvMinShift = 4, kKvMaxShift = 8;

struct KvGeom {
  int pages, seqs, max_pages, layers, kv_heads, shift, bits;
};

QTTS_HD long long kv_tile_bytes(const KvGeom& g) {
  return (long long)(g.bits == 16 ? 2 * kKvDim : kKvCodeBytes + 2 * kKvGroups) << g.shift;
}
QTTS_HD long long kv_page_bytes(const KvGeom& g) {
  return (long long)g.layers * 2 * g.kv_heads * kv_tile_bytes(g);
}
// First byte of the tile of (physical page, layer, 0 = K / 1 = V, kv head).
QTTS_HD long long kv_tile_at(const KvGeom& g, int page, int layer, int which, int head) {
  return page * kv_page_bytes(g) +
         ((long long)(layer * 2 + which) * g.kv_heads + head) * kv_tile_bytes(g);
}
// Within a tile: byte of a row's values / codes, and of its scales (4 bits).
QTTS_HD int kv_row_at(const KvGeom& g, int row) {
  return row * (g.bits == 16 ? 2 * kKvDim : kKvCodeBytes);
}
QTTS_HD int kv_scale_at(const KvGeom& g, int row) {
  return (kKvCodeBytes << g.shift) + row * 2 * kKvGroups;
}
// Byte, within a row's 64 code bytes, of the 32-bit word that holds dim d.
QTTS_HD int kv_code_word_at(int d) { return 4 * (4 * ((d >> 3) & 3) + (d >> 5)); }
// Positions the page table of one sequence can name.
QTTS_HD long long kv_capacity(const KvGeom& g) { return (long long)g.max_pages << g.shift; }

// What the row at `pos` sees: [0, sink_end) and [first, pos]. window 0: all.
// A sink that the window reaches anyway is left to the window.
struct KvSpan {
  int sink_end, first;
};
QTTS_HD KvSpan kv_span(int pos, int window, int sinks) {
  KvSpan s;
  s.first = window > 0 && pos >= window ? pos - window + 1 : 0;
  s.sink_end = sinks < s.first ? sinks : s.first;
  return s;
}
QTTS_HD bool kv_sees(int pos, int key, int window, int sinks) {
  return key <= pos && (window == 0 || pos - key < window || key < sinks);
}
// Whether logical page j holds nothing that the newest row (position len - 1)
// or a later one sees.
QTTS_HD bool kv_page_behind(int j, int shift, int len, int window, int sinks) {
  const long long b = (long long)j << shift, e = b + (1LL << shift);
  return b >= sinks && e <= (long long)len - window;
}

}  // namespace qtts
