// Attention of many rows over a paged key / value cache, on the tensor cores
// (tcgen05, accumulators in TMEM), bound by the matrix products and the
// exponentials.
//
// A CTA serves 128 matrix rows: the query heads of one kv head (innermost) for
// consecutive rows of one sequence. It walks the visible positions in blocks
// of 64 (sinks first, then the window): S = Q K^T (128 x 64, two buffers in
// TMEM), a thread per row turns its 64 scores into weights P with a running
// maximum and sum, and O += P V (128 x 128, TMEM). Everything between is in
// shared memory as K-major operands in the 128-byte swizzle.
//
// Warps: 0-3 softmax and output (thread = matrix row = TMEM lane), 4-7 bring
// blocks from the pages (16-bit K straight to shared memory by cp.async; the
// rest through registers, two blocks in flight: V is transposed by byte
// permutes, codes become values), 8 issues the matrix instructions. Nine warps
// leave 168 registers a thread; thirteen (two groups of loaders) leave 128,
// which spilled.
//
// Number forms. 16-bit pages: bf16 operands as they are; rows of bf16 take Q
// as it is and P as two bf16 parts (16 bits: one part would add an error of
// the size of the output's own rounding); fp32 rows take Q and P as three
// bf16 parts (24 bits). 4-bit pages: fp16 operands. A code times its bf16
// scale has 11 significant bits, so it is exact in fp16 for scales of 2^-14 to
// 2^12; queries are scaled per row by a power of two into fp16's range; P is
// rounded to fp16 (2^-12), fp32 rows take two parts of each (22 bits). Scales
// outside that range, and NaN or infinity in places that only some of the
// rows see, send the CTA's rows to the row-by-row form (kv_attend_row).
//
// The running maximum is raised only when a row's score exceeds it by more
// than 2^8 (the weights then stay below 256, no trouble for fp32 sums), so
// the rescaling of O in TMEM is rare.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"
#include "kv.cuh"
#include "sm100.cuh"

namespace qtts {
namespace {

constexpr int kRowsM = 128;   // matrix rows of a CTA
constexpr int kKeys = 64;     // positions per block
constexpr int kLoadGroup = 128;  // loader threads
constexpr int kMmaWarp = 8;
constexpr int kTileThreads = 128 + kLoadGroup + 32;
constexpr unsigned long long kTileWaitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f;

template <int BITS, bool F32>
struct Form {
  static constexpr int qp = !F32 ? 1 : BITS == 16 ? 3 : 2;                   // parts of Q
  static constexpr int pp = BITS == 16 ? (F32 ? 3 : 2) : (F32 ? 2 : 1);     // parts of P
  static constexpr int q_bytes = qp * kRowsM * kKvDim * 2;
  static constexpr int p_bytes = pp * kRowsM * kKeys * 2;
  static constexpr int kv_bytes = kKeys * kKvDim * 2;          // K or V of one block
  static constexpr int stages = F32 && BITS == 16 ? 2 : 3;
  static constexpr int smem = q_bytes + p_bytes + stages * 2 * kv_bytes + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of one SM");
};

struct Bars {
  uint64_t kfull[3], kempty[3], vfull[3], vempty[3], sfull[2], sempty[2], pfull, pempty, done;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int BITS>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (BITS == 16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int BITS>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
  if constexpr (BITS == 16) return make_float2(bf16lo(w), bf16hi(w));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// Byte of 16-byte chunk `ch` (0..7) of row `r` in a [rows][64] swizzled tile.
__device__ __forceinline__ int swz(int r, int ch) { return r * 128 + ((ch ^ (r & 7)) << 4); }

// Eight values as `PARTS` operands of 16 bits, each what the ones before left.
template <int BITS, int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], uint4 (&out)[PARTS]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_pair<BITS>(r[2 * i], r[2 * i + 1]);
      if (p + 1 < PARTS) {
        const float2 f = unpack_pair<BITS>(w[i]);
        r[2 * i] -= f.x;
        r[2 * i + 1] -= f.y;
      }
    }
    out[p] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// What loaders meet in a tile's blocks. 4-bit scales: below 2^-14 (tiny) a
// product is rounded to multiples of 2^-24, which matters only where no scale
// of 2^-8 or more (big) sets the size of the values.
enum : int { kOdd = 1, kTinyK = 2, kBigK = 4, kTinyV = 8, kBigV = 16 };
__device__ __forceinline__ bool row_by_row(int seen) {
  return (seen & kOdd) || ((seen & kTinyK) && !(seen & kBigK)) ||
         ((seen & kTinyV) && !(seen & kBigV));
}

// The group of blockIdx.x: its rows and sequence. Same checks as kv_place.
__device__ __forceinline__ bool group_rows(const KvArgs& c, const KvRows& r, int group, int* seq,
                                           int* begin, int* end, int* len) {
  *begin = r.row_start ? __ldg(r.row_start + group) : group;
  *end = r.row_start ? __ldg(r.row_start + group + 1) : group + 1;
  if (*begin < 0 || *end > r.rows || *begin >= *end) {
    // rows outside the tensor; an empty group is in order
    if (threadIdx.x == 0 && *begin != *end) kv_bad(c);
    *begin = max(*begin, 0);
    *end = min(*end, r.rows);
    if (*begin >= *end) return false;
  }
  *seq = r.seqs ? __ldg(r.seqs + group) : group;
  *len = 0;
  if ((unsigned)*seq >= (unsigned)c.g.seqs) {
    if (threadIdx.x == 0) kv_bad(c);
    *seq = 0;
    *len = -1;
    return true;
  }
  *len = kv_length(c, *seq);
  if (*len < 0 || *len > kv_capacity(c.g)) {
    if (threadIdx.x == 0) kv_bad(c);
    *len = -1;
  }
  return true;
}

// One block of 64 positions in a loader thread's registers.
template <int BITS>
struct Block;
template <>
struct Block<16> {
  uint4 v[8];       // keys 8 kb + i, dims 8 db ..
};
template <>
struct Block<4> {
  uint32_t k[8];    // K: dims 8 per word, row lt / 16 + 8 i
  uint32_t ks[8];   // the scale of that group, bf16 in the low half
  uint32_t v[8];    // V: keys 8 kb + i, dims 8 db ..
  uint32_t vs[8];
};

template <int BITS, bool F32>
__global__ void __launch_bounds__(kTileThreads, 1)
    k_kv_tiles(KvArgs c, KvRows r, KvAttend a, int chunks, int gheads, int rows_per, int tiles) {
  using Fm = Form<BITS, F32>;
  constexpr int QP = Fm::qp, PP = Fm::pp, ST = Fm::stages;
  extern __shared__ uint8_t tile_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(tile_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* sp = sq + Fm::q_bytes;
  uint8_t* skv = sp + Fm::p_bytes;  // stage s: K at 2 s, V at 2 s + 1 (kv_bytes each)
  __shared__ Bars b;
  __shared__ uint32_t s_tmem;
  __shared__ int s_seen;  // what the loaders met (kOdd ..)
  __shared__ int s_dead;  // a wait ran out

  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = blockIdx.x % r.groups;
  const int head = blockIdx.y / chunks, chunk = blockIdx.y % chunks;
  const int per_head = a.q_heads / c.g.kv_heads;
  const int heads = min(gheads, per_head - chunk * gheads);
  const int qh0 = head * per_head + chunk * gheads;
  int seq, begin, end, len;
  if (!group_rows(c, r, group, &seq, &begin, &end, &len)) return;
  if (a.halt && __ldcg(a.halt + (long long)group * a.halt_stride)) return;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&b.kfull[i], kLoadGroup / 32);
      mbar_init(&b.vfull[i], kLoadGroup / 32);
      mbar_init(&b.kempty[i], 1);
      mbar_init(&b.vempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b.sfull[i], 1);
      mbar_init(&b.sempty[i], 4);
    }
    mbar_init(&b.pfull, 4);
    mbar_init(&b.pempty, 1);
    mbar_init(&b.done, 1);
    fence_mbar_init();
    s_dead = 0;
  }
  if (warp == kMmaWarp) tmem_alloc(&s_tmem, 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm_s = s_tmem, tm_o = s_tmem + 128;

  // bounded waits: of one thread, and of a warp (all lanes give up together)
  auto wait = [&](uint64_t* bar, unsigned parity) {
    if (mbar_wait_ns(bar, parity & 1, kTileWaitNs)) return true;
    atomicExch(&s_dead, 1);
    return false;
  };
  auto wait_warp = [&](uint64_t* bar, unsigned parity) {
    return __all_sync(0xffffffffu, wait(bar, parity)) != 0;
  };

  int base = 0;        // blocks of the tiles before this one (stage and phase run on)
  unsigned dones = 0;  // tiles finished
  // more row tiles than the launch was told of are taken in turn
  for (int tile = tiles - 1 - (int)(blockIdx.x / r.groups); tile * rows_per < end - begin;
       tile += tiles) {
    const int row0 = begin + tile * rows_per;
    const int n = min(rows_per, end - row0);
    const int pos0 = len - (end - row0);            // position of the tile's first row
    const int last = len < 0 ? -1 : pos0 + n - 1;   // < 0: no row holds a position
    const int low = max(pos0, 0);
    // blocks that some row sees: [0, ns) and [ws, last / 64]
    const KvSpan s_lo = kv_span(low, a.window, a.sinks), s_hi = kv_span(max(last, 0), a.window, a.sinks);
    const int ns = (s_hi.sink_end + kKeys - 1) / kKeys;
    const int ws = max(s_lo.first / kKeys, ns);
    const int blocks = last < 0 ? 0 : ns + max(0, last / kKeys - ws + 1);
    auto block_pos = [&](int j) { return (j < ns ? j : j - ns + ws) * kKeys; };
    // every row sees every position of the block
    auto whole = [&](int p0) {
      return pos0 >= 0 && p0 + kKeys - 1 <= pos0 &&
             (a.window == 0 || p0 > last - a.window || p0 + kKeys <= a.sinks);
    };
    if (threadIdx.x == 0) s_seen = 0;
    float q_scale = 1.f;  // softmax threads: what undoes the row's power of two
    if (warp < 4) {
      // ---- Q: this thread's matrix row
      const int m = threadIdx.x, rr = m / heads, hh = m - rr * heads;
      const bool in = rr < n;
      const long long off = (long long)(row0 + rr) * a.q.row + (long long)(qh0 + hh) * a.q.head;
      float up = 1.f;
      if constexpr (BITS == 4) {
        float top = 0.f;
        if (in)
#pragma unroll 8
          for (int d = 0; d < kKvDim; d += 4) {
            const float4 x = kv_load4(a.q.p, off + d, a.type);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))));
          }
        if (top > 0.f && isfinite(top)) {
          // largest magnitude into [2^8, 2^9); the limits keep both factors normal
          const int e = min(max((int)((__float_as_uint(top) >> 23) & 255) - 127, -110), 110);
          up = __uint_as_float((unsigned)(127 + 8 - e) << 23);
          q_scale = __uint_as_float((unsigned)(127 - 8 + e) << 23);
        }
      }
#pragma unroll 4
      for (int ch = 0; ch < 16; ++ch) {
        float x[8];
        if (in) {
          const float4 y = kv_load4(a.q.p, off + 8 * ch, a.type);
          const float4 z = kv_load4(a.q.p, off + 8 * ch + 4, a.type);
          x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
          x[4] = z.x; x[5] = z.y; x[6] = z.z; x[7] = z.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = 0.f;
        }
        // a negative scale goes into Q, so that masked scores are -inf either way
        const float u = a.scale < 0.f ? -up : up;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= u;
        uint4 w[QP];
        split8<BITS, QP>(x, w);
#pragma unroll
        for (int p = 0; p < QP; ++p)
          *reinterpret_cast<uint4*>(sq + (2 * p + (ch >> 3)) * (kRowsM * 128) + swz(m, ch & 7)) = w[p];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();

    if (warp == kMmaWarp) {
      // ---- matrix instructions, one thread
      if (lane == 0) {
        constexpr uint32_t is = BITS == 16 ? umma_idesc_bf16(kRowsM, kKeys) : umma_idesc_f16(kRowsM, kKeys);
        constexpr uint32_t io = BITS == 16 ? umma_idesc_bf16(kRowsM, kKvDim) : umma_idesc_f16(kRowsM, kKvDim);
        bool ok = true;
        auto scores = [&](int j) {
          const int g = base + j, s = g % ST;
          if (!wait(&b.kfull[s], g / ST) || !wait(&b.sempty[g & 1], (g >> 1) + 1)) return false;
          tc_fence_after();
#pragma unroll
          for (int p = 0; p < QP; ++p)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint64_t dq = umma_desc_sw128(sq + (2 * p + h) * (kRowsM * 128));
              const uint64_t dk = umma_desc_sw128(skv + 2 * s * Fm::kv_bytes + h * (kKeys * 128));
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_bf16(tm_s + (g & 1) * kKeys, dq + 2 * k, dk + 2 * k, is, (p | h | k) != 0);
            }
          umma_commit(&b.kempty[s]);
          umma_commit(&b.sfull[g & 1]);
          return true;
        };
        if (blocks) ok = scores(0);
        for (int j = 0; j < blocks && ok; ++j) {
          if (j + 1 < blocks && !scores(j + 1)) break;
          const int g = base + j, s = g % ST;
          if (!wait(&b.vfull[s], g / ST) || !wait(&b.pfull, g)) break;
          tc_fence_after();
#pragma unroll
          for (int p = 0; p < PP; ++p) {
            const uint64_t dp = umma_desc_sw128(sp + p * (kRowsM * 128));
            const uint64_t dv = umma_desc_sw128(skv + (2 * s + 1) * Fm::kv_bytes);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_bf16(tm_o, dp + 2 * k, dv + 2 * k, io, j > 0 || (p | k) != 0);
          }
          umma_commit(&b.vempty[s]);
          umma_commit(&b.pempty);
        }
        umma_commit(&b.done);
      }
    } else if (warp >= 4) {
      // ---- loaders
      const int lt = threadIdx.x - 128;
      const int kb = lt & 7, db = lt >> 3;          // V: keys 8 kb .., dims 8 db ..
      const int krow = lt >> 4, kch = lt & 15;      // K: rows krow + 8 i, dims 8 kch ..
      const long long tile_bytes = kv_tile_bytes(c.g), page_bytes = kv_page_bytes(c.g);
      const unsigned char* kbase = c.pool + kv_tile_at(c.g, 0, a.layer, 0, head);
      const unsigned char* vbase = kbase + tile_bytes * c.g.kv_heads;
      const int mask = (1 << c.g.shift) - 1;
      // pages of a block's four quarters (a page is at least one of them)
      auto pages = [&](int p0, int (&pg)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = p0 + 16 * i;
          pg[i] = p <= last ? kv_page(c, seq, p >> c.g.shift) : -1;
        }
      };
      // 16 bits: K of block j to its stage; positions that are not there become 0
      auto copy_k = [&](int j) {
        const int g = base + j, s = g % ST, p0 = block_pos(j);
        int pg[4];
        pages(p0, pg);
        if (!wait_warp(&b.kempty[s], g / ST + 1)) return false;
        const uint32_t sk = smem_u32(skv + 2 * s * Fm::kv_bytes + (kch >> 3) * (kKeys * 128));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int kr = krow + 8 * i, page = pg[i >> 1];
          const bool ok = page >= 0 && p0 + kr <= last;
          const unsigned char* src =
              kbase + (ok ? page : 0) * page_bytes + ((p0 + kr) & mask) * 256 + kch * 16;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sk + swz(kr, kch & 7)),
                       "l"(src), "r"(ok ? 16 : 0)
                       : "memory");
        }
        return true;
      };
      auto load = [&](Block<BITS>& x, int p0) {
        int pg[4];
        pages(p0, pg);
        if constexpr (BITS == 4) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int kr = krow + 8 * i;             // in quarter i / 2
            const int page = pg[i >> 1], prow = (p0 + kr) & mask;
            const bool ok = page >= 0 && p0 + kr <= last;
            const unsigned char* t = kbase + (ok ? page : 0) * page_bytes;
            x.k[i] = ok ? __ldcg(reinterpret_cast<const uint32_t*>(t + prow * 64 + kv_code_word_at(8 * kch)))
                        : 0x88888888u;
            x.ks[i] = ok ? __ldcg(reinterpret_cast<const uint16_t*>(t + (kKvCodeBytes << c.g.shift)) +
                                  prow * 4 + (kch >> 2))
                         : 0u;
          }
        }
        const int vq = kb >> 1;                      // the quarter of this thread's keys
        const int vpage = vq == 0 ? pg[0] : vq == 1 ? pg[1] : vq == 2 ? pg[2] : pg[3];
        const int prow0 = (p0 + 8 * kb) & mask;      // eight rows of one page
        const unsigned char* t = vbase + max(vpage, 0) * page_bytes;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int prow = prow0 + i;
          const bool ok = vpage >= 0 && p0 + 8 * kb + i <= last;
          if constexpr (BITS == 16) {
            x.v[i] = ok ? __ldcg(reinterpret_cast<const uint4*>(t + prow * 256) + db)
                        : make_uint4(0u, 0u, 0u, 0u);
          } else {
            x.v[i] = ok ? __ldcg(reinterpret_cast<const uint32_t*>(t + prow * 64 + kv_code_word_at(8 * db)))
                        : 0x88888888u;
            x.vs[i] = ok ? __ldcg(reinterpret_cast<const uint16_t*>(t + (kKvCodeBytes << c.g.shift)) +
                                  prow * 4 + (db >> 2))
                         : 0u;
          }
        }
      };
      // a 4-bit scale as fp16 (both halves)
      int seen = 0;
      auto half_scale = [&](uint32_t s16, int tiny, int big) {
        const float s = __uint_as_float(s16 << 16);
        seen |= (s <= 4096.f ? 0 : kOdd) | (s != 0.f && s < 6.103515625e-05f ? tiny : 0) |
                (s >= 0.00390625f ? big : 0);
        return __half2half2(__float2half_rn(s));
      };
      // eight codes (one word) times a scale: four words of two fp16 values,
      // pair i = nibbles i and i + 4
      auto values = [&](uint32_t w, __half2 s, uint32_t (&o)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;  // 1024 + code
          const __half2 nv = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1032.f, 1032.f));
          const __half2 v = __hmul2(nv, s);
          o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
      };
      auto store = [&](Block<BITS>& x, int j) {
        const int g = base + j, s = g % ST;
        uint8_t* sk = skv + 2 * s * Fm::kv_bytes;
        uint8_t* sv = sk + Fm::kv_bytes;
        const int p0 = block_pos(j);
        if constexpr (BITS == 16) {
          // the copies of block j are the oldest of at most ST - 1 groups in flight
          asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        } else {
          if (!wait_warp(&b.kempty[s], g / ST + 1)) return false;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t o[4];
            values(x.k[i], half_scale(x.ks[i], kTinyK, kBigK), o);
            // dims in order: pairs (0, 1), (2, 3) from nibbles (i, i + 4)
            *reinterpret_cast<uint4*>(sk + (kch >> 3) * (kKeys * 128) + swz(krow + 8 * i, kch & 7)) =
                make_uint4(__byte_perm(o[0], o[1], 0x5410), __byte_perm(o[2], o[3], 0x5410),
                           __byte_perm(o[0], o[1], 0x7632), __byte_perm(o[2], o[3], 0x7632));
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.kfull[s]);
        if (!wait_warp(&b.vempty[s], g / ST + 1)) return false;
        if constexpr (BITS == 16) {
          if (!whole(p0)) {
            // NaN or infinity where only some rows look
            uint32_t bad = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const uint32_t w = k == 0 ? x.v[i].x : k == 1 ? x.v[i].y : k == 2 ? x.v[i].z : x.v[i].w;
                bad |= ((w & 0x7f80u) == 0x7f80u) | ((w & 0x7f800000u) == 0x7f800000u);
              }
            if (bad) seen |= kOdd;
          }
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const unsigned sel = d & 1 ? 0x7632u : 0x5410u;
            auto at = [&](int i) {
              return d / 2 == 0 ? x.v[i].x : d / 2 == 1 ? x.v[i].y : d / 2 == 2 ? x.v[i].z : x.v[i].w;
            };
            *reinterpret_cast<uint4*>(sv + swz(8 * db + d, kb)) =
                make_uint4(__byte_perm(at(0), at(1), sel), __byte_perm(at(2), at(3), sel),
                           __byte_perm(at(4), at(5), sel), __byte_perm(at(6), at(7), sel));
          }
        } else {
          // nibbles to pairs (dim d, dim d + 4) per key, then to pairs of keys
          uint32_t o[8][4];
#pragma unroll
          for (int i = 0; i < 8; ++i) values(x.v[i], half_scale(x.vs[i], kTinyV, kBigV), o[i]);
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const unsigned sel = d >= 4 ? 0x7632u : 0x5410u;
            *reinterpret_cast<uint4*>(sv + swz(8 * db + d, kb)) =
                make_uint4(__byte_perm(o[0][d & 3], o[1][d & 3], sel),
                           __byte_perm(o[2][d & 3], o[3][d & 3], sel),
                           __byte_perm(o[4][d & 3], o[5][d & 3], sel),
                           __byte_perm(o[6][d & 3], o[7][d & 3], sel));
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.vfull[s]);
        return true;
      };
      // K runs ST - 1 blocks ahead (one group of copies per block, empty past
      // the end), V two
      auto ahead = [&](int j) {
        bool fine = true;
        if constexpr (BITS == 16) {
          if (j < blocks) fine = copy_k(j);
          asm volatile("cp.async.commit_group;" ::: "memory");
        }
        return fine;
      };
      Block<BITS> x, y;
      bool fine = true;
      if (blocks > 0) load(x, block_pos(0));
      for (int j = 0; j < ST - 1 && fine; ++j) fine = ahead(j);
      for (int j = 0; j < blocks && fine; j += 2) {
        if (j + 1 < blocks) load(y, block_pos(j + 1));
        fine = ahead(j + ST - 1) && store(x, j);
        if (!fine || j + 1 >= blocks) break;
        if (j + 2 < blocks) load(x, block_pos(j + 2));
        fine = ahead(j + ST) && store(y, j + 1);
      }
      if constexpr (BITS == 16) asm volatile("cp.async.wait_all;" ::: "memory");
      if (seen) atomicOr(&s_seen, seen);
    } else {
      // ---- softmax: thread = matrix row
      const int m = threadIdx.x, rr = m / heads;
      const int pos = rr < n ? pos0 + rr : -1;
      const uint32_t quad = (uint32_t)(warp * 32) << 16;
      // (a scale of 0 stays a positive factor: -inf * 0 is not a number)
      const float f = fmaxf(fabsf(a.scale) * kLog2e * q_scale, 1.2e-38f);
      float top = -INFINITY, sum = 0.f;  // top: in units of log2, of scaled scores
      // lanes 0-3: the pages of the next block's quarters
      auto quarter = [&](int j) {
        const int p = block_pos(j) + 16 * lane;
        return lane < 4 && j < blocks && p <= last ? kv_page(c, seq, p >> c.g.shift) : -1;
      };
      int page = quarter(0);
      for (int j = 0; j < blocks; ++j) {
        const int g = base + j;
        const int p0 = block_pos(j);
        float x[kKeys];
        const unsigned present = __ballot_sync(0xffffffffu, page >= 0) & 15u;
        page = quarter(j + 1);
        if (!wait_warp(&b.sfull[g & 1], g >> 1)) break;
        tc_fence_after();
        tmem_ld32(tm_s + quad + (g & 1) * kKeys, x);
        tmem_ld32(tm_s + quad + (g & 1) * kKeys + 32, x + 32);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.sempty[g & 1]);
        if (!whole(p0) || present != 15) {
          const int hi = pos - p0;
          const int lo = a.window ? hi - a.window : -1;  // seen: lo < i <= hi, or i < sinks - p0
          const int si = a.sinks - p0;
#pragma unroll
          for (int i = 0; i < kKeys; ++i) {
            const bool v = i <= hi && (a.window == 0 || i > lo || i < si) && ((present >> (i >> 4)) & 1);
            if (!v) x[i] = -INFINITY;
          }
        }
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < kKeys; ++i) mx = fmaxf(mx, x[i]);
        const float bt = mx * f;
        // the first scores set the maximum; later it moves when exceeded by 2^8
        const bool raise = bt > top + 8.f || (top == -INFINITY && bt > -INFINITY);
        float corr = 1.f;
        if (raise) {
          corr = exp2_fast(top - bt);
          top = bt;
          sum *= corr;
        }
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < kKeys; ++i) x[i] = exp2_fast(fmaf(x[i], f, -ref));
        float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kKeys; ++i) s4[i & 3] += x[i];
        sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
        // the products of the block before are done: P and O may change
        if (!wait_warp(&b.pempty, g + 1)) break;
        tc_fence_after();
        if (j > 0 && __any_sync(0xffffffffu, raise)) {
          float o[32];
#pragma unroll 1
          for (int k = 0; k < kKvDim; k += 32) {
            tmem_ld32(tm_o + quad + k, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= corr;
            tmem_st32(tm_o + quad + k, o);
          }
          tmem_st_wait();
        }
#pragma unroll
        for (int ch = 0; ch < 8; ++ch) {
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = x[8 * ch + i];
          uint4 w[PP];
          split8<BITS, PP>(y, w);
#pragma unroll
          for (int p = 0; p < PP; ++p)
            *reinterpret_cast<uint4*>(sp + p * (kRowsM * 128) + swz(m, ch)) = w[p];
        }
        tc_fence_before();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&b.pfull);
      }
      // the matrix products are waited for even after an error: neither TMEM nor
      // shared memory may go while they run
      wait_warp(&b.done, dones);
      tc_fence_after();
      const float il = sum == 0.f ? 0.f : 1.0f / sum;
      const long long off = (long long)(row0 + rr) * a.out.row +
                            (long long)(qh0 + m - rr * heads) * a.out.head;
#pragma unroll 1
      for (int k = 0; k < kKvDim; k += 32) {
        float o[32];
        if (blocks) {
          tmem_ld32(tm_o + quad + k, o);
          tmem_ld_wait();
        }
        if (rr >= n) continue;
        const bool none = blocks == 0 || sum == 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          kv_store4(a.out.p, off + k + i, a.type,
                    none ? make_float4(0.f, 0.f, 0.f, 0.f)
                         : make_float4(o[i] * il, o[i + 1] * il, o[i + 2] * il, o[i + 3] * il));
      }
      tc_fence_before();
    }
    base += blocks;
    ++dones;
    __syncthreads();
    if (s_dead) break;
    if (row_by_row(s_seen)) {
      for (int m = warp; m < n * heads; m += kTileThreads / 32) {
        const int rr = m / heads;
        if (pos0 + rr >= 0) kv_attend_row(c, a, seq, pos0 + rr, row0 + rr, qh0 + m - rr * heads);
      }
      __syncthreads();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && s_dead) kv_status(c, kKvTimeout);
  if (warp == kMmaWarp) tmem_free(s_tmem, 256);
}

template <int BITS, bool F32>
cudaError_t tiles(const KvArgs& c, const KvRows& r, const KvAttend& a, cudaStream_t stream) {
  auto kernel = k_kv_tiles<BITS, F32>;
  constexpr int smem = Form<BITS, F32>::smem;
  static std::mutex mu;
  static bool ready[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!ready[dev]) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
      ready[dev] = true;
    }
  }
  const int group = a.q_heads / c.g.kv_heads;
  const int gheads = std::min(group, kRowsM), chunks = (group + gheads - 1) / gheads;
  const int rows_per = kRowsM / gheads;
  const int n = (r.max_rows + rows_per - 1) / rows_per;
  return launch(kernel, dim3((unsigned)((long long)n * r.groups), (unsigned)(c.g.kv_heads * chunks)),
                dim3(kTileThreads), (size_t)smem, stream, c, r, a, chunks, gheads, rows_per, n);
}

}  // namespace

cudaError_t launch_kv_tiles(const KvArgs& c, const KvRows& r, const KvAttend& a,
                            cudaStream_t stream) {
  if (c.g.bits == 16)
    return a.type == KV_F32 ? tiles<16, true>(c, r, a, stream) : tiles<16, false>(c, r, a, stream);
  return a.type == KV_F32 ? tiles<4, true>(c, r, a, stream) : tiles<4, false>(c, r, a, stream);
}

}  // namespace qtts
