// Attention of many rows over a paged key / value cache, on the tensor cores
// (tcgen05, accumulators in TMEM), bound by the matrix products and the
// exponentials.
//
// A CTA serves 128 matrix rows: the query heads of one kv head (innermost) for
// consecutive rows of one sequence. It walks the visible positions in blocks
// of 64 (sinks first, then the window): S = Q K^T (128 x 64, two buffers in
// TMEM), a thread per row turns its 64 scores into weights P with a running
// maximum and sum, and O += P V (128 x 128, TMEM). Everything between is in
// shared memory in the 128-byte swizzle; V is the transposed operand, so K and
// V keep the pages' own order of rows.
//
// Four warpgroups: two of softmax (thread = matrix row = TMEM lane), which
// take alternate blocks with statistics and an O of their own that are merged
// at the end, so that one's exponentials hide the other's waits; one that
// brings blocks from the pages (16 bits: cp.async, blocks ahead; 4 bits:
// through registers, two blocks in flight, codes become values); one whose
// first warp issues the matrix instructions. Registers are moved from the last
// two to the first two.
//
// Number forms. 16-bit pages, bf16 rows: Q K^T in bf16 as it is; P in fp16
// (2^-12) with V in fp16, which holds a bf16 value exactly from 2^-14 to 2^16.
// 16-bit pages, fp32 rows: Q and P as three bf16 parts (24 bits). 4-bit pages:
// a code times its bf16 scale has 11 significant bits, so it is exact in fp16
// for scales of 2^-14 to 2^12; queries are scaled per row by a power of two
// into fp16's range; fp32 rows take Q and P as two fp16 parts (22 bits).
// Values outside fp16's range, and NaN or infinity in places that only some
// of the rows see, send the CTA's rows to the row-by-row form (kv_attend_row).
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
constexpr int kGroup = 128;   // threads of a warpgroup
constexpr int kTileThreads = 4 * kGroup;
constexpr int kMmaWarp = 12;
// Registers per thread of the warpgroups (128 at launch): they add up to 512.
constexpr int kRegsSoftmax = 176, kRegsLoad = 112, kRegsMma = 48;
static_assert(2 * kRegsSoftmax + kRegsLoad + kRegsMma <= 4 * 128, "registers the block was given");
constexpr long long kTileWaitCycles = 4000000000ll;  // two seconds at 2 GHz
constexpr float kLog2e = 1.4426950408889634f;

template <int BITS, bool F32>
struct Form {
  static constexpr bool qk16 = BITS == 4;           // Q and K in fp16 (else bf16)
  static constexpr bool pv16 = !(BITS == 16 && F32);  // P and V in fp16
  static constexpr int qp = !F32 ? 1 : BITS == 16 ? 3 : 2;  // parts of Q
  static constexpr int pp = qp;                             // parts of P
  // softmax warpgroups at work: shared memory has no room for two P of three parts
  static constexpr int groups = BITS == 16 && F32 ? 1 : 2;
  static constexpr int q_bytes = qp * kRowsM * kKvDim * 2;
  static constexpr int p_bytes = pp * kRowsM * kKeys * 2;
  static constexpr int kv_bytes = kKeys * kKvDim * 2;          // K or V of one block
  static constexpr int stages = F32 ? 2 : 4;
  static constexpr int smem = q_bytes + groups * p_bytes + stages * 2 * kv_bytes + 1024;
  static_assert(smem + 2304 <= 227 * 1024, "shared memory of one SM");
};

constexpr int kMaxStages = 4;
struct Bars {
  uint64_t kfull[kMaxStages], kempty[kMaxStages], vfull[kMaxStages], vempty[kMaxStages];
  uint64_t sfull[2], sempty[2], pfull[2], pempty[2], done;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool HALF>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (!HALF) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// Byte of 16-byte chunk `ch` (0..7) of row `r` in a [rows][64] swizzled tile.
__device__ __forceinline__ int swz(int r, int ch) { return r * 128 + ((ch ^ (r & 7)) << 4); }

// Eight values as `PARTS` operands of 16 bits, each what the ones before left.
template <bool HALF, int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], uint4 (&out)[PARTS]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!HALF && p + 1 < PARTS) {
        // cut, not rounded: one permute, and the next part takes the rest
        const uint32_t a = __float_as_uint(r[2 * i]), b = __float_as_uint(r[2 * i + 1]);
        w[i] = __byte_perm(a, b, 0x7632);
        r[2 * i] -= __uint_as_float(a & 0xffff0000u);
        r[2 * i + 1] -= __uint_as_float(b & 0xffff0000u);
        continue;
      }
      w[i] = pack_pair<HALF>(r[2 * i], r[2 * i + 1]);
      if (p + 1 < PARTS) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        r[2 * i] -= f.x;
        r[2 * i + 1] -= f.y;
      }
    }
    out[p] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// What loaders meet in a tile's blocks: odd values (NaN, infinity, past fp16);
// and whether what fp16 rounds (below 2^-14, to multiples of 2^-24) is small
// beside the rest: some K, some V of at least 2^-11 (a scale for 4 bits), or
// nothing but zeros.
enum : int { kOdd = 1, kAnyK = 2, kBigK = 4, kAnyV = 8, kBigV = 16 };
__device__ __forceinline__ bool row_by_row(int seen) {
  return (seen & kOdd) || ((seen & kAnyK) && !(seen & kBigK)) ||
         ((seen & kAnyV) && !(seen & kBigV));
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

// 4 bits: one block of 64 positions in a loader thread's registers. K and V:
// row krow + 8 i, the word of dims 8 kch .. and (bf16, low half) its scale.
struct Codes {
  uint32_t k[8], ks[8], v[8], vs[8];
};

template <int REGS, bool MORE>
__device__ __forceinline__ void set_registers() {
  if constexpr (MORE)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
  else
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int ID, int THREADS>
__device__ __forceinline__ void bar() {
  asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(THREADS) : "memory");
}

// The row tiles of one CTA, the same for every role.
struct Walk {
  int begin, end, len, rows_per, window, sinks;
  int row0, n, pos0, last, ns, ws, blocks;

  __device__ __forceinline__ void tile(int t) {
    row0 = begin + t * rows_per;
    n = min(rows_per, end - row0);
    pos0 = len - (end - row0);              // position of the tile's first row
    last = len < 0 ? -1 : pos0 + n - 1;     // < 0: no row holds a position
    // blocks that some row sees: [0, ns) and [ws, last / 64]
    const KvSpan lo = kv_span(max(pos0, 0), window, sinks), hi = kv_span(max(last, 0), window, sinks);
    ns = (hi.sink_end + kKeys - 1) / kKeys;
    ws = max(lo.first / kKeys, ns);
    blocks = last < 0 ? 0 : ns + max(0, last / kKeys - ws + 1);
  }
  __device__ __forceinline__ int block_pos(int j) const { return (j < ns ? j : j - ns + ws) * kKeys; }
  // every row sees every position of the block at p0
  __device__ __forceinline__ bool whole(int p0) const {
    return pos0 >= 0 && p0 + kKeys - 1 <= pos0 &&
           (window == 0 || p0 > last - window || p0 + kKeys <= sinks);
  }
  // Pages of the quarters of eight blocks, one per lane (a page is at least a
  // quarter), read together when the first of them is wanted.
  __device__ __forceinline__ void refill(const KvArgs& c, int seq, int j, int& held) const {
    const int lane = threadIdx.x & 31, jj = (j & ~7) + (lane >> 2);
    const int p = block_pos(jj) + 16 * (lane & 3);
    held = jj < blocks && p <= last ? kv_page(c, seq, p >> c.g.shift) : -1;
  }
};

template <int BITS, bool F32>
__global__ void __launch_bounds__(kTileThreads, 1)
    k_kv_tiles(KvArgs c, KvRows r, KvAttend a, int chunks, int gheads, int rows_per, int tiles) {
  using Fm = Form<BITS, F32>;
  constexpr int QP = Fm::qp, PP = Fm::pp, ST = Fm::stages, NG = Fm::groups;
  extern __shared__ uint8_t tile_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(tile_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sq = smem;
  uint8_t* sp = sq + Fm::q_bytes;                 // NG buffers
  uint8_t* skv = sp + NG * Fm::p_bytes;           // stage s: K at 2 s, V at 2 s + 1 (kv_bytes each)
  __shared__ Bars b;
  __shared__ uint32_t s_tmem;
  __shared__ int s_seen;  // what the loaders met (kOdd ..)
  __shared__ int s_dead;  // a wait ran out
  __shared__ float s_top[2][kRowsM], s_sum[2][kRowsM];

  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = blockIdx.x % r.groups;
  const int head = blockIdx.y / chunks, chunk = blockIdx.y % chunks;
  const int per_head = a.q_heads / c.g.kv_heads;
  const int heads = min(gheads, per_head - chunk * gheads);
  const int qh0 = head * per_head + chunk * gheads;
  Walk w;
  int seq;
  if (!group_rows(c, r, group, &seq, &w.begin, &w.end, &w.len)) return;
  if (a.halt && __ldcg(a.halt + (long long)group * a.halt_stride)) return;
  w.rows_per = rows_per;
  w.window = a.window;
  w.sinks = a.sinks;
  // tiles with more positions first; more row tiles than the launch was told
  // of are taken in turn
  const int tile0 = tiles - 1 - (int)(blockIdx.x / r.groups);
  auto more = [&](int t) { return (long long)t * rows_per < w.end - w.begin; };

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&b.kfull[i], kGroup / 32);
      mbar_init(&b.vfull[i], kGroup / 32);
      mbar_init(&b.kempty[i], 1);
      mbar_init(&b.vempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b.sfull[i], 1);
      mbar_init(&b.sempty[i], 4);
      mbar_init(&b.pfull[i], 4);
      mbar_init(&b.pempty[i], 1);
    }
    mbar_init(&b.done, 1);
    fence_mbar_init();
    s_dead = 0;
    s_seen = 0;
  }
  if (warp == kMmaWarp) tmem_alloc(&s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Dependents may start once every CTA holds its TMEM: one that took columns
  // first and then waited for this grid would never let it finish.
  pdl_trigger();
  const uint32_t tm_s = s_tmem, tm_o = s_tmem + 2 * kKeys;  // O of group w at + 128 w

  // Bounded waits of a warp: all lanes give up together.
  auto wait = [&](uint64_t* bar, unsigned parity) {
    const bool ok = mbar_wait_cycles(bar, parity & 1, kTileWaitCycles);
    if (!ok) atomicExch(&s_dead, 1);
    return __all_sync(0xffffffffu, ok) != 0;
  };
  // Per row tile, every role: bar 0 (Q is in place), its blocks, bar 0 (all are
  // done with the tile). `base`: blocks of the tiles before (stages and phases
  // run on). After a wait ran out the tiles that are left are skipped.
  int base = 0;

  if (warp >= kMmaWarp) {
    // ---- matrix instructions: the warp walks together (its operands stay in
    // uniform registers), one lane issues
    set_registers<kRegsMma, false>();
    constexpr uint32_t is = Fm::qk16 ? umma_idesc_f16(kRowsM, kKeys) : umma_idesc_bf16(kRowsM, kKeys);
    constexpr uint32_t io = (Fm::pv16 ? umma_idesc_f16(kRowsM, kKvDim) : umma_idesc_bf16(kRowsM, kKvDim)) |
                            kUmmaTransposeB;
    const uint64_t dq = umma_desc_sw128(sq), dp = umma_desc_sw128(sp), dkv = umma_desc_sw128(skv),
                   dvt = umma_desc_sw128_mn(skv, kKeys * 128);
    for (int t = tile0; more(t); t += tiles) {
      w.tile(t);
      bar<0, kTileThreads>();
      if (warp == kMmaWarp) {
        auto scores = [&](int j) {
          const int g = base + j, s = g % ST;
          if (!wait(&b.kfull[s], g / ST) || !wait(&b.sempty[g & 1], (g >> 1) + 1)) return false;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int p = 0; p < QP; ++p)
#pragma unroll
              for (int k = 0; k < 8; ++k)  // halves of 64 dims, four steps of 32 bytes in each
                umma_bf16(tm_s + (g & 1) * kKeys,
                          dq + (((2 * p + (k >> 2)) * (kRowsM * 128)) >> 4) + 2 * (k & 3),
                          dkv + ((2 * s * Fm::kv_bytes + (k >> 2) * (kKeys * 128)) >> 4) + 2 * (k & 3),
                          is, (p | k) != 0);
            umma_commit(&b.kempty[s]);
            umma_commit(&b.sfull[g & 1]);
          }
          __syncwarp();
          return true;
        };
        bool fine = (w.blocks < 1 || scores(0)) && (w.blocks < 2 || scores(1));
        for (int j = 0; j < w.blocks && fine; ++j) {
          const int g = base + j, s = g % ST, wg = g % NG;
          if (!wait(&b.vfull[s], g / ST) || !wait(&b.pfull[wg], g / NG)) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int p = 0; p < PP; ++p)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_bf16(tm_o + wg * kKvDim, dp + ((wg * Fm::p_bytes + p * (kRowsM * 128)) >> 4) + 2 * k,
                          dvt + (((2 * s + 1) * Fm::kv_bytes + k * 16 * 128) >> 4), io,
                          j >= NG || (p | k) != 0);
            umma_commit(&b.vempty[s]);
            umma_commit(&b.pempty[wg]);
          }
          __syncwarp();
          fine = j + 2 >= w.blocks || scores(j + 2);
        }
        // the output is read, and the next tile begun, after every product
        if (elect_one()) umma_commit(&b.done);
        __syncwarp();
      }
      base += w.blocks;
      bar<0, kTileThreads>();
      if (s_dead) break;
    }
    tc_fence_before();
    bar<0, kTileThreads>();
    tc_fence_after();
    if (warp == kMmaWarp) {
      if (lane == 0 && s_dead) kv_status(c, kKvTimeout);
      tmem_free(s_tmem, 512);
    }
    return;
  }

  if (warp >= 8) {
    // ---- loaders
    set_registers<kRegsLoad, false>();
    const int lt = threadIdx.x - 2 * kGroup;
    const int krow = lt >> 4, kch = lt & 15;      // rows krow + 8 i, dims 8 kch ..
    const long long page_bytes = kv_page_bytes(c.g);
    const unsigned char* kbase = c.pool + kv_tile_at(c.g, 0, a.layer, 0, head);
    const long long v_off = kv_tile_bytes(c.g) * c.g.kv_heads;  // from K's tile to V's
    const int mask = (1 << c.g.shift) - 1;
    const int at0 = (kch >> 3) * (kKeys * 128) + swz(krow, kch & 7);  // row krow + 8 i: + 1024 i
    for (int t = tile0; more(t); t += tiles) {
      w.tile(t);
      bar<0, kTileThreads>();
      int seen = 0;
      if constexpr (BITS == 16) {
        // Copies: group a holds K of block a + 1 and V of block a (K first: its
        // product comes earlier), group -1 K of block 0. They are started ST - 2
        // groups ahead; positions that are not there become 0.
        int held[2] = {-1, -1};
        auto start = [&](int j, int which) {  // block j, 0: K, 1: V
          if (j >= w.blocks) return true;
          const int g = base + j, s = g % ST, p0 = w.block_pos(j);
          if ((j & 7) == 0) w.refill(c, seq, j, held[which]);
          if (!wait(which ? &b.vempty[s] : &b.kempty[s], g / ST + 1)) return false;
          const uint32_t dst = smem_u32(skv + (2 * s + which) * Fm::kv_bytes) + at0;
          const unsigned char* from = kbase + (which ? v_off : 0) + krow * 256 + kch * 16;
#pragma unroll
          for (int qu = 0; qu < 4; ++qu) {
            const int page = __shfl_sync(0xffffffffu, held[which], 4 * (j & 7) + qu);
            const int p = p0 + 16 * qu;
            const unsigned char* src = from + max(page, 0) * page_bytes + (p & mask) * 256;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const bool ok = page >= 0 && p + krow + 8 * h <= w.last;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + 2048 * qu + 1024 * h),
                           "l"(src + 2048 * h), "r"(ok ? 16 : 0)
                           : "memory");
            }
          }
          return true;
        };
        auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
        auto give = [&](uint64_t* full) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(full);
        };
        unsigned top = 0u;  // largest magnitudes of V, per half word
        bool fine = start(0, 0);
        commit();
        for (int i = 0; i < ST - 2 && fine; ++i) {
          fine = start(i + 1, 0) && start(i, 1);
          commit();
        }
        if (fine && w.blocks > 0) {
          asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
          give(&b.kfull[base % ST]);
        }
        for (int j = 0; j < w.blocks && fine; ++j) {
          if constexpr (ST == 2) {  // nothing ahead: started now
            fine = start(j + 1, 0) && start(j, 1);
            commit();
            if (!fine) break;
          }
          asm volatile("cp.async.wait_group %0;" ::"n"(ST >= 3 ? ST - 3 : 0) : "memory");
          if (j + 1 < w.blocks) give(&b.kfull[(base + j + 1) % ST]);
          const int s = (base + j) % ST;
          uint8_t* sv = skv + (2 * s + 1) * Fm::kv_bytes + at0;
          // pv16: bf16 becomes fp16, and the largest magnitude says whether it fits;
          // else only NaN or infinity where some rows look and others do not matters
          if (Fm::pv16 || !w.whole(w.block_pos(j))) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              uint4 v = *reinterpret_cast<const uint4*>(sv + 1024 * i);
              top = __vmaxu2(top, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                           __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
              if constexpr (Fm::pv16) {
                v.x = pack_pair<true>(bf16lo(v.x), bf16hi(v.x));
                v.y = pack_pair<true>(bf16lo(v.y), bf16hi(v.y));
                v.z = pack_pair<true>(bf16lo(v.z), bf16hi(v.z));
                v.w = pack_pair<true>(bf16lo(v.w), bf16hi(v.w));
                *reinterpret_cast<uint4*>(sv + 1024 * i) = v;
              }
            }
          }
          give(&b.vfull[s]);
          if constexpr (ST > 2) {
            fine = start(j + ST - 1, 0) && start(j + ST - 2, 1);
            commit();
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        const unsigned m = max(top & 0xffffu, top >> 16);
        // bf16 bits: 0x7f80 infinity; fp16 ends below 2^16 (0x4780); 2^-11 is 0x3a00
        seen = m >= (Fm::pv16 ? 0x4780u : 0x7f80u) ? kOdd : 0;
        if (Fm::pv16) seen |= (m ? kAnyV : 0) | (m >= 0x3a00u ? kBigV : 0);
      } else {
        int held = -1;
        auto load = [&](Codes& x, int j) {
          const int p0 = w.block_pos(j);
          if ((j & 7) == 0) w.refill(c, seq, j, held);
          const unsigned char* from = kbase + krow * 64 + kv_code_word_at(8 * kch);
          const unsigned char* from_s = kbase + (kKvCodeBytes << c.g.shift) + krow * 8 + 2 * (kch >> 2);
#pragma unroll
          for (int qu = 0; qu < 4; ++qu) {
            const int page = __shfl_sync(0xffffffffu, held, 4 * (j & 7) + qu);
            const int p = p0 + 16 * qu;
            const long long at = max(page, 0) * page_bytes;
            const unsigned char* src = from + at + (p & mask) * 64;
            const unsigned char* src_s = from_s + at + (p & mask) * 8;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const bool ok = page >= 0 && p + krow + 8 * h <= w.last;
              const int i = 2 * qu + h;
              x.k[i] = ok ? __ldcg(reinterpret_cast<const uint32_t*>(src + 512 * h)) : 0u;
              x.v[i] = ok ? __ldcg(reinterpret_cast<const uint32_t*>(src + v_off + 512 * h)) : 0u;
              x.ks[i] = ok ? __ldcg(reinterpret_cast<const uint16_t*>(src_s + 64 * h)) : 0u;
              x.vs[i] = ok ? __ldcg(reinterpret_cast<const uint16_t*>(src_s + v_off + 64 * h)) : 0u;
            }
          }
        };
        // Eight codes (one word) times their scale, in fp16, dims in order.
        auto put = [&](uint8_t* dst, uint32_t x, uint32_t s16, int any, int big) {
          const float s = __uint_as_float(s16 << 16);
          seen |= (s <= 4096.f ? 0 : kOdd) | (s != 0.f ? any : 0) | (s >= 0.00048828125f ? big : 0);
          const __half2 sc = __half2half2(__float2half_rn(s));
          uint32_t o[4];  // pair i: nibbles i and i + 4
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t u = ((x >> (4 * i)) & 0x000f000fu) | 0x64006400u;  // 1024 + code
            const __half2 n =
                __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1032.f, 1032.f));
            const __half2 v = __hmul2(n, sc);
            o[i] = *reinterpret_cast<const uint32_t*>(&v);
          }
          *reinterpret_cast<uint4*>(dst) =
              make_uint4(__byte_perm(o[0], o[1], 0x5410), __byte_perm(o[2], o[3], 0x5410),
                         __byte_perm(o[0], o[1], 0x7632), __byte_perm(o[2], o[3], 0x7632));
        };
        auto store = [&](const Codes& x, int j) {
          const int g = base + j, s = g % ST;
          uint8_t* sk = skv + 2 * s * Fm::kv_bytes + at0;
          if (!wait(&b.kempty[s], g / ST + 1)) return false;
#pragma unroll
          for (int i = 0; i < 8; ++i) put(sk + 1024 * i, x.k[i], x.ks[i], kAnyK, kBigK);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&b.kfull[s]);
          if (!wait(&b.vempty[s], g / ST + 1)) return false;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            put(sk + Fm::kv_bytes + 1024 * i, x.v[i], x.vs[i], kAnyV, kBigV);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&b.vfull[s]);
          return true;
        };
        Codes x, y;
        if (w.blocks > 0) load(x, 0);
        for (int j = 0; j < w.blocks; j += 2) {
          if (j + 1 < w.blocks) load(y, j + 1);
          if (!store(x, j) || j + 1 >= w.blocks) break;
          if (j + 2 < w.blocks) load(x, j + 2);
          if (!store(y, j + 1)) break;
        }
      }
      if (seen) atomicOr(&s_seen, seen);
      base += w.blocks;
      bar<0, kTileThreads>();
      if (s_dead) break;
    }
    bar<0, kTileThreads>();
    return;
  }

  // ---- softmax: thread = matrix row
  set_registers<kRegsSoftmax, true>();
  const int wg = warp >> 2, m = threadIdx.x & (kGroup - 1);
  const int rr = m / heads, hh = m - rr * heads;
  const uint32_t quad = (uint32_t)(warp & 3) << 21;  // TMEM lane 32 (warp % 4)
  unsigned dones = 0;
  for (int t = tile0; more(t); t += tiles) {
    w.tile(t);
    float q_scale = 1.f;  // what undoes the row's power of two
    {
      // Q: with two groups each stores half of the dims of its row
      const bool in = rr < w.n;
      const long long off = (long long)(w.row0 + rr) * a.q.row + (long long)(qh0 + hh) * a.q.head;
      float up = 1.f;
      if constexpr (Fm::qk16) {
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
      // a negative scale goes into Q, so that masked scores are -inf either way
      if (a.scale < 0.f) up = -up;
#pragma unroll 4
      for (int ch = 8 * wg; ch < 8 * wg + 8; ++ch) {
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (in) {
          const float4 y = kv_load4(a.q.p, off + 8 * ch, a.type);
          const float4 z = kv_load4(a.q.p, off + 8 * ch + 4, a.type);
          x[0] = y.x * up; x[1] = y.y * up; x[2] = y.z * up; x[3] = y.w * up;
          x[4] = z.x * up; x[5] = z.y * up; x[6] = z.z * up; x[7] = z.w * up;
        }
        uint4 o[QP];
        split8<Fm::qk16, QP>(x, o);
#pragma unroll
        for (int p = 0; p < QP; ++p)
          *reinterpret_cast<uint4*>(sq + (2 * p + (ch >> 3)) * (kRowsM * 128) + swz(m, ch & 7)) = o[p];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    bar<0, kTileThreads>();
    const int pos = rr < w.n ? w.pos0 + rr : -1;
    // (a scale of 0 stays a positive factor: -inf * 0 is not a number)
    const float f = fmaxf(fabsf(a.scale) * kLog2e * q_scale, 1.2e-38f);
    float top = -INFINITY, sum = 0.f;  // top: in units of log2, of scaled scores
    int held = -1, held_at = -1;
    int first = NG == 1 ? 0 : (wg - base) & 1;  // this group's blocks: (base + j) % 2 == wg
    if (wg >= NG) first = w.blocks;
    for (int j = first; j < w.blocks; j += NG) {
      const int g = base + j;
      const int p0 = w.block_pos(j);
      float x[kKeys];
      if ((j >> 3) != held_at) {
        held_at = j >> 3;
        w.refill(c, seq, j, held);
      }
      const unsigned present = (__ballot_sync(0xffffffffu, held >= 0) >> (4 * (j & 7))) & 15u;
      if (!wait(&b.sfull[g & 1], g >> 1)) break;
      tc_fence_after();
      tmem_ld32(tm_s + quad + (g & 1) * kKeys, x);
      tmem_ld32(tm_s + quad + (g & 1) * kKeys + 32, x + 32);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.sempty[g & 1]);
      if (!w.whole(p0) || present != 15) {
        // bit i: this row sees position p0 + i
        auto below = [](int n) {  // the n lowest bits
          return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull;
        };
        unsigned long long v = below(pos - p0 + 1);
        if (a.window) v &= ~below(pos - p0 - a.window + 1) | below(a.sinks - p0);
        const unsigned lo16 = (present & 1 ? 0xffffu : 0u) | (present & 2 ? 0xffff0000u : 0u);
        const unsigned hi16 = (present & 4 ? 0xffffu : 0u) | (present & 8 ? 0xffff0000u : 0u);
        const unsigned v0 = (unsigned)v & lo16, v1 = (unsigned)(v >> 32) & hi16;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (!(v0 & (1u << i))) x[i] = -INFINITY;
          if (!(v1 & (1u << i))) x[32 + i] = -INFINITY;
        }
      }
      float m4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
      for (int i = 4; i < kKeys; ++i) m4[i & 3] = fmaxf(m4[i & 3], x[i]);
      const float bt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * f;
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
      // this group's products before are done: its P and O may change
      if (!wait(&b.pempty[g % NG], g / NG + 1)) break;
      tc_fence_after();
      if (j >= NG && __any_sync(0xffffffffu, raise)) {
        float o[32];
#pragma unroll 1
        for (int k = 0; k < kKvDim; k += 32) {
          tmem_ld32(tm_o + (g % NG) * kKvDim + quad + k, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] *= corr;
          tmem_st32(tm_o + (g % NG) * kKvDim + quad + k, o);
        }
        tmem_st_wait();
      }
      uint8_t* pb = sp + (g % NG) * Fm::p_bytes;
#pragma unroll
      for (int ch = 0; ch < 8; ++ch) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[8 * ch + i];
        uint4 o[PP];
        split8<Fm::pv16, PP>(y, o);
#pragma unroll
        for (int p = 0; p < PP; ++p)
          *reinterpret_cast<uint4*>(pb + p * (kRowsM * 128) + swz(m, ch)) = o[p];
      }
      tc_fence_before();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&b.pfull[g % NG]);
    }
    // The groups' statistics meet; each then writes half of the dims. The matrix
    // products are waited for even after an error: neither TMEM nor shared
    // memory may go while they run.
    s_top[wg][m] = top;
    s_sum[wg][m] = sum;
    wait(&b.done, dones);
    tc_fence_after();
    bar<1, 2 * kGroup>();
    const float t0 = s_top[0][m], t1 = s_top[1][m];
    const float both = fmaxf(t0, t1), ref = both == -INFINITY ? 0.f : both;
    const float e0 = exp2_fast(t0 - ref), e1 = exp2_fast(t1 - ref);
    const float l = e0 * s_sum[0][m] + e1 * s_sum[1][m];
    const float il = l == 0.f ? 0.f : 1.0f / l;
    const float w0 = e0 * il, w1 = e1 * il;
    // the O of a group that had no block in this tile was never written
    const int g0 = base % NG;  // the group of block 0
    const bool has0 = w.blocks > (g0 == 0 ? 0 : 1), has1 = NG == 2 && w.blocks > (g0 == 1 ? 0 : 1);
    const long long off = (long long)(w.row0 + rr) * a.out.row + (long long)(qh0 + hh) * a.out.head;
#pragma unroll 1
    for (int k = 64 * wg; k < 64 * wg + 64; k += 32) {
      float o[32], u[32];
      if (has0) tmem_ld32(tm_o + quad + k, o);
      if (has1) tmem_ld32(tm_o + kKvDim + quad + k, u);
      tmem_ld_wait();
      if (rr >= w.n) continue;
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = (has0 ? o[i] * w0 : 0.f) + (has1 ? u[i] * w1 : 0.f);
#pragma unroll
      for (int i = 0; i < 32; i += 4)
        kv_store4(a.out.p, off + k + i, a.type,
                  l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                           : make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]));
    }
    tc_fence_before();
    base += w.blocks;
    ++dones;
    bar<0, kTileThreads>();
    if (s_dead) break;
    const int seen = s_seen;
    bar<1, 2 * kGroup>();
    if (threadIdx.x == 0) s_seen = 0;  // before the next tile's first bar 0
    if (row_by_row(seen))
      for (int i = warp; i < w.n * heads; i += 8) {
        const int ri = i / heads;
        if (w.pos0 + ri >= 0) kv_attend_row(c, a, seq, w.pos0 + ri, w.row0 + ri, qh0 + i - ri * heads);
      }
  }
  bar<0, kTileThreads>();
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
