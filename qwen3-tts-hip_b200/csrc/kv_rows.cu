// Storing rows into a paged key / value cache and loading them back.
#include <cuda_bf16.h>

#include "common.cuh"
#include "kv.cuh"

namespace qtts {
namespace {

constexpr int kRowThreads = 256;

// One warp per (row, K or V, kv head); lane l holds dims 4 l .. 4 l + 3, so
// eight lanes share a group's scale. Every byte is touched once: the rows in,
// the codes and scales out.
template <bool READ>
__global__ void __launch_bounds__(kRowThreads)
    k_kv_rows(KvArgs c, KvRows r, int layer, KvTensor k, KvTensor v, int type) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const long long unit = ((long long)blockIdx.x * kRowThreads + threadIdx.x) >> 5;
  const int per = 2 * c.g.kv_heads;
  const int row = (int)(unit / per), u = (int)(unit - (long long)row * per);
  if (row >= r.rows) return;
  const int which = u / c.g.kv_heads, head = u - which * c.g.kv_heads;
  const KvPlace at = kv_place(c, r, row, !READ);
  if (at.group < 0) return;
  const KvTensor& t = which ? v : k;
  const long long off = (long long)row * t.row + (long long)head * t.head + 4 * lane;
  const int page = at.ok ? kv_page(c, at.seq, at.pos >> c.g.shift) : -1;
  if (page < 0) {
    // nothing is held there: nothing is written, and a row read is zeros
    if (READ) kv_store4(t.p, off, type, make_float4(0.f, 0.f, 0.f, 0.f));
    else if (at.ok) kv_bad(c);
    return;
  }
  const int prow = at.pos & ((1 << c.g.shift) - 1);
  unsigned char* tile = c.pool + kv_tile_at(c.g, page, layer, which, head);
  unsigned char* cell = tile + kv_row_at(c.g, prow);
  if (c.g.bits == 16) {
    uint2* w = reinterpret_cast<uint2*>(cell) + lane;
    if (READ) {
      const uint2 x = *w;
      kv_store4(t.p, off, type,
                make_float4(bf16lo(x.x), bf16hi(x.x), bf16lo(x.y), bf16hi(x.y)));
    } else {
      const float4 x = kv_load4(t.p, off, type);
      const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
      *w = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
    }
    return;
  }
  uint16_t* code = reinterpret_cast<uint16_t*>(cell + kv_code_word_at(4 * lane)) + (lane & 1);
  __nv_bfloat16* sc = reinterpret_cast<__nv_bfloat16*>(tile + kv_scale_at(c.g, prow)) + (lane >> 3);
  if (READ) {
    const unsigned n = *code;
    const float s = __bfloat162float(*sc);
    kv_store4(t.p, off, type,
              make_float4((float)((int)(n & 15u) - 8) * s, (float)((int)((n >> 4) & 15u) - 8) * s,
                          (float)((int)((n >> 8) & 15u) - 8) * s, (float)((int)(n >> 12) - 8) * s));
    return;
  }
  const float4 x = kv_load4(t.p, off, type);
  float s;
  *code = (uint16_t)kv_quantise4(x, &s);
  if ((lane & 7) == 0) *sc = __float2bfloat16_rn(s);
}

template <bool READ>
cudaError_t rows_op(const KvArgs& c, const KvRows& r, int layer, const KvTensor& k,
                    const KvTensor& v, int type, cudaStream_t stream) {
  const long long warps = (long long)r.rows * 2 * c.g.kv_heads;
  if (warps == 0) return cudaSuccess;
  const long long ctas = (warps * 32 + kRowThreads - 1) / kRowThreads;
  return launch(k_kv_rows<READ>, dim3((unsigned)ctas), dim3(kRowThreads), 0, stream, c, r, layer, k,
                v, type);
}

}  // namespace

cudaError_t launch_kv_append(const KvArgs& c, const KvRows& r, int layer, const KvTensor& k,
                             const KvTensor& v, int type, cudaStream_t stream) {
  return rows_op<false>(c, r, layer, k, v, type, stream);
}
cudaError_t launch_kv_read(const KvArgs& c, const KvRows& r, int layer, const KvTensor& k,
                           const KvTensor& v, int type, cudaStream_t stream) {
  return rows_op<true>(c, r, layer, k, v, type, stream);
}
// Few rows per sequence: the kernel that gives each its own CTA or cluster and
// streams the cache once per row; more: tiles of rows on the tensor cores.
cudaError_t launch_kv_attend(const KvArgs& c, const KvRows& r, const KvAttend& a,
                             cudaStream_t stream) {
  if (r.rows == 0) return cudaSuccess;
  return r.max_rows <= 8 ? launch_kv_step(c, r, a, stream) : launch_kv_tiles(c, r, a, stream);
}

}  // namespace qtts
