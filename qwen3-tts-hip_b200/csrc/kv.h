// Paged key / value caches (16 or 4 bits): launchers of the kernels that
// store, load and attend to rows, and of those that manage pages.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_layout.h"

namespace qtts {

// Bits of the status word (work[0]).
constexpr int kKvOutOfPages = 1;  // a resize or fork found too few free pages and changed nothing
constexpr int kKvBadIndex = 2;    // a page, sequence, length or row count out of range was skipped
constexpr int kKvTimeout = 4;     // a wait inside a kernel ran out (its bound is two seconds)

constexpr int kKvMaxList = 1024;  // sequences of one page-management call

struct KvArgs {
  KvGeom g;
  unsigned char* pool;
  int* table;    // [seqs][max_pages]
  int* lengths;  // length of sequence s: lengths[s * len_stride] + len_add (null: len_add)
  int len_stride, len_add;
  int* refs;     // [pages]; page management only
  int* work;     // status word, then scratch; may be null where only `status` is needed
};

// Rows of a call: group i is rows [row_start[i], row_start[i + 1]) of sequence
// seqs[i], its last rows in order. Null row_start: one row each. Null seqs: i.
struct KvRows {
  const int* seqs;
  const int* row_start;
  int groups, rows, max_rows, max_length;
  int one_group;  // with null row_start: all rows are group 0
};

enum KvType : int { KV_F32 = 0, KV_BF16 = 1 };

struct KvTensor {  // [rows][heads][128], the last dim contiguous; strides in elements
  void* p;
  long long row, head;
};

struct KvAttend {
  KvTensor q, out;
  int type, q_heads;
  float scale;
  int window, sinks, layer;
  const int* halt;  // group i is skipped while halt[i * halt_stride] (null: never)
  int halt_stride;
};

size_t kv_work_ints(const KvGeom& g);

cudaError_t launch_kv_append(const KvArgs& c, const KvRows& r, int layer, const KvTensor& k,
                             const KvTensor& v, int type, cudaStream_t stream);
cudaError_t launch_kv_read(const KvArgs& c, const KvRows& r, int layer, const KvTensor& k,
                           const KvTensor& v, int type, cudaStream_t stream);
// One CTA or cluster per row (and kv head).
cudaError_t launch_kv_step(const KvArgs& c, const KvRows& r, const KvAttend& a,
                           cudaStream_t stream);
// Tiles of rows on the tensor cores.
cudaError_t launch_kv_tiles(const KvArgs& c, const KvRows& r, const KvAttend& a,
                            cudaStream_t stream);
cudaError_t launch_kv_attend(const KvArgs& c, const KvRows& r, const KvAttend& a,
                             cudaStream_t stream);

// QK-RMSNorm and RoPE of projected rows [q | k | v]: q to q_out (fp32), k and v
// stored as launch_kv_append does.
struct KvPrep {
  const float* qkv;        // [rows][ld]
  int ld, q_heads;
  const float *q_gamma, *k_gamma;  // [128]
  float eps;
  const float *rope_cos, *rope_sin;  // [positions][64]
  float* q_out;            // [rows][q_heads * 128]
  int layer;
  const int* halt;         // as KvAttend
  int halt_stride;
};
cudaError_t launch_kv_prep(const KvArgs& c, const KvRows& r, const KvPrep& p, cudaStream_t stream);

struct KvList {
  int n;
  int a[kKvMaxList], b[kKvMaxList];
};
cudaError_t launch_kv_resize(const KvArgs& c, const KvList& l, cudaStream_t stream);
cudaError_t launch_kv_fork(const KvArgs& c, const KvList& l, cudaStream_t stream);
// Drops the pages of the listed sequences: all of them (window < 0), or those
// that lie wholly behind the window and past the sinks.
cudaError_t launch_kv_drop(const KvArgs& c, const KvList& l, int window, int sinks,
                           cudaStream_t stream);
cudaError_t launch_kv_compact(const KvArgs& c, cudaStream_t stream);

}  // namespace qtts
