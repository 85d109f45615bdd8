// The paged 8-bit cache as its kernels see it, and how a workgroup finds its work in a
// ragged batch.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cp_host.h"

namespace cp {

struct KvCacheArgs {
  uint8_t *k, *v;           // [pages][heads][block][d], [pages][heads][d][block]
  float *k_scale, *v_scale; // [pages][heads]
  const int* table;         // [batch][max_pages]; an entry outside [0, pages) is no page
  int pages, heads, block, d, max_pages;
};

struct KvBatch {
  const int* offsets;  // [batch + 1] first row of each sequence; null: one row each
  int batch;
};

// Work item `at` of a ragged batch: sequence b, its item'th piece, its first row and row
// count, where count(b, rows of b) says how many pieces a sequence has. Every wave scans
// the batch by itself, 64 sequences a step, so nothing is planned on the host, which does
// not know the lengths. False: the grid is an upper bound and this item is past the end; *item
// is then which one past it.
template <class F>
__device__ __forceinline__ bool kv_locate(const KvBatch& q, int at, F count, int* b, int* item,
                                          int64_t* row0, int* n) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < q.batch; base += 64) {
    const int s = base + lane;
    int r = 0, m = 0, pieces = 0;
    if (s < q.batch) {
      r = q.offsets ? q.offsets[s] : s;
      m = q.offsets ? q.offsets[s + 1] - r : 1;
      m = m < 0 ? 0 : m;
      pieces = count(s, m);
    }
    int sum = pieces;  // inclusive scan
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const int o = __shfl_up(sum, k);
      if (lane >= k) sum += o;
    }
    const int total = __builtin_amdgcn_readlane(sum, 63);
    if (at < total) {
      const unsigned long long hit = __ballot(sum > at);
      const int l = __ffsll(hit) - 1;
      *b = base + l;
      *item = at - __builtin_amdgcn_readlane(sum - pieces, l);
      *row0 = __builtin_amdgcn_readlane(r, l);
      *n = __builtin_amdgcn_readlane(m, l);
      return true;
    }
    at -= total;
  }
  *item = at;
  return false;
}

// Rows that no sequence has: [0, lead) and [tail, rows). Work items past the end of the batch, of
// which a launch with offsets has one at least, clear them in the outputs.
struct KvUnowned {
  int64_t lead, tail;
};

__device__ __forceinline__ KvUnowned kv_unowned(const KvBatch& q, int64_t rows) {
  const int64_t lead = min(max((int64_t)q.offsets[0], (int64_t)0), rows);
  return {lead, min(max((int64_t)q.offsets[q.batch], lead), rows)};
}

int kv_check_cache(const cp_kv_cache* c);
int kv_check_batch(const int* table, int64_t batch, int64_t max_pages, int64_t rows, const int* offsets);
KvCacheArgs kv_args(const cp_kv_cache* c, const int* table, int64_t max_pages);

}  // namespace cp
