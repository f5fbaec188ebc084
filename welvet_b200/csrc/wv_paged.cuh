// The paged key/value cache's layout and the device-side reading of a batch, shared by the kernels that write, read and attend
// over it. include/welvet_cuda.h (WvKvPages, WvKvBatch) has the definitions.
#pragma once
#include "wv_common.cuh"
#include <cuda_fp16.h>

// Byte offsets inside a block (one page of one kv head). Every part starts on a 16-byte boundary: page_size and head_dim are
// multiples of 16.
struct WvKvGeom {
  unsigned char* pool;
  int num_pages, page, kvh, hd;
  int code;                       // bytes of a row's codes
  int kscale, vscale, ksub, vsub; // K codes start at 0, V codes at page * code
  long long block;
};
__host__ __device__ inline WvKvGeom wv_kv_geom(const WvKvPages& p) {
  WvKvGeom g;
  g.pool = static_cast<unsigned char*>(p.pool);
  g.num_pages = p.num_pages; g.page = p.page_size; g.kvh = p.num_kv_heads; g.hd = p.head_dim;
  g.code = p.head_dim * p.bits / 8;
  g.kscale = 2 * p.page_size * g.code;
  g.vscale = g.kscale + 4 * p.page_size;
  g.ksub = g.vscale + 4 * p.page_size;
  const int sub = p.bits == 4 ? p.page_size * (p.head_dim / 16) : 0;
  g.vsub = g.ksub + sub;
  g.block = (long long)g.vsub + sub;
  return g;
}

// Codes in the sticky status word of paged calls.
#define WV_PAGED_LENGTH 1        // q_start or kv_len outside its bounds
#define WV_PAGED_PAGE 2          // a page number outside the pool
__device__ __forceinline__ void wv_paged_report(int* err, int code) { if (err) atomicCAS_system(err, 0, code); }

// A sequence of the batch, cut to the call's bounds: rows q0 .. q1 - 1 of q, the first of them at position p0; kv tokens in the cache.
// Of more than max_q new tokens the first ones stay, at their places.
struct WvSeq { int q0, q1, kv, p0; };
__device__ __forceinline__ WvSeq wv_seq(const WvKvBatch& b, int page, int s, int* err) {
  WvSeq q;
  const int a = b.q_start[s], e = b.q_start[s + 1], k = b.kv_len[s];
  q.q0 = min(max(a, 0), b.total_q);
  q.q1 = min(max(e, q.q0), b.total_q);
  q.kv = min(max(k, 0), b.max_kv);      // max_kv <= table_stride * page_size: the host checked
  q.p0 = q.kv - (q.q1 - q.q0);
  if (q.q0 != a || q.q1 != e || q.kv != k || q.q1 - q.q0 > b.max_q) wv_paged_report(err, WV_PAGED_LENGTH);
  if (q.q1 - q.q0 > b.max_q) q.q1 = q.q0 + b.max_q;
  return q;
}
// The sequence that row `row` of q belongs to (num_seqs: none), found by a whole warp: the first s with q_start[s + 1] > row.
// The loads of 32 sequences at a time do not depend on one another; a binary search would be a chain of round trips to L2.
__device__ __forceinline__ int wv_seq_of_row(const WvKvBatch& b, int row) {
  const int lane = threadIdx.x & 31;
  for (int s0 = 0; s0 < b.num_seqs; s0 += 128) {
    bool past[4];
#pragma unroll
    for (int u = 0; u < 4; u++) { const int s = s0 + 32 * u + lane; past[u] = s < b.num_seqs && b.q_start[s + 1] > row; }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const unsigned m = __ballot_sync(0xffffffffu, past[u]);
      if (m) return s0 + 32 * u + __ffs(m) - 1;
    }
  }
  return b.num_seqs;
}

int* wv_paged_err_ptr();          // wv_gemv_tma.cu: device address of the paged calls' status word (mapped host memory)
