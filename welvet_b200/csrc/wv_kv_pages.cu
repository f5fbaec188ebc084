// The pages of a paged cache as a table on the device (include/welvet_cuda.h, WvKvTable): sequences are forked, extended, trimmed and
// freed, and a scattered pool is moved to its front.
//
// The table's calls read a few integers a sequence and the pool's counts once: what bounds them is latency, a chain of three or
// four dependent loads and the launch. Which pages are free follows from the counts alone (no list that a call could leave behind in another
// order), and a call gives them out in rising order to the sequences in theirs, so every result is the same in each run: the places come from
// sums over warps' counts, not from atomics. One cluster of eight CTAs walks the counts, each of its 128 warps its own stretch, twice: once
// to count, once to write down what it found, with one exchange of the 128 counts between (distributed shared memory).
// Measured, us from a graph: trimming 64 sequences 1.7; extending 64 by a token each 6.2 for a pool of 2000 pages, 6.4 of 20,000, 8.9 of 200,000, 18.5 of
// a million; compacting with nothing to move 6.4, 6.6, 14.0, 45.8 (its walk writes both lists, and a million pages are 8192 a warp).
//
// Copies of pages are bound by HBM: a block of 256 threads moves 16 KB at a time, four 16-byte pieces a thread under way. A compaction that moves 322 MB
// takes 126 us, 5.1 TB/s of reads and writes together where a plain copy reaches 6.5.
#include "wv_paged.cuh"
#include "wv_lease.h"
#include <algorithm>
#include <cooperative_groups.h>
#include <limits.h>
namespace cg = cooperative_groups;

int wv_sm_count();
int wv_api_bind_device();

#define KP_CTAS 8               // of the cluster
#define KP_THREADS 512
#define KP_WARPS (KP_THREADS / 32)
#define KP_ALL (KP_CTAS * KP_WARPS)
#define KP_ENTRY 128            // threads of a trim's or a fork's entry
#define KP_POOLS 128            // pools of a copy's launch
#define KP_PIECES 1024u         // 16-byte pieces of a copy's item
#define KP_MOST (1 << 30)       // pages, sequences and a row's places: the walks look up to 512 places ahead in 32 bits

__device__ __forceinline__ void kp_start() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// The tokens of sequence s, cut to what its row of the table holds.
__device__ __forceinline__ int kp_len(const WvKvTable& t, int s, int* err) {
  const int n = t.kv_len[s];
  const long long most = (long long)t.table_stride * t.page_size;
  const int cut = n < 0 ? 0 : n > most ? (int)most : n;
  if (cut != n) wv_paged_report(err, WV_PAGED_LENGTH);
  return cut;
}
__device__ __forceinline__ int kp_pages(const WvKvTable& t, long long tokens) { return (int)((tokens + t.page_size - 1) / t.page_size); }
__device__ __forceinline__ bool kp_in(const WvKvTable& t, int page, int* err) {
  if (page >= 0 && page < t.num_pages) return true;
  wv_paged_report(err, WV_PAGED_PAGE);
  return false;
}
// Whether any of v[0 .. n) is x, by the whole block.
__device__ __forceinline__ bool kp_any(const int* v, int n, int x) {
  bool hit = false;
  for (int i = threadIdx.x; i < n; i += KP_ENTRY) hit |= v[i] == x;
  return __syncthreads_or(hit) != 0;
}

// ------------------------------------------------------------------ a block an entry
__global__ void __launch_bounds__(KP_ENTRY) kv_trim_kernel(const WvKvTable t, const int* __restrict__ seqs, const int* __restrict__ keep, int* err) {
  kp_start();
  const int e = blockIdx.x, s = seqs ? seqs[e] : e;
  if (seqs) {
    if (s < 0 || s >= t.num_seqs) { if (threadIdx.x == 0) wv_paged_report(err, WV_PAGED_SEQ); return; }
    if (kp_any(seqs, e, s)) { if (threadIdx.x == 0) wv_paged_report(err, WV_PAGED_SEQ); return; }      // the first entry of a sequence counts
  }
  const int len = kp_len(t, s, err), k = keep ? keep[e] : 0;
  if (k < 0) { if (threadIdx.x == 0) wv_paged_report(err, WV_PAGED_LENGTH); return; }
  if (k >= len) return;
  int* row = t.pages + (size_t)s * t.table_stride;
  for (int j = kp_pages(t, k) + threadIdx.x, held = kp_pages(t, len); j < held; j += KP_ENTRY) {
    const int p = row[j];
    if (kp_in(t, p, err) && atomicSub(&t.refs[p], 1) <= 0) { atomicAdd(&t.refs[p], 1); wv_paged_report(err, WV_PAGED_REFS); }
    row[j] = -1;
  }
  __syncthreads();                                       // every thread has read the length
  if (threadIdx.x == 0) t.kv_len[s] = k;
}

__global__ void __launch_bounds__(KP_ENTRY) kv_fork_kernel(const WvKvTable t, const int* __restrict__ src, const int* __restrict__ dst, const int* __restrict__ keep, int n, int* err) {
  kp_start();
  const int e = blockIdx.x, a = src[e], b = dst[e];
  bool ok = a >= 0 && a < t.num_seqs && b >= 0 && b < t.num_seqs && a != b;
  if (ok) ok = !kp_any(dst, e, b) && !kp_any(dst, n, a); // the first entry of a target counts, and no target is a source
  if (ok) ok = t.kv_len[b] == 0;
  if (!ok) { if (threadIdx.x == 0) wv_paged_report(err, WV_PAGED_SEQ); return; }
  int len = kp_len(t, a, err);
  if (keep) {
    const int k = keep[e];
    if (k < 0) { if (threadIdx.x == 0) wv_paged_report(err, WV_PAGED_LENGTH); return; }
    len = min(len, k);
  }
  const int* from = t.pages + (size_t)a * t.table_stride;
  int* to = t.pages + (size_t)b * t.table_stride;
  for (int j = threadIdx.x, held = kp_pages(t, len); j < held; j += KP_ENTRY) {
    const int p = from[j];
    if (kp_in(t, p, err)) atomicAdd(&t.refs[p], 1);
    to[j] = p;
  }
  __syncthreads();
  if (threadIdx.x == 0) t.kv_len[b] = len;
}

// ------------------------------------------------------------------ the cluster's walk over the counts
struct KpShared { int used[KP_WARPS], idle[KP_WARPS], gaps[KP_WARPS], need; };
// A warp's stretch of the pool's pages, and what it holds.
struct KpWalk {
  int first, last, lane;                                 // pages [first, last)
  int idle0, used0, idle, used;                          // free and held pages before the stretch, and in the whole pool
};
// counts -> S.idle, S.used of this warp
__device__ __forceinline__ void kp_count(const WvKvTable& t, KpShared& S, KpWalk& w, int gw) {
  const int each = ((t.num_pages + KP_ALL - 1) / KP_ALL + 31) & ~31;
  w.lane = threadIdx.x & 31;
  w.first = (int)min((long long)gw * each, (long long)t.num_pages);
  w.last = (int)min((long long)w.first + each, (long long)t.num_pages);
  int idle = 0;
  for (int p = w.first + w.lane; p < w.last; p += 256) {
    int r[8];
#pragma unroll
    for (int u = 0; u < 8; u++) r[u] = p + 32 * u < w.last ? t.refs[p + 32 * u] : 1;
#pragma unroll
    for (int u = 0; u < 8; u++) idle += r[u] == 0;
  }
  idle = __reduce_add_sync(0xffffffffu, idle);
  if (w.lane == 0) { S.idle[threadIdx.x >> 5] = idle; S.used[threadIdx.x >> 5] = w.last - w.first - idle; }
}
// after the cluster's barrier: the sums before this warp and over all, out of every CTA's shared memory
__device__ __forceinline__ void kp_sums(cg::cluster_group& cluster, KpShared& S, KpWalk& w, int gw) {
  int idle0 = 0, used0 = 0, idle = 0, used = 0;
#pragma unroll
  for (int i = 0; i < KP_ALL / 32; i++) {
    const int at = 32 * i + w.lane;
    const KpShared* o = cluster.map_shared_rank(&S, at / KP_WARPS);
    const int a = o->idle[at % KP_WARPS], b = o->used[at % KP_WARPS];
    idle += a; used += b;
    if (at < gw) { idle0 += a; used0 += b; }
  }
  w.idle0 = __reduce_add_sync(0xffffffffu, idle0); w.used0 = __reduce_add_sync(0xffffffffu, used0);
  w.idle = __reduce_add_sync(0xffffffffu, idle); w.used = __reduce_add_sync(0xffffffffu, used);
}
// f(page, free?, rank among its kind) for every page of the stretch
template <class F> __device__ __forceinline__ void kp_walk(const WvKvTable& t, const KpWalk& w, F f) {
  int idle = w.idle0, used = w.used0;
  const unsigned below = (1u << w.lane) - 1u;
  for (int p0 = w.first; p0 < w.last; p0 += 256) {
    int r[8];
#pragma unroll
    for (int u = 0; u < 8; u++) { const int p = p0 + 32 * u + w.lane; r[u] = p < w.last ? t.refs[p] : 1; }
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const int p = p0 + 32 * u + w.lane;
      const unsigned here = __ballot_sync(0xffffffffu, p < w.last), m = __ballot_sync(0xffffffffu, r[u] == 0);
      if (p < w.last) f(p, r[u] == 0, r[u] == 0 ? idle + __popc(m & below) : used + __popc(here & ~m & below));
      idle += __popc(m);
      used += __popc(here & ~m);
    }
  }
}

// Scratch of a call in ints: extend: {jobs, -}, place of each sequence's first page among the free ones and its need, the free pages, the
// copies' sources and targets. compact: {jobs, -}, held pages in order, free pages in order, the new numbers.
struct KpScratch { int *head, *a, *b, *c, *d; };

// Sequence s wants add[s] tokens: its new pages, one of them for a copy of its last page (bit 30) if that is shared and partly filled; -1: it
// cannot have them whatever is free.
__device__ __forceinline__ int kp_need(const WvKvTable& t, const int* add, int s, int* err) {
  const int n = add[s], len = t.kv_len[s];
  if (n == 0) return 0;
  const long long most = min((long long)t.table_stride * t.page_size, (long long)INT_MAX);
  if (n < 0 || len < 0 || len > most) { wv_paged_report(err, WV_PAGED_LENGTH); return -1; }
  if ((long long)len + n > most) return -1;
  const int held = kp_pages(t, len);
  int need = kp_pages(t, (long long)len + n) - held;
  if (len % t.page_size) {
    const int p = t.pages[(size_t)s * t.table_stride + held - 1];
    if (!kp_in(t, p, err)) return -1;
    if (t.refs[p] > 1) need = (need + 1) | 1 << 30;
  }
  return need;
}

__global__ void __launch_bounds__(KP_THREADS) __cluster_dims__(KP_CTAS, 1, 1) kv_extend_kernel(const WvKvTable t, const int* __restrict__ add, int* __restrict__ granted, const KpScratch x, int* err) {
  __shared__ KpShared S;
  __shared__ long long s_sum[KP_WARPS];
  cg::cluster_group cluster = cg::this_cluster();
  kp_start();
  const int rank = (int)cluster.block_rank(), tid = threadIdx.x, warp = tid >> 5, gw = rank * KP_WARPS + warp;
  KpWalk w;
  kp_count(t, S, w, gw);
  if (rank == 0) {                                       // what the sequences want, and where each one's pages begin among the free ones
    if (tid == 0) x.head[0] = 0;
    long long before = 0;
    for (int s0 = 0; s0 < t.num_seqs; s0 += KP_THREADS) {
      const int s = s0 + tid, need = s < t.num_seqs ? kp_need(t, add, s, err) : 0, n = need < 0 ? 0 : need & ~(1 << 30);
      long long upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const long long v = __shfl_up_sync(0xffffffffu, upto, o); if (w.lane >= o) upto += v; }
      if (w.lane == 31) s_sum[warp] = upto;
      __syncthreads();
      long long at = before;
#pragma unroll
      for (int i = 0; i < KP_WARPS; i++) { at += i < warp ? s_sum[i] : 0; before += s_sum[i]; }
      if (s < t.num_seqs) { x.a[s] = (int)min(at + upto - n, (long long)INT_MAX); x.b[s] = need; }
      __syncthreads();
    }
    if (tid == 0) S.need = (int)min(before, (long long)INT_MAX);
  }
  cluster.sync();
  kp_sums(cluster, S, w, gw);
  const int need = cluster.map_shared_rank(&S, 0)->need;
  if (w.idle0 < need) kp_walk(t, w, [&](int p, bool idle, int r) { if (idle && r < need) x.c[r] = p; });
  cluster.sync();                                        // the list is there, and nobody reads the counts as they were any more
  for (int s = rank * KP_THREADS + tid; s < t.num_seqs; s += KP_CTAS * KP_THREADS) {
    const int want = x.b[s], n = want & ~(1 << 30), at = x.a[s];
    const bool ok = want >= 0 && (n == 0 || (long long)at + n <= w.idle);
    if (granted) granted[s] = ok;
    if (!ok || add[s] == 0) continue;
    const int len = t.kv_len[s], held = kp_pages(t, len);
    int* row = t.pages + (size_t)s * t.table_stride;
    int k = 0;
    if (want >> 30 & 1) {
      const int old = row[held - 1], p = x.c[at];
      atomicSub(&t.refs[old], 1);
      t.refs[p] = 1;
      row[held - 1] = p;
      const int j = atomicAdd(x.head, 1);                // the copies' order is no result
      x.d[2 * j] = old; x.d[2 * j + 1] = p;
      k = 1;
    }
    for (int j = held; k < n; k++, j++) { const int p = x.c[at + k]; t.refs[p] = 1; row[j] = p; }
    t.kv_len[s] = len + add[s];
  }
}

__global__ void __launch_bounds__(KP_THREADS) __cluster_dims__(KP_CTAS, 1, 1) kv_compact_kernel(const WvKvTable t, const KpScratch x, int* __restrict__ live) {
  __shared__ KpShared S;
  cg::cluster_group cluster = cg::this_cluster();
  kp_start();
  const int rank = (int)cluster.block_rank(), tid = threadIdx.x, warp = tid >> 5, gw = rank * KP_WARPS + warp;
  KpWalk w;
  kp_count(t, S, w, gw);
  cluster.sync();
  kp_sums(cluster, S, w, gw);
  const int L = w.used;
  int gaps = 0;                                          // free pages in front of L: as many as there are held ones from L on
  kp_walk(t, w, [&](int p, bool idle, int r) {
    (idle ? x.b : x.a)[r] = p;
    gaps += idle && p < L;
    if (idle && p >= L) x.c[p] = p;                      // a table that holds a page nobody counted keeps it
  });
  gaps = __reduce_add_sync(0xffffffffu, gaps);
  if (w.lane == 0) S.gaps[warp] = gaps;
  cluster.sync();
  int m = 0;
#pragma unroll
  for (int i = 0; i < KP_ALL / 32; i++) {
    const int at = 32 * i + w.lane;
    m += cluster.map_shared_rank(&S, at / KP_WARPS)->gaps[at % KP_WARPS];
  }
  m = __reduce_add_sync(0xffffffffu, m);
  for (int k = rank * KP_THREADS + tid; k < m; k += KP_CTAS * KP_THREADS) {
    const int src = x.a[L - m + k], dst = x.b[k];
    x.c[src] = dst;
    t.refs[dst] = t.refs[src];
    t.refs[src] = 0;
    x.d[2 * k] = src; x.d[2 * k + 1] = dst;
  }
  if (rank == 0 && tid == 0) { x.head[0] = m; x.head[1] = L; *live = L; }
  cluster.sync();                                        // nobody leaves while another reads its shared memory
}
// The tables' entries after a compaction.
__global__ void __launch_bounds__(256) kv_renumber_kernel(const WvKvTable t, const KpScratch x, int* err) {
  kp_start();
  const int L = x.head[1];
  if (x.head[0] == 0) return;
  for (int s = blockIdx.x; s < t.num_seqs; s += gridDim.x) {
    int* row = t.pages + (size_t)s * t.table_stride;
    for (int j = blockIdx.y * 256 + threadIdx.x, held = kp_pages(t, kp_len(t, s, err)); j < held; j += 256 * gridDim.y) {
      const int p = row[j];
      if (p < L && p >= 0) continue;
      if (!kp_in(t, p, err)) continue;
      row[j] = x.c[p];
    }
  }
}

// ------------------------------------------------------------------ copies
struct KpPools { unsigned char* p[KP_POOLS]; unsigned n16[KP_POOLS]; int n; unsigned chunks; };      // 16-byte pieces of a page; items of the largest page
// Job i copies page src[i * step] to dst[i * step] in all pools; there are *count of them, n at most.
__global__ void __launch_bounds__(256) kv_copy_kernel(const __grid_constant__ KpPools P, const int* __restrict__ src, const int* __restrict__ dst, int step, const int* __restrict__ count, int n,
                                                      int num_pages, int* err) {
  kp_start();
  if (count) n = min(n, *count);
  const long long all = (long long)n * P.n * P.chunks;
  for (long long i = blockIdx.x; i < all; i += gridDim.x) {
    const long long of = i / P.chunks;
    const unsigned c = (unsigned)(i - of * P.chunks);
    const int job = (int)(of / P.n), k = (int)(of - (long long)job * P.n);
    const int a = src[(size_t)job * step], b = dst[(size_t)job * step];
    if (a < 0 || a >= num_pages || b < 0 || b >= num_pages) { if (threadIdx.x == 0) wv_paged_report(err, WV_PAGED_PAGE); continue; }
    if (a == b) continue;
    const unsigned n16 = P.n16[k];
    const uint4* from = reinterpret_cast<const uint4*>(P.p[k]) + (size_t)a * n16;
    uint4* to = reinterpret_cast<uint4*>(P.p[k]) + (size_t)b * n16;
    uint4 v[KP_PIECES / 256];
#pragma unroll
    for (unsigned u = 0; u < KP_PIECES / 256; u++) { const unsigned at = c * KP_PIECES + u * 256 + threadIdx.x; if (at < n16) v[u] = from[at]; }
#pragma unroll
    for (unsigned u = 0; u < KP_PIECES / 256; u++) { const unsigned at = c * KP_PIECES + u * 256 + threadIdx.x; if (at < n16) to[at] = v[u]; }
  }
}

// ------------------------------------------------------------------ host
template <class... K, class... A> static cudaError_t kp_go(void (*kern)(K...), dim3 grid, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  cfg.gridDim = grid; cfg.blockDim = dim3((unsigned)threads); cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, K(args)...);
}
static int kp_done(const char* who, cudaError_t e) {
  if (e == cudaSuccess) return WV_OK;
  cudaGetLastError();
  wv_set_error("%s: launch: %s", who, cudaGetErrorString(e));
  return WV_ECUDA;
}
static int kp_table(const char* who, const WvKvTable* t) {
  if (!t || !t->refs || !t->pages || !t->kv_len) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  if (t->num_pages < 1 || t->num_seqs < 1 || t->table_stride < 1 || !wv_kv_shape_ok(16, t->page_size, 16)) {
    wv_set_error("%s: %d pages of %d, %d sequences of up to %d pages (a page holds a multiple of 16 tokens)", who, t->num_pages, t->page_size, t->num_seqs, t->table_stride);
    return WV_ESHAPE;
  }
  if (std::max(t->num_pages, std::max(t->num_seqs, t->table_stride)) > KP_MOST) {
    wv_set_error("%s: %d pages, %d sequences of up to %d pages (at most %d each)", who, t->num_pages, t->num_seqs, t->table_stride, KP_MOST);
    return WV_ESHAPE;
  }
  return WV_OK;
}
// pools of one geometry of pages; num_pages, page_size 0: those of the first
static int kp_pools(const char* who, const WvKvPages* pools, int num, int num_pages, int page_size) {
  if (num < 0 || (num > 0 && !pools)) { wv_set_error("%s: %d pools at %p", who, num, (const void*)pools); return WV_EARG; }
  for (int i = 0; i < num; i++) {
    const WvKvPages& k = pools[i];
    if (!k.pool) { wv_set_error("%s: pool %d is null", who, i); return WV_EARG; }
    if (k.bits != 16 && k.bits != 8 && k.bits != 4) { wv_set_error("%s: %d bits (16, 8 or 4)", who, k.bits); return WV_EFORMAT; }
    if (!wv_kv_shape_ok(k.bits, k.page_size, k.head_dim) || k.num_kv_heads < 1 || wv_kv_geom(k).block / 16 * k.num_kv_heads > UINT_MAX - KP_PIECES) {
      wv_set_error("%s: pool %d: pages of %d, %d kv heads of %d", who, i, k.page_size, k.num_kv_heads, k.head_dim);
      return WV_ESHAPE;
    }
    if (k.num_pages != num_pages || k.page_size != page_size) {
      wv_set_error("%s: pool %d has %d pages of %d tokens, not %d of %d", who, i, k.num_pages, k.page_size, num_pages, page_size); return WV_ESHAPE;
    }
    if (reinterpret_cast<uintptr_t>(k.pool) & 15) { wv_set_error("%s: pool %d is not 16-byte aligned", who, i); return WV_EARG; }
  }
  return WV_OK;
}
static cudaError_t kp_copy(const WvKvPages* pools, int num, const int* src, const int* dst, int step, const int* count, int n, cudaStream_t st) {
  for (int i0 = 0; i0 < num && n > 0; i0 += KP_POOLS) {
    KpPools P = {};
    P.n = std::min(KP_POOLS, num - i0);
    unsigned most = 0;
    for (int i = 0; i < P.n; i++) {
      P.p[i] = static_cast<unsigned char*>(pools[i0 + i].pool);
      P.n16[i] = (unsigned)(wv_kv_geom(pools[i0 + i]).block / 16 * pools[i0 + i].num_kv_heads);
      most = std::max(most, P.n16[i]);
    }
    P.chunks = (most + KP_PIECES - 1) / KP_PIECES;
    const long long items = (long long)n * P.n * P.chunks;
    const unsigned grid = (unsigned)std::min(items, 8LL * wv_sm_count());
    const cudaError_t e = kp_go(kv_copy_kernel, dim3(grid), 256, st, P, src, dst, step, count, n, pools[0].num_pages, wv_paged_err_ptr());
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

extern "C" int wv_kv_trim_dev(const WvKvTable* table, const int* d_seqs, const int* d_keep, int n, void* stream) {
  const char* who = "wv_kv_trim_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = kp_table(who, table))) return rc;
  if (n < 0 || n > table->num_seqs) { wv_set_error("%s: %d entries of %d sequences", who, n, table->num_seqs); return WV_ESHAPE; }
  if (n == 0) return WV_OK;
  return kp_done(who, kp_go(kv_trim_kernel, dim3((unsigned)n), KP_ENTRY, static_cast<cudaStream_t>(stream), *table, d_seqs, d_keep, wv_paged_err_ptr()));
}

extern "C" int wv_kv_fork_dev(const WvKvTable* table, const int* d_src, const int* d_dst, const int* d_keep, int n, void* stream) {
  const char* who = "wv_kv_fork_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = kp_table(who, table))) return rc;
  if (n < 0 || n > table->num_seqs) { wv_set_error("%s: %d entries of %d sequences", who, n, table->num_seqs); return WV_ESHAPE; }
  if (n == 0) return WV_OK;
  if (!d_src || !d_dst) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  return kp_done(who, kp_go(kv_fork_kernel, dim3((unsigned)n), KP_ENTRY, static_cast<cudaStream_t>(stream), *table, d_src, d_dst, d_keep, n, wv_paged_err_ptr()));
}

extern "C" int wv_kv_extend_dev(const WvKvTable* table, const int* d_add, int* d_granted, const WvKvPages* pools, int num_pools, void* stream) {
  const char* who = "wv_kv_extend_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = kp_table(who, table)) || (rc = kp_pools(who, pools, num_pools, table->num_pages, table->page_size))) return rc;
  if (!d_add) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  WvLease lease;
  const size_t ns = (size_t)table->num_seqs;
  if ((rc = wv_lease(lease, 4 + 4 * ns + (size_t)table->num_pages, st, "wv_kv_extend_dev: the free pages"))) return rc;
  int* p = reinterpret_cast<int*>(lease.p);
  const KpScratch x = {p, p + 4, p + 4 + ns, p + 4 + 4 * ns, p + 4 + 2 * ns};
  cudaError_t e = kp_go(kv_extend_kernel, dim3(KP_CTAS), KP_THREADS, st, *table, d_add, d_granted, x, wv_paged_err_ptr());
  if (e == cudaSuccess) e = kp_copy(pools, num_pools, x.d, x.d + 1, 2, x.head, table->num_seqs, st);
  return kp_done(who, e);
}

extern "C" int wv_kv_compact_dev(const WvKvTable* table, const WvKvPages* pools, int num_pools, int* d_live, void* stream) {
  const char* who = "wv_kv_compact_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = kp_table(who, table)) || (rc = kp_pools(who, pools, num_pools, table->num_pages, table->page_size))) return rc;
  if (!d_live) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  WvLease lease;
  const size_t np = (size_t)table->num_pages;
  if ((rc = wv_lease(lease, 4 + 5 * np, st, "wv_kv_compact_dev: the pages' order"))) return rc;
  int* p = reinterpret_cast<int*>(lease.p);
  const KpScratch x = {p, p + 4, p + 4 + np, p + 4 + 2 * np, p + 4 + 3 * np};
  cudaError_t e = kp_go(kv_compact_kernel, dim3(KP_CTAS), KP_THREADS, st, *table, x, d_live);
  if (e == cudaSuccess) {
    const unsigned rows = (unsigned)std::min(table->num_seqs, 1024);
    const unsigned cols = (unsigned)std::min((table->table_stride + 255) / 256, std::max(1, 2048 / (int)rows));
    e = kp_go(kv_renumber_kernel, dim3(rows, cols), 256, st, *table, x, wv_paged_err_ptr());
  }
  // half of the pages at most lie behind as many free ones
  if (e == cudaSuccess) e = kp_copy(pools, num_pools, x.d, x.d + 1, 2, x.head, table->num_pages / 2, st);
  return kp_done(who, e);
}

extern "C" int wv_kv_copy_dev(const WvKvPages* pools, int num_pools, const int* d_src, const int* d_dst, int n, void* stream) {
  const char* who = "wv_kv_copy_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if (num_pools < 1 || !pools) { wv_set_error("%s: %d pools at %p", who, num_pools, (const void*)pools); return WV_EARG; }
  if (pools[0].num_pages < 1) { wv_set_error("%s: %d pages", who, pools[0].num_pages); return WV_ESHAPE; }
  if ((rc = kp_pools(who, pools, num_pools, pools[0].num_pages, pools[0].page_size))) return rc;
  if (n < 0) { wv_set_error("%s: %d pages to copy", who, n); return WV_ESHAPE; }
  if (n == 0) return WV_OK;
  if (!d_src || !d_dst) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  return kp_done(who, kp_copy(pools, num_pools, d_src, d_dst, 1, nullptr, n, static_cast<cudaStream_t>(stream)));
}
