// The next token of each of many rows of logits: temperature, top-k, top-p, min-p and a draw (include/welvet_cuda.h,
// wv_sample_rows_dev).
//
// Candidates are ordered by a 64-bit word (ordered bits of logit / T : ~index), all distinct. Every cut keeps a prefix of that
// order, so the kept weight is the smallest of the prefixes' weights, and the token is the first one whose running weight
// reaches u times that: what has to be found is where the running count reaches k, where the running weight reaches the
// line of top-p, and where it reaches the draw. Weights count as whole numbers in units of 2^-31, so no sum depends on its order.
//
// A row is read once. A cluster of eight CTAs (one up to 8192 logits) holds its logits / T in shared memory and sorts them into 2048
// bins of 1/64 by their distance from the largest, count and weight of each; the sums over the cluster (distributed shared memory)
// say in which bin each of the three places lies. Where the bins down to the last of those hold no more than 2048 candidates (any
// top-k up to there, any nucleus of so many), these are gathered and sorted, and the rest is a scan over them. Otherwise the
// places are found one after the other, each among the gathered candidates of its own bin; a bin with too many (equal logits) is
// first cut down by further digits of the word.
//
// Bound: HBM for many rows (4 bytes a logit), the cluster's four or five barriers for one. A row that does not fit the cluster's
// shared memory (more than 360448 logits) is walked digit by digit over global memory by one CTA.
#include "wv_common.cuh"
#include <cooperative_groups.h>
#include <math.h>

namespace cg = cooperative_groups;
typedef unsigned long long u64;

__device__ __forceinline__ u64 smp_word(float v, int i) {
  const unsigned u = __float_as_uint(v == 0.f ? 0.f : v);                // -0 and 0 are equal
  const unsigned key = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((u64)key << 32) | (u64)(0xFFFFFFFFu - (unsigned)i);
}
__device__ __forceinline__ float smp_value(u64 w) {
  const unsigned u = (unsigned)(w >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}
__device__ __forceinline__ int smp_index(u64 w) { return (int)(0xFFFFFFFFu - (unsigned)w); }
__device__ __forceinline__ float smp_weight(float y, float top) { return y == top ? 1.f : expf(__fsub_rn(y, top)); }
__device__ __forceinline__ unsigned smp_units(float w) { return __float2uint_rn(w * 2147483648.f); }
// The smallest whole number that is at least f * total, between 1 and total.
__device__ __forceinline__ u64 smp_target(double f, u64 total) {
  const double t = ceil(f * (double)total);
  if (!(t > 1.0)) return 1ull;
  return t >= (double)total ? total : (u64)t;
}
// logit / T; NaN for what is no candidate. A finite logit may become an infinity by the division: it stays a candidate.
__device__ __forceinline__ float smp_y(float x, float t, bool greedy) { return !(x > -INFINITY) ? NAN : greedy ? x : __fdiv_rn(x, t); }

#define SMP_THREADS 512
#define SMP_WARPS (SMP_THREADS / 32)
#define SMP_CLUSTER 8
#define SMP_SMALL 8192
#define SMP_BINS 2048
#define SMP_LIST 2048
#define SMP_CACHE (44 * 1024)              // logits a CTA holds at most

struct SmpArgs {
  const float* logits; int n; long long ld;
  const float* temperature; const int* top_k; const float* top_p; const float* min_p; const double* u;
  int* index; float* prob;
};
// A bin, what comes before it (counts and weight), and its count.
struct SmpSel { int bin; unsigned before, count, pad; u64 weight_before; };

struct __align__(16) SmpShared {
  union {
    unsigned hist[3][SMP_BINS];            // counts, low and high halves of the weights
    u64 run[SMP_LIST];                     // afterwards: the list's running weights
  };
  u64 list[SMP_LIST];
  u64 part[SMP_WARPS], tot_w[SMP_CLUSTER];
  unsigned partc[SMP_WARPS], tot_c[SMP_CLUSTER];
  u64 best, least_sum, result_word, result_cum;
  SmpSel sel[2];
  unsigned filled, turn;
  int place;
};

__device__ __forceinline__ int smp_bin(float y, float top) {
  if (y == top) return 0;
  return min((int)(__fsub_rn(top, y) * 64.f), SMP_BINS - 1);             // rises as y falls: each step rounds monotonously
}

// A CTA adds up its share of the bins over the cluster, the shares' totals go to every CTA, and a place is announced by the CTA whose
// share it is in: reading all bins of all CTAs everywhere (196 KB over distributed shared memory) took 10 us a row.
template <int NCTA> struct SmpScan {
  static constexpr int SHARE = SMP_BINS / NCTA, NB = SHARE > SMP_THREADS ? SHARE / SMP_THREADS : 1;
  unsigned c0, c[NB];                      // counts before the thread's bins, and up to and including each
  u64 w0, w[NB];
  unsigned count;
  u64 all;
};
template <int NCTA>
__device__ __forceinline__ void smp_scan(cg::cluster_group& cluster, SmpShared& S, SmpScan<NCTA>& r) {
  using R = SmpScan<NCTA>;
  constexpr int NB = R::NB;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = NCTA == 1 ? 0 : (int)cluster.block_rank();
  const bool on = tid * NB < R::SHARE;
  unsigned c[NB];
  u64 w[NB];
#pragma unroll
  for (int i = 0; i < NB; i++) { c[i] = 0; w[i] = 0; }
  if (on) {
    const int b0 = rank * R::SHARE + tid * NB;
#pragma unroll
    for (int q = 0; q < NCTA; q++) {
      const SmpShared* o = NCTA == 1 ? &S : cluster.map_shared_rank(&S, q);
#pragma unroll
      for (int i = 0; i < NB; i++) { c[i] += o->hist[0][b0 + i]; w[i] += o->hist[1][b0 + i] + ((u64)o->hist[2][b0 + i] << 16); }
    }
  }
  unsigned ct = 0;
  u64 wt = 0;
#pragma unroll
  for (int i = 0; i < NB; i++) { ct += c[i]; wt += w[i]; }
  const unsigned c_own = ct;
  const u64 w_own = wt;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned a = __shfl_up_sync(0xffffffffu, ct, o);
    const u64 b = __shfl_up_sync(0xffffffffu, wt, o);
    if (lane >= o) { ct += a; wt += b; }
  }
  if (lane == 31) { S.partc[warp] = ct; S.part[warp] = wt; }
  __syncthreads();
  unsigned tc = 0;
  u64 tw = 0;
#pragma unroll
  for (int q = 0; q < SMP_WARPS; q++) {
    if (q == warp) { ct += tc; wt += tw; }
    tc += S.partc[q]; tw += S.part[q];
  }
  if (tid < NCTA) {
    SmpShared* o = NCTA == 1 ? &S : cluster.map_shared_rank(&S, tid);
    o->tot_c[rank] = tc; o->tot_w[rank] = tw;
  }
  if (NCTA == 1) __syncthreads(); else cluster.sync();                   // and every CTA is past its reads of the others' bins
  unsigned cb = 0;
  u64 wb = 0;
  r.count = 0; r.all = 0;
#pragma unroll
  for (int q = 0; q < NCTA; q++) { if (q < rank) { cb += S.tot_c[q]; wb += S.tot_w[q]; } r.count += S.tot_c[q]; r.all += S.tot_w[q]; }
  r.c0 = cb + ct - c_own; r.w0 = wb + wt - w_own;
  unsigned a = r.c0;
  u64 b = r.w0;
#pragma unroll
  for (int i = 0; i < NB; i++) { a += c[i]; b += w[i]; r.c[i] = a; r.w[i] = b; }
}
// The bin in which the running count (or weight) reaches target.
template <int NCTA>
__device__ __forceinline__ SmpSel smp_select(cg::cluster_group& cluster, SmpShared& S, const SmpScan<NCTA>& r, bool by_weight, u64 target, int& turn) {
  using R = SmpScan<NCTA>;
  const int rank = NCTA == 1 ? 0 : (int)cluster.block_rank();
  unsigned cb = r.c0;
  u64 wb = r.w0;
  turn ^= 1;                               // the place of the select before this one may still be read
#pragma unroll
  for (int i = 0; i < R::NB; i++) {
    if (by_weight ? (wb < target && r.w[i] >= target) : (cb < target && r.c[i] >= target)) {
      const SmpSel s{rank * R::SHARE + (int)threadIdx.x * R::NB + i, cb, r.c[i] - cb, 0u, wb};
#pragma unroll
      for (int q = 0; q < NCTA; q++) (NCTA == 1 ? &S : cluster.map_shared_rank(&S, q))->sel[turn] = s;
    }
    cb = r.c[i]; wb = r.w[i];
  }
  if (NCTA == 1) __syncthreads(); else cluster.sync();
  return S.sel[turn];
}
// The first cnt words of the list from the largest down, and their running weights. Up to 256 of them each find their own rank.
__device__ __forceinline__ void smp_sort(SmpShared& S, int cnt, float top) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (cnt <= 256) {
    const u64 mine = tid < cnt ? S.list[tid] : 0ull;
    int at = 0;
    if (warp * 32 < cnt) {
#pragma unroll 4
      for (int j = 0; j < cnt; j++) at += S.list[j] > mine ? 1 : 0;
    }
    __syncthreads();
    if (tid < cnt) S.list[at] = mine;
  } else {
    int p2 = 512;
    while (p2 < cnt) p2 <<= 1;
    for (int i = cnt + tid; i < p2; i += SMP_THREADS) S.list[i] = 0ull;
    __syncthreads();
    for (int size = 2; size <= p2; size <<= 1)
      for (int stride = size >> 1; stride > 0; stride >>= 1) {
        for (int i = tid; i < p2 / 2; i += SMP_THREADS) {
          const int a = 2 * i - (i & (stride - 1)), b = a + stride;
          const u64 x = S.list[a], y = S.list[b];
          if (((a & size) == 0) ? (x < y) : (x > y)) { S.list[a] = y; S.list[b] = x; }
        }
        // steps of up to 32 stay within the 64 words of a warp
        const int next = stride > 1 ? stride >> 1 : size;
        if (stride > 32 || next > 32 || p2 > 2 * SMP_THREADS) __syncthreads(); else __syncwarp();
      }
  }
  __syncthreads();
  constexpr int PER = SMP_LIST / SMP_THREADS;
  u64 v[PER], t = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) { const int q = PER * tid + i; if (q < cnt) t += smp_units(smp_weight(smp_value(S.list[q]), top)); v[i] = t; }
  u64 s = t;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const u64 b = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += b; }
  if (lane == 31) S.part[warp] = s;
  __syncthreads();
  for (int q = 0; q < warp; q++) s += S.part[q];
#pragma unroll
  for (int i = 0; i < PER; i++) S.run[PER * tid + i] = s - t + v[i];
  __syncthreads();
}
// The place in S.run[0 .. cnt) (rising) where the running weight reaches target; the last place if it does not.
__device__ __forceinline__ int smp_place(SmpShared& S, int cnt, u64 target) {
  if (threadIdx.x == 0) S.place = cnt - 1;
  __syncthreads();
  constexpr int PER = SMP_LIST / SMP_THREADS;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int q = PER * (int)threadIdx.x + i;
    if (q < cnt && S.run[q] >= target && (q == 0 || S.run[q - 1] < target)) S.place = q;
  }
  __syncthreads();
  const int at = S.place;
  __syncthreads();
  return at;
}

template <int NCTA>
__global__ void __launch_bounds__(SMP_THREADS, 2) sample_rows_kernel(const SmpArgs A, int per) {
  extern __shared__ __align__(16) unsigned char smp_smem[];
  SmpShared& S = *reinterpret_cast<SmpShared*>(smp_smem);
  float* s_y = reinterpret_cast<float*>(smp_smem + sizeof(SmpShared));
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = NCTA == 1 ? 0 : (int)cluster.block_rank(), row = blockIdx.x / NCTA;
  const int tid = threadIdx.x, lane = tid & 31;
  const int i0 = min(A.n, rank * per), mine = min(A.n - i0, per);
  auto all_sync = [&]() { if (NCTA == 1) __syncthreads(); else cluster.sync(); };
  auto other = [&](int q) { return NCTA == 1 ? &S : cluster.map_shared_rank(&S, q); };
  for (int i = tid; i < 3 * SMP_BINS; i += SMP_THREADS) S.hist[0][i] = 0u;
  if (tid == 0) { S.best = 0ull; S.least_sum = 0ull; S.filled = 0u; }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const float* x = A.logits + (size_t)row * A.ld + i0;
  const float t = A.temperature[row];
  const int k = A.top_k[row];
  const bool greedy = t <= 0.f || k == 1;
  const float least = A.min_p[row];
  const double tp = (double)A.top_p[row], u = A.u[row];
  __syncthreads();
  // ---- the row's logits / T into shared memory, and the largest word
  {
    float best = -INFINITY;
    int at = -1;
    auto take = [&](float v, int i) {
      const float y = smp_y(v, t, greedy);
      if (y > best || (y == best && at < 0)) { best = y; at = i; }       // a thread's places rise: the first of equals
      return y;
    };
    if ((reinterpret_cast<uintptr_t>(x) & 15) == 0 && (per & 3) == 0) {  // i0 is a multiple of per
      constexpr int U = 8;
      const int n4 = mine >> 2;
      for (int b = tid; b < n4; b += U * SMP_THREADS) {
        float4 v[U];
#pragma unroll
        for (int q = 0; q < U; q++) if (b + q * SMP_THREADS < n4) v[q] = __ldcs(reinterpret_cast<const float4*>(x) + b + q * SMP_THREADS);
#pragma unroll
        for (int q = 0; q < U; q++) {
          const int i = 4 * (b + q * SMP_THREADS);
          if (i >= 4 * n4) break;
          const float y0 = take(v[q].x, i), y1 = take(v[q].y, i + 1), y2 = take(v[q].z, i + 2), y3 = take(v[q].w, i + 3);
          *reinterpret_cast<float4*>(s_y + i) = make_float4(y0, y1, y2, y3);
        }
      }
      if (tid < (mine & 3)) { const int i = 4 * n4 + tid; s_y[i] = take(x[i], i); }
    } else {
      for (int b = tid; b < mine; b += 16 * SMP_THREADS) {
        float v[16];
#pragma unroll
        for (int q = 0; q < 16; q++) v[q] = b + q * SMP_THREADS < mine ? __ldcs(x + b + q * SMP_THREADS) : NAN;
#pragma unroll
        for (int q = 0; q < 16; q++) {
          const int i = b + q * SMP_THREADS;
          if (i >= mine) break;
          s_y[i] = take(v[q], i);
        }
      }
    }
    u64 w = at < 0 ? 0ull : smp_word(best, i0 + at);
#pragma unroll
    for (int o = 16; o; o >>= 1) w = max(w, __shfl_xor_sync(0xffffffffu, w, o));
    if (lane == 0 && w) atomicMax(&S.best, w);
  }
  all_sync();
  u64 best = 0ull;
#pragma unroll
  for (int q = 0; q < NCTA; q++) best = max(best, other(q)->best);
  const float top = smp_value(best);
  if (best == 0ull || greedy) {
    if (rank == 0 && tid == 0) { A.index[row] = best ? smp_index(best) : -1; if (A.prob) A.prob[row] = best ? 1.f : 0.f; }
    all_sync();                            // nobody leaves while its shared memory may be read
    return;
  }
  // ---- counts and weights of the bins, and the weight that min-p leaves. Up to 1024 of top-k need the counts alone: the weights of
  // those candidates are taken when they have been sorted.
  auto bins = [&](bool weights) {
    u64 ms = 0ull;
    for (int i = tid; i < mine; i += SMP_THREADS) {
      const float y = s_y[i];
      if (y != y) continue;
      const int b = smp_bin(y, top);
      atomicAdd(&S.hist[0][b], 1u);
      if (weights) {
        const float f = smp_weight(y, top);
        const unsigned w = smp_units(f);
        if (w) { atomicAdd(&S.hist[1][b], w & 0xffffu); atomicAdd(&S.hist[2][b], w >> 16); }
        if (f >= least) ms += w;
      }
    }
    if (weights) {
#pragma unroll
      for (int o = 16; o; o >>= 1) ms += __shfl_xor_sync(0xffffffffu, ms, o);
      if (lane == 0 && ms) atomicAdd(&S.least_sum, ms);
    }
    all_sync();
  };
  int turn = 0;
  SmpScan<NCTA> scan;
  const bool few = k > 0 && k <= SMP_LIST / 2;
  bins(!few);
  smp_scan<NCTA>(cluster, S, scan);
  const bool cut_k = k > 0 && (unsigned)k < scan.count, cut_p = !(tp >= 1.0);
  u64 wmin = 0ull;
  SmpSel end;
  auto least_weight = [&]() {
    wmin = 0ull;
#pragma unroll
    for (int q = 0; q < NCTA; q++) wmin += other(q)->least_sum;
    if (!(least <= 1.f)) wmin = 1ull;      // only the first candidate, and the draw finds no other
  };
  if (!few) least_weight();
  if (few && !cut_k) end = SmpSel{SMP_BINS - 1, 0u, scan.count, 0u, 0ull};
  else end = cut_k ? smp_select<NCTA>(cluster, S, scan, false, (u64)k, turn) : smp_select<NCTA>(cluster, S, scan, true, min(cut_p ? smp_target(tp, scan.all) : scan.all, wmin), turn);

  // words of the logits in bins first .. last whose digits above `himask` are `prefix`, into CTA 0's list
  auto gather = [&](int first, int last, u64 himask, u64 prefix) {
    unsigned* filled = &other(0)->filled;
    u64* list = other(0)->list;
    const float from = (float)first, to = last >= SMP_BINS - 1 ? INFINITY : (float)(last + 1);
    for (int i = tid; i < mine; i += SMP_THREADS) {
      const float y = s_y[i];
      if (y != y) continue;
      const float d = y == top ? 0.f : __fsub_rn(top, y) * 64.f;        // what smp_bin cuts to a whole number
      if (!(d >= from && (d < to || to == INFINITY))) continue;
      const u64 w = smp_word(y, i0 + i);
      if ((w & himask) != prefix) continue;
      const unsigned at = atomicAdd(filled, 1u);
      if (at < SMP_LIST) list[at] = w;
    }
    all_sync();
  };
  auto finish = [&](u64 word, u64 kept) {
    A.index[row] = smp_index(word);
    if (A.prob) A.prob[row] = (float)((double)smp_weight(smp_value(word), top) * 2147483648.0 / (double)kept);
  };

  if (end.before + end.count <= SMP_LIST) {
    gather(0, end.bin, 0ull, 0ull);
    if (rank != 0) return;
    const int cnt = (int)(end.before + end.count);
    smp_sort(S, cnt, top);
    const u64 wk = cut_k ? S.run[k - 1] : few ? S.run[cnt - 1] : scan.all;
    if (few) {                             // the list's first ones that are heavy enough (or all of it, which is more than is kept)
      int heavy = 0;
      for (int q = tid; q < cnt; q += SMP_THREADS) heavy += smp_weight(smp_value(S.list[q]), top) >= least ? 1 : 0;
#pragma unroll
      for (int o = 16; o; o >>= 1) heavy += __shfl_xor_sync(0xffffffffu, heavy, o);
      if (lane == 0) S.partc[tid >> 5] = (unsigned)heavy;
      __syncthreads();
      heavy = 0;
#pragma unroll
      for (int q = 0; q < SMP_WARPS; q++) heavy += (int)S.partc[q];
      wmin = least <= 1.f ? S.run[max(heavy, 1) - 1] : 1ull;
    }
    u64 kept = wk;
    if (cut_p) { const u64 line = smp_target(tp, wk); kept = wmin < line ? wmin : S.run[smp_place(S, cut_k ? k : cnt, line)]; }
    if (wmin < kept) kept = wmin;
    if (!(least <= 1.f)) kept = 1ull << 31;
    const int at = least <= 1.f ? smp_place(S, cnt, smp_target(u, kept)) : 0;
    if (tid == 0) finish(S.list[at], kept);
    return;
  }

  // ---- too many to sort together: the three places one after the other
  if (few) {                               // with weights, after all
    all_sync();
    for (int i = tid; i < 3 * SMP_BINS; i += SMP_THREADS) S.hist[0][i] = 0u;
    __syncthreads();
    bins(true);
    smp_scan<NCTA>(cluster, S, scan);
    least_weight();
  }
  auto find = [&](bool by_weight, u64 target, u64& cum) -> u64 {
    SmpSel s = smp_select<NCTA>(cluster, S, scan, by_weight, target, turn);
    const int bin = s.bin;
    u64 himask = 0ull, prefix = 0ull, before_w = s.weight_before;
    u64 left = target - (by_weight ? s.weight_before : (u64)s.before);
    for (int shift = 64 - 11; s.count > SMP_LIST; shift = max(shift - 11, 0)) {
      for (int i = tid; i < 3 * SMP_BINS; i += SMP_THREADS) S.hist[0][i] = 0u;
      __syncthreads();
      for (int i = tid; i < mine; i += SMP_THREADS) {
        const float y = s_y[i];
        if (y != y || smp_bin(y, top) != bin) continue;
        const u64 w = smp_word(y, i0 + i);
        if ((w & himask) != prefix) continue;
        const int d = SMP_BINS - 1 - (int)((w >> shift) & (SMP_BINS - 1));          // the largest digit first
        const unsigned f = smp_units(smp_weight(y, top));
        atomicAdd(&S.hist[0][d], 1u);
        if (f) { atomicAdd(&S.hist[1][d], f & 0xffffu); atomicAdd(&S.hist[2][d], f >> 16); }
      }
      all_sync();
      SmpScan<NCTA> fine;
      smp_scan<NCTA>(cluster, S, fine);
      s = smp_select<NCTA>(cluster, S, fine, by_weight, left, turn);
      left -= by_weight ? s.weight_before : (u64)s.before;
      before_w += s.weight_before;
      himask = shift ? ~0ull << shift : ~0ull;
      prefix = (prefix & ~((u64)(SMP_BINS - 1) << shift)) | (u64)(SMP_BINS - 1 - s.bin) << shift;
    }
    gather(bin, bin, himask, prefix);
    if (rank == 0) {
      const int cnt = (int)s.count;
      smp_sort(S, cnt, top);
      const int at = by_weight ? smp_place(S, cnt, left) : (int)left - 1;
      if (tid < NCTA) { SmpShared* o = other(tid); o->result_word = S.list[at]; o->result_cum = before_w + S.run[at]; }      // a thread for each CTA tells it
      if (tid == 0) S.filled = 0u;
    }
    all_sync();
    cum = S.result_cum;
    return S.result_word;
  };
  u64 kept = scan.all, cum;
  if (cut_k) { find(false, (u64)k, cum); kept = cum; }
  if (cut_p) { const u64 line = smp_target(tp, kept); if (wmin < line) kept = wmin; else { find(true, line, cum); kept = cum; } }
  if (wmin < kept) kept = wmin;
  const u64 word = least <= 1.f ? find(true, smp_target(u, kept), cum) : best;
  if (!(least <= 1.f)) kept = 1ull << 31;
  if (rank == 0 && tid == 0) finish(word, kept);
  all_sync();
}

// ------------------------------------------------------------------ a row beyond the cluster's shared memory
#define SMW_THREADS 1024
struct SmwRow {
  const float* x; int n; float t; float top;
  __device__ __forceinline__ float y(int i) const { return smp_y(x[i], t, false); }
};
// The word where the running total from the largest down reaches `target`, and the weight up to it. BY_WEIGHT: of weights, else of counts.
template <bool BY_WEIGHT>
__device__ u64 smw_find(const SmwRow& r, u64 target) {
  __shared__ u64 s_hist[256], s_prefix, s_left;
  u64 prefix = 0ull;
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += SMW_THREADS) s_hist[i] = 0ull;
    __syncthreads();
    const u64 himask = shift == 56 ? 0ull : (~0ull << (shift + 8));
    for (int i = threadIdx.x; i < r.n; i += SMW_THREADS) {
      const float v = r.y(i);
      if (v != v) continue;
      const u64 w = smp_word(v, i);
      if ((w & himask) != prefix) continue;
      atomicAdd(&s_hist[(w >> shift) & 255u], BY_WEIGHT ? (u64)smp_units(smp_weight(v, r.top)) : 1ull);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 left = target;
      int d = 255;
      for (; d > 0 && s_hist[d] < left; d--) left -= s_hist[d];
      s_prefix = prefix | ((u64)d << shift);
      s_left = left;
    }
    __syncthreads();
    prefix = s_prefix; target = s_left;
    __syncthreads();
  }
  return prefix;
}
template <typename F> __device__ u64 smw_reduce(u64 v, F f) {
  __shared__ u64 s_part[32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = s_part[0];
  for (int i = 1; i < SMW_THREADS / 32; i++) t = f(t, s_part[i]);
  __syncthreads();
  return t;
}
__global__ void __launch_bounds__(SMW_THREADS, 1) sample_wide_kernel(const SmpArgs A) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int row = blockIdx.x, k = A.top_k[row];
  SmwRow r;
  r.x = A.logits + (size_t)row * A.ld; r.n = A.n; r.t = A.temperature[row];
  const bool greedy = r.t <= 0.f || k == 1;
  auto add = [](u64 a, u64 b) { return a + b; };
  u64 best = 0ull, count = 0ull;
  for (int i = threadIdx.x; i < A.n; i += SMW_THREADS) { const float v = smp_y(r.x[i], r.t, greedy); if (v == v) { best = max(best, smp_word(v, i)); count++; } }
  best = smw_reduce(best, [](u64 a, u64 b) { return max(a, b); });
  count = smw_reduce(count, add);
  if (best == 0ull || greedy) {
    if (threadIdx.x == 0) { A.index[row] = best ? smp_index(best) : -1; if (A.prob) A.prob[row] = best ? 1.f : 0.f; }
    return;
  }
  r.top = smp_value(best);
  // weight of the words from `from` on that are at least `least`
  auto total = [&](u64 from, float least) {
    u64 t = 0;
    for (int i = threadIdx.x; i < A.n; i += SMW_THREADS) {
      const float v = r.y(i);
      if (v != v || smp_word(v, i) < from) continue;
      const float f = smp_weight(v, r.top);
      if (f >= least) t += smp_units(f);
    }
    return smw_reduce(t, add);
  };
  const float least = A.min_p[row];
  const double tp = (double)A.top_p[row];
  u64 kept = total(k > 0 && (u64)k < count ? smw_find<false>(r, (u64)k) : 0ull, 0.f);
  if (!(tp >= 1.0)) kept = total(smw_find<true>(r, smp_target(tp, kept)), 0.f);
  kept = least <= 1.f ? min(kept, total(0ull, least)) : 1ull << 31;
  const u64 word = least <= 1.f ? smw_find<true>(r, smp_target(A.u[row], kept)) : best;
  if (threadIdx.x == 0) {
    A.index[row] = smp_index(word);
    if (A.prob) A.prob[row] = (float)((double)smp_weight(smp_value(word), r.top) * 2147483648.0 / (double)kept);
  }
}

int wv_api_bind_device();
extern "C" int wv_sample_rows_dev(const float* d_logits, int rows, int n, int64_t ld, const float* d_temperature, const int* d_top_k,
                                  const float* d_top_p, const float* d_min_p, const double* d_u, int* d_index, float* d_prob, void* stream) {
  const int dev = wv_api_bind_device();
  if (dev < 0) return dev;
  if (!d_logits || !d_temperature || !d_top_k || !d_top_p || !d_min_p || !d_u || !d_index) { wv_set_error("wv_sample_rows_dev: null pointer"); return WV_EARG; }
  if (rows < 0 || n < 1) { wv_set_error("wv_sample_rows_dev: %d rows of %d logits", rows, n); return WV_ESHAPE; }
  if (ld == 0) ld = n;
  if (ld < n) { wv_set_error("wv_sample_rows_dev: the row stride %lld is less than %d", (long long)ld, n); return WV_ESHAPE; }
  if (rows > INT_MAX / SMP_CLUSTER) { wv_set_error("wv_sample_rows_dev: %d rows are too many", rows); return WV_ESHAPE; }
  if (rows == 0) return WV_OK;
  const SmpArgs A = {d_logits, n, (long long)ld, d_temperature, d_top_k, d_top_p, d_min_p, d_u, d_index, d_prob};
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.stream = static_cast<cudaStream_t>(stream);
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  cudaError_t e;
  if (n > SMP_CLUSTER * SMP_CACHE) {
    cfg.gridDim = dim3(rows); cfg.blockDim = dim3(SMW_THREADS);
    e = cudaLaunchKernelEx(&cfg, sample_wide_kernel, A);
  } else {
    const int ncta = n <= SMP_SMALL ? 1 : SMP_CLUSTER, per = ((n - 1) / ncta + 4) & ~3;
    auto kern = ncta == 1 ? sample_rows_kernel<1> : sample_rows_kernel<SMP_CLUSTER>;
    static unsigned long long attr_mask = 0;     // the attribute is set once per device
    if (dev >= 64 || !(attr_mask & (1ull << dev))) {
      const int most = (int)(sizeof(SmpShared) + SMP_CACHE * 4);
      if (cudaFuncSetAttribute(sample_rows_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess ||
          cudaFuncSetAttribute(sample_rows_kernel<SMP_CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) {
        wv_set_error("wv_sample_rows_dev: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA;
      }
      if (dev < 64) attr_mask |= 1ull << dev;
    }
    cfg.gridDim = dim3((unsigned)(rows * ncta)); cfg.blockDim = dim3(SMP_THREADS); cfg.dynamicSmemBytes = sizeof(SmpShared) + (size_t)per * 4;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)ncta; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kern, A, per);
  }
  if (e != cudaSuccess) { wv_set_error("wv_sample_rows_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA; }
  return WV_OK;
}
