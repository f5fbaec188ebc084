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
// say in which bin each of the three places lies. With top-k up to 1024 the bins hold the threads' largest alone, an entry a thread
// instead of one a logit. Where the bins down to the last of the places hold no more than 2048 candidates, these are gathered and
// sorted, and the rest is a scan over them. Otherwise the places are found one after the other, each among the gathered candidates of
// its own bin; a bin with too many (equal logits) is first cut down by further digits of the word.
//
// Bound: the cluster's five to ten barriers (0.8 us each, more beside another cluster on the same SMs), with the load, a scan or a sort
// of 1 to 3 us between two of them. One row of 128256 logits with top-k 40 takes 11.6 us (16 with an entry a logit and division by
// division), 128 rows with mixed cuts 71 us, 0.9 TB/s: 33 clusters run at once, for a CTA holds 64 KB of logits beside 41 KB of bins
// and list, and a row without top-k takes 25 us of which 7 are the three sums of every logit in its bin. A row that does not fit the
// cluster's shared memory (more than 360448 logits) is walked digit by digit over global memory by one CTA.
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
// top - y; 0 for the largest itself, be it an infinity.
__device__ __forceinline__ float smp_distance(float y, float top) { return fmaxf(__fsub_rn(top, y), 0.f); }
__device__ __forceinline__ float smp_weight(float y, float top) { return expf(-smp_distance(y, top)); }
__device__ __forceinline__ unsigned smp_units(float w) { return __float2uint_rn(w * 2147483648.f); }
// The smallest whole number that is at least f * total, between 1 and total.
__device__ __forceinline__ u64 smp_target(double f, u64 total) {
  const double t = ceil(f * (double)total);
  if (!(t > 1.0)) return 1ull;
  return t >= (double)total ? total : (u64)t;
}
// logit / T; NaN for what is no candidate. A finite logit may become an infinity by the division: it stays a candidate.
__device__ __forceinline__ float smp_y(float x, float t, bool greedy) { return !(x > -INFINITY) ? NAN : greedy ? x : __fdiv_rn(x, t); }
// The same for four logits, by the reciprocal: with r the rounded 1/t, q within an ulp of x/t and the remainder x - q t exact, q + (x - q t) r
// rounds to the rounded quotient (P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990). The
// product x r is within one and a half ulps, so the step is done twice: 2.5 instructions a logit in pairs, where the division with its
// test and branch takes about 14. The remainder is exact and nothing overflows for 2^-20 <= t <= 2^20 (`quick`) and
// 2^-100 <= |x| <= 2^100; a group of four with another number is divided one by one. NaN stays NaN.
__device__ __forceinline__ float4 smp_y4(float4 x, float t, float r, bool quick) {
  const float hi = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
  const float lo = fminf(fminf(fabsf(x.x), fabsf(x.y)), fminf(fabsf(x.z), fabsf(x.w)));
  if (!(quick && hi <= 0x1p100f && lo >= 0x1p-100f)) return make_float4(smp_y(x.x, t, false), smp_y(x.y, t, false), smp_y(x.z, t, false), smp_y(x.w, t, false));
  const float2 a = make_float2(x.x, x.y), b = make_float2(x.z, x.w), rr = make_float2(r, r), nt = make_float2(-t, -t);
  float2 p = __fmul2_rn(a, rr), q = __fmul2_rn(b, rr);
#pragma unroll
  for (int i = 0; i < 2; i++) {
    p = __ffma2_rn(__ffma2_rn(p, nt, a), rr, p);
    q = __ffma2_rn(__ffma2_rn(q, nt, b), rr, q);
  }
  return make_float4(p.x, p.y, q.x, q.y);
}

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
  unsigned filled, own, from;              // words in CTA 0's list, the CTA's own of them, and where those begin
  int place[2];
};

// The whole part of 64 times the distance, at most 2047, by a sum that rounds down: it rises as y falls, for each step rounds monotonously.
__device__ __forceinline__ int smp_bin(float y, float top) {
  const float d = fminf(smp_distance(y, top), 31.999998f);
  return __float_as_int(__fmaf_rd(d, 64.f, 8388608.f)) - 0x4b000000;
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
// The words of the list in 2048 buckets of equal width over bins first .. last, those of a bucket by their ranks among themselves. Nothing is
// done, and false returned, where a bucket has more than 32 (equal logits).
__device__ __forceinline__ bool smp_buckets(SmpShared& S, int cnt, float top, int first, int last) {
  constexpr int PER = SMP_LIST / SMP_THREADS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float width = (float)SMP_BINS / (float)(last - first + 1);
  unsigned* start = S.hist[2];             // beyond what S.run takes
  u64* spread = S.run;
#pragma unroll
  for (int q = 0; q < PER; q++) start[tid + q * SMP_THREADS] = 0u;
  __syncthreads();
  u64 w[PER];
  int b[PER];
  unsigned slot[PER];
#pragma unroll
  for (int q = 0; q < PER; q++) {
    const int i = tid + q * SMP_THREADS;
    if (i >= cnt) break;
    w[q] = S.list[i];
    const float d = __fmul_rn(__fsub_rn(smp_distance(smp_value(w[q]), top) * 64.f, (float)first), width);   // rises as the word falls
    b[q] = (int)fminf(fmaxf(d, 0.f), (float)(SMP_BINS - 1));
    slot[q] = atomicAdd(&start[b[q]], 1u);
  }
  __syncthreads();
  unsigned c[PER], t = 0, most = 0;
#pragma unroll
  for (int q = 0; q < PER; q++) { const unsigned n = start[PER * tid + q]; c[q] = t; t += n; most = max(most, n); }
  unsigned s = t;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const unsigned a = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += a; }
  if (lane == 31) S.partc[warp] = s;
  if (__syncthreads_or(most > 32)) return false;
#pragma unroll
  for (int q = 0; q < SMP_WARPS; q++) s += q < warp ? S.partc[q] : 0u;
#pragma unroll
  for (int q = 0; q < PER; q++) start[PER * tid + q] = s - t + c[q];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; q++) { if (tid + q * SMP_THREADS >= cnt) break; spread[start[b[q]] + slot[q]] = w[q]; }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; q++) {
    if (tid + q * SMP_THREADS >= cnt) break;
    const unsigned from = start[b[q]], to = b[q] + 1 < SMP_BINS ? start[b[q] + 1] : (unsigned)cnt;
    unsigned at = from;
    for (unsigned j = from; j < to; j++) at += spread[j] > w[q] ? 1u : 0u;
    S.list[at] = w[q];
  }
  return true;
}
// The first cnt words of the list, all of bins first .. last, from the largest down, and their running weights. Up to 128 of them each find
// their own rank; more are spread over buckets (2 us less than the 55 to 66 steps of a bitonic sort, which is left for many equal logits).
__device__ __forceinline__ void smp_sort(SmpShared& S, int cnt, float top, int first, int last) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (cnt <= 128) {
    const u64 mine = tid < cnt ? S.list[tid] : 0ull;
    int at = 0;
    if (warp * 32 < cnt) {
#pragma unroll 4
      for (int j = 0; j < cnt; j++) at += S.list[j] > mine ? 1 : 0;
    }
    __syncthreads();
    if (tid < cnt) S.list[at] = mine;
  } else if (!smp_buckets(S, cnt, top, first, last)) {
    int p2 = 256;
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
#pragma unroll
  for (int q = 0; q < SMP_WARPS; q++) s += q < warp ? S.part[q] : 0ull;
#pragma unroll
  for (int i = 0; i < PER; i++) S.run[PER * tid + i] = s - t + v[i];
  __syncthreads();
}
// The place in S.run[0 .. cnt) (rising) where the running weight reaches target; the last place if it does not. The places of two calls in
// a row stand apart, so that one barrier a call is enough.
__device__ __forceinline__ int smp_place(SmpShared& S, int cnt, u64 target, int which) {
  constexpr int PER = SMP_LIST / SMP_THREADS;
  const u64 to = min(target, S.run[cnt - 1]);
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const int q = PER * (int)threadIdx.x + i;
    if (q < cnt && S.run[q] >= to && (q == 0 || S.run[q - 1] < to)) S.place[which] = q;
  }
  __syncthreads();
  return S.place[which];
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
  // ---- the row's logits / T into shared memory (a greedy row's stay where they are), and the largest
  const int n4 = mine >> 2, n4up = (mine + 3) >> 2;                      // what pads the last four is no candidate
  const bool quick = t >= 0x1p-20f && t <= 0x1p20f;
  const float r = __frcp_rn(t);
  float own = greedy ? -INFINITY : NAN;    // the thread's largest logit (or logit / T; NaN: no candidate)
  int at = 0;                              // greedy: its place, the first of equals (a thread's places rise)
  {
    auto four = [&](float4 v, int i, int step) {
      const float m = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
      if (greedy) {
        if (m > own) { own = m; at = v.x == m ? i : v.y == m ? i + step : v.z == m ? i + 2 * step : i + 3 * step; }
        return v;
      }
      const float4 y = smp_y4(v, t, r, quick);
      own = fmaxf(own, quick ? m : fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
      return y;
    };
    if ((reinterpret_cast<uintptr_t>(x) & 15) == 0 && (per & 3) == 0) {  // i0 is a multiple of per
      constexpr int U = 8;
      for (int b = tid; b < n4; b += U * SMP_THREADS) {
        float4 v[U];
#pragma unroll
        for (int q = 0; q < U; q++) if (b + q * SMP_THREADS < n4) v[q] = __ldcs(reinterpret_cast<const float4*>(x) + b + q * SMP_THREADS);
#pragma unroll
        for (int q = 0; q < U; q++) {
          const int i = b + q * SMP_THREADS;
          if (i >= n4) break;
          const float4 y = four(v[q], 4 * i, 1);
          if (!greedy) *reinterpret_cast<float4*>(s_y + 4 * i) = y;
        }
      }
      if (tid == 0 && n4 < n4up) {
        const int i = 4 * n4, left = mine & 3;
        const float4 v = make_float4(x[i], left > 1 ? x[i + 1] : NAN, left > 2 ? x[i + 2] : NAN, NAN), y = four(v, i, 1);
        if (!greedy) *reinterpret_cast<float4*>(s_y + i) = y;
      }
    } else {
      constexpr int U = 16;
      for (int b = tid; b < 4 * n4up; b += U * SMP_THREADS) {
        float v[U];
#pragma unroll
        for (int q = 0; q < U; q++) v[q] = b + q * SMP_THREADS < mine ? __ldcs(x + b + q * SMP_THREADS) : NAN;
#pragma unroll
        for (int q = 0; q < U; q += 4) {
          const int i = b + q * SMP_THREADS;
          const float4 y = four(make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]), i, SMP_THREADS);
          if (greedy) continue;
          if (i < 4 * n4up) s_y[i] = y.x;
          if (i + SMP_THREADS < 4 * n4up) s_y[i + SMP_THREADS] = y.y;
          if (i + 2 * SMP_THREADS < 4 * n4up) s_y[i + 2 * SMP_THREADS] = y.z;
          if (i + 3 * SMP_THREADS < 4 * n4up) s_y[i + 3 * SMP_THREADS] = y.w;
        }
      }
    }
    if (quick && !greedy) own = smp_y(own, t, false);                     // the order of the quotients is that of the logits
    u64 w = own != own || (greedy && !(own > -INFINITY)) ? 0ull : smp_word(own, i0 + at);
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
  auto clear = [&]() {
    for (int i = tid; i < 3 * SMP_BINS; i += SMP_THREADS) S.hist[0][i] = 0u;
    __syncthreads();
  };
  // ---- counts (and weights) of the bins, and the weight that min-p leaves
  auto bins = [&](bool weights) {
    u64 ms = 0ull;
    auto one = [&](float y) {
      if (y != y) return;
      const int b = smp_bin(y, top);
      atomicAdd(&S.hist[0][b], 1u);
      if (weights) {
        const float f = smp_weight(y, top);
        const unsigned w = smp_units(f);
        if (w) { atomicAdd(&S.hist[1][b], w & 0xffffu); atomicAdd(&S.hist[2][b], w >> 16); }
        if (f >= least) ms += w;
      }
    };
    for (int i = tid; i < n4up; i += SMP_THREADS) {
      const float4 y = *reinterpret_cast<const float4*>(s_y + 4 * i);
      one(y.x); one(y.y); one(y.z); one(y.w);
    }
    if (weights) {
#pragma unroll
      for (int o = 16; o; o >>= 1) ms += __shfl_xor_sync(0xffffffffu, ms, o);
      if (lane == 0 && ms) atomicAdd(&S.least_sum, ms);
    }
    all_sync();
  };
  // Up to 1024 of top-k: the k-th largest of the threads' largest is no larger than the k-th largest of all, so the bins down to its bin
  // hold the k, and (4096 threads) hardly more than those: one entry a thread in place of one a logit. The weights of those
  // candidates are taken when they have been sorted. Fewer threads than k with a candidate: the counts of all.
  int turn = 0;
  SmpScan<NCTA> scan;
  const bool few = k > 0 && k <= SMP_LIST / 2;
  bool part = few;                         // the bins hold the threads' largest alone
  if (few) {
    if (own == own) atomicAdd(&S.hist[0][smp_bin(own, top)], 1u);
    all_sync();
    smp_scan<NCTA>(cluster, S, scan);
    part = scan.count >= (unsigned)k;
    if (!part) clear();
  }
  if (!part) {
    bins(!few);
    smp_scan<NCTA>(cluster, S, scan);
  }
  const bool cut_k = part || (k > 0 && (unsigned)k < scan.count), cut_p = !(tp >= 1.0);
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

  // Words of the logits in bins first .. last whose digits above `himask` are `prefix`: each CTA collects its own where the bins were, and
  // writes them to CTA 0's list from a place that one atomic for all of them gives. More than fit the list: only their number.
  auto gather = [&](int first, int last, u64 himask, u64 prefix) -> unsigned {
    if (tid == 0) S.own = 0u;
    __syncthreads();
    // a distance that rounds to less than (last + 1) / 64 is less than that: all but the bins asked for go by one comparison
    const float from = last >= SMP_BINS - 1 ? -INFINITY : __fsub_rd(top, (float)(last + 1) * 0.015625f);
    auto one = [&](float y, int i) {
      if (!(y >= from)) return;
      const int b = smp_bin(y, top);
      if (b < first || b > last) return;
      const u64 w = smp_word(y, i0 + i);
      if ((w & himask) != prefix) return;
      const unsigned at = atomicAdd(&S.own, 1u);
      if (at < SMP_LIST) S.run[at] = w;
    };
    for (int i = tid; i < n4up; i += SMP_THREADS) {
      const float4 y = *reinterpret_cast<const float4*>(s_y + 4 * i);
      if (!(fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)) >= from)) continue;
      one(y.x, 4 * i); one(y.y, 4 * i + 1); one(y.z, 4 * i + 2); one(y.w, 4 * i + 3);
    }
    __syncthreads();
    const unsigned n = S.own;
    if (tid == 0) S.from = atomicAdd(&other(0)->filled, n);
    __syncthreads();
    const unsigned at = S.from;
    u64* list = other(0)->list;
    if (at + n <= SMP_LIST) for (unsigned i = tid; i < n; i += SMP_THREADS) list[at + i] = S.run[i];
    all_sync();
    const unsigned got = other(0)->filled;
    if (NCTA > 1) cluster.barrier_arrive(); else __syncthreads();         // has read it: see `leave`
    return got;
  };
  auto leave = [&]() { if (NCTA > 1) cluster.barrier_wait(); };         // all CTAs have read the number
  auto finish = [&](u64 word, u64 kept) {
    A.index[row] = smp_index(word);
    if (A.prob) A.prob[row] = (float)((double)smp_weight(smp_value(word), top) * 2147483648.0 / (double)kept);
  };

  if (end.before + end.count <= SMP_LIST) {
    const unsigned got = gather(0, end.bin, 0ull, 0ull);
    if (got <= SMP_LIST) {
      if (rank != 0) { leave(); return; }
      const int cnt = (int)got;
      smp_sort(S, cnt, top, 0, end.bin);
      const u64 wk = cut_k ? S.run[k - 1] : few ? S.run[cnt - 1] : scan.all;
      if (few && least > 0.f) {              // the list's first ones that are heavy enough (or all of it, which is more than is kept)
        int heavy = 0;
        for (int q = tid; q < cnt; q += SMP_THREADS) heavy += smp_weight(smp_value(S.list[q]), top) >= least ? 1 : 0;
        heavy = __reduce_add_sync(0xffffffffu, heavy);
        if (lane == 0) S.partc[tid >> 5] = (unsigned)heavy;
        __syncthreads();
        heavy = 0;
#pragma unroll
        for (int q = 0; q < SMP_WARPS; q++) heavy += (int)S.partc[q];
        wmin = least <= 1.f ? S.run[max(heavy, 1) - 1] : 1ull;
      } else if (few) wmin = least <= 0.f ? S.run[cnt - 1] : 1ull;       // NaN: the first candidate alone
      u64 kept = wk;
      if (cut_p) { const u64 line = smp_target(tp, wk); kept = wmin < line ? wmin : S.run[smp_place(S, cut_k ? k : cnt, line, 0)]; }
      if (wmin < kept) kept = wmin;
      if (!(least <= 1.f)) kept = 1ull << 31;
      const int at = least <= 1.f ? smp_place(S, cnt, smp_target(u, kept), 1) : 0;
      if (tid == 0) finish(S.list[at], kept);
      leave();
      return;
    }
    leave();
    if (rank == 0 && tid == 0) S.filled = 0u;
  }

  // ---- too many to sort together: the three places one after the other
  if (few) {                               // with weights, after all
    all_sync();
    clear();
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
      clear();
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
    const int cnt = (int)gather(bin, bin, himask, prefix);
    leave();
    if (rank == 0) {
      smp_sort(S, cnt, top, bin, bin);
      const int at = by_weight ? smp_place(S, cnt, left, 0) : (int)left - 1;
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
  const u64 word = find(true, least <= 1.f ? smp_target(u, kept) : 1ull, cum);
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
