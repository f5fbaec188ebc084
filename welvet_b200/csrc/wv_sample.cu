// The next token of each of many rows of logits: temperature, top-k, top-p, min-p and a draw (include/welvet_cuda.h,
// wv_sample_rows_dev).
//
// Candidates are ordered by a 64-bit word (ordered bits of logit / T : ~index), all distinct. Every cut is a prefix of that order,
// so each step looks for one word: the k-th largest by count, the last one that top-p keeps and the drawn one by weight. Weights
// are integers in units of 2^-shift, so that no sum depends on its order; each search walks the word's digits from the top with a
// histogram a digit.
#include "wv_common.cuh"
#include <math.h>

#define SMP_THREADS 1024

// exp(d), d <= 0, in units of 2^-shift, rounded to nearest: exp rounds to float32, the rest is integer arithmetic on its bits.
__device__ __forceinline__ unsigned long long smp_fixed(float w, int shift) {
  const unsigned u = __float_as_uint(w);
  const int e = (int)(u >> 23);
  if (e == 0) return 0ull;                                        // below 2^-126
  const unsigned long long m = (u & 0x7fffffu) | 0x800000u;
  const int s = e - 150 + shift;                                  // w = m 2^(e - 150)
  if (s >= 0) return m << s;
  return s < -25 ? 0ull : (m + (1ull << (-s - 1))) >> -s;
}

struct SmpRow {
  const float* x; int n; float t; bool greedy; float top; int shift;
  // logit / T; NaN for what is no candidate. A finite logit may become an infinity by the division: it stays a candidate.
  __device__ __forceinline__ float y(int i) const { const float v = x[i]; return !(v > -INFINITY) ? NAN : greedy ? v : __fdiv_rn(v, t); }
  static __device__ __forceinline__ unsigned long long word(float v, int i) {
    const unsigned u = __float_as_uint(v == 0.f ? 0.f : v);       // -0 and 0 are equal
    const unsigned key = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)key << 32) | (unsigned long long)(0xFFFFFFFFu - (unsigned)i);
  }
  __device__ __forceinline__ float w(float v) const { return v == top ? 1.f : expf(__fsub_rn(v, top)); }
};

// The word where the running total (from the largest word down, over words >= floor) reaches `target`; BY_WEIGHT: of weights
// w >= least, else of counts.
template <bool BY_WEIGHT>
__device__ unsigned long long smp_find(const SmpRow& r, unsigned long long floor_word, float least, unsigned long long target) {
  __shared__ unsigned long long s_hist[256], s_prefix, s_left;
  unsigned long long prefix = 0ull;
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += SMP_THREADS) s_hist[i] = 0ull;
    __syncthreads();
    const unsigned long long himask = shift == 56 ? 0ull : (~0ull << (shift + 8));
    for (int i = threadIdx.x; i < r.n; i += SMP_THREADS) {
      const float v = r.y(i);
      if (v != v) continue;
      const unsigned long long w = SmpRow::word(v, i);
      if (w < floor_word || (w & himask) != prefix) continue;
      if (BY_WEIGHT) {
        const float f = r.w(v);
        if (f >= least) atomicAdd(&s_hist[(w >> shift) & 255u], smp_fixed(f, r.shift));
      } else atomicAdd(&s_hist[(w >> shift) & 255u], 1ull);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long left = target;
      int d = 255, last = -1;
      for (; d >= 0; d--) {
        if (s_hist[d]) last = d;
        if (s_hist[d] >= left && s_hist[d]) break;
        left -= s_hist[d];
      }
      s_prefix = prefix | ((unsigned long long)(d >= 0 ? d : (last >= 0 ? last : 0)) << shift);
      s_left = left;
    }
    __syncthreads();
    prefix = s_prefix; target = s_left;
    __syncthreads();
  }
  return prefix;
}

template <typename T> __device__ T smp_sum(T v) {
  __shared__ T s_part[32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
  __syncthreads();
  T t = 0;
  for (int i = 0; i < SMP_THREADS / 32; i++) t += s_part[i];
  __syncthreads();
  return t;
}
__device__ unsigned long long smp_max(unsigned long long v) {
  __shared__ unsigned long long s_part[32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long t = 0;
  for (int i = 0; i < SMP_THREADS / 32; i++) t = max(t, s_part[i]);
  __syncthreads();
  return t;
}
// The smallest whole number that is at least f * total, between 1 and total.
__device__ __forceinline__ unsigned long long smp_target(double f, unsigned long long total) {
  const double t = ceil(f * (double)total);
  if (!(t > 1.0)) return 1ull;
  return t >= (double)total ? total : (unsigned long long)t;
}

__global__ void __launch_bounds__(SMP_THREADS, 1) sample_rows_kernel(const float* __restrict__ logits, int n, long long ld, const float* __restrict__ temperature,
                                                                     const int* __restrict__ top_k, const float* __restrict__ top_p,
                                                                     const float* __restrict__ min_p, const double* __restrict__ u, int shift,
                                                                     int* __restrict__ index, float* __restrict__ prob) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int row = blockIdx.x;
  SmpRow r;
  r.x = logits + (size_t)row * ld; r.n = n; r.t = temperature[row]; r.shift = shift;
  const int k = top_k[row];
  r.greedy = r.t <= 0.f || k == 1;
  unsigned long long best = 0ull;
  for (int i = threadIdx.x; i < n; i += SMP_THREADS) { const float v = r.y(i); if (v == v) best = max(best, SmpRow::word(v, i)); }
  best = smp_max(best);
  if (best == 0ull || r.greedy) {
    if (threadIdx.x == 0) { index[row] = best ? (int)(0xFFFFFFFFu - (unsigned)best) : -1; if (prob) prob[row] = best ? 1.f : 0.f; }
    return;
  }
  r.top = r.y((int)(0xFFFFFFFFu - (unsigned)best));
  unsigned long long cut = 0ull;
  if (k > 0 && k < n) {
    unsigned long long c = 0;
    for (int i = threadIdx.x; i < n; i += SMP_THREADS) { const float v = r.y(i); c += v == v ? 1 : 0; }
    c = smp_sum(c);
    if (c > (unsigned long long)k) cut = smp_find<false>(r, 0ull, 0.f, (unsigned long long)k);
  }
  auto total = [&](unsigned long long from, float least) {
    unsigned long long t = 0;
    for (int i = threadIdx.x; i < n; i += SMP_THREADS) {
      const float v = r.y(i);
      if (v != v || SmpRow::word(v, i) < from) continue;
      const float f = r.w(v);
      if (f >= least) t += smp_fixed(f, shift);
    }
    return smp_sum(t);
  };
  const unsigned long long all = total(cut, 0.f);
  const double tp = (double)top_p[row];
  if (!(tp >= 1.0)) cut = smp_find<true>(r, cut, 0.f, smp_target(tp, all));
  const float least = min_p[row];
  if (!(least <= 1.f)) cut = best;             // only the first one, whose weight is 1
  const unsigned long long kept = total(cut, fminf(least, 1.f));
  const unsigned long long pick = smp_find<true>(r, cut, fminf(least, 1.f), smp_target(u[row], kept));
  if (threadIdx.x == 0) {
    const int i = (int)(0xFFFFFFFFu - (unsigned)pick);
    index[row] = i;
    if (prob) prob[row] = (float)((double)smp_fixed(r.w(r.y(i)), shift) / (double)kept);
  }
}

int wv_api_bind_device();
extern "C" int wv_sample_rows_dev(const float* d_logits, int rows, int n, int64_t ld, const float* d_temperature, const int* d_top_k,
                                  const float* d_top_p, const float* d_min_p, const double* d_u, int* d_index, float* d_prob, void* stream) {
  const int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if (!d_logits || !d_temperature || !d_top_k || !d_top_p || !d_min_p || !d_u || !d_index) { wv_set_error("wv_sample_rows_dev: null pointer"); return WV_EARG; }
  if (rows < 0 || n < 1) { wv_set_error("wv_sample_rows_dev: %d rows of %d logits", rows, n); return WV_ESHAPE; }
  if (ld == 0) ld = n;
  if (ld < n) { wv_set_error("wv_sample_rows_dev: the row stride %lld is less than %d", (long long)ld, n); return WV_ESHAPE; }
  if (rows == 0) return WV_OK;
  int bits = 0;
  while (bits < 31 && (1ll << bits) < n) bits++;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows); cfg.blockDim = dim3(SMP_THREADS); cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sample_rows_kernel, d_logits, n, (long long)ld, d_temperature, d_top_k, d_top_p, d_min_p, d_u, 62 - bits, d_index, d_prob) != cudaSuccess) {
    wv_set_error("wv_sample_rows_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA;
  }
  return WV_OK;
}
