// Attention of the new tokens of a batch over the paged cache (include/welvet_cuda.h, wv_attn_paged_dev).
//
// One warp per (new token, query head): the keys one after the other with the running maximum and sum of the softmax, a lane
// holding the values lane, lane + 32, ... of the head.
#include "wv_paged.cuh"
#include <math.h>

template <int BITS>
__device__ __forceinline__ float kv_code(const WvKvGeom& g, const unsigned char* block, bool is_v, int slot, int d) {
  const unsigned char* codes = block + (is_v ? g.page * g.code : 0) + slot * g.code;
  if (BITS == 16) return __half2float(reinterpret_cast<const __half*>(codes)[d]);
  if (BITS == 8) return (float)(int)reinterpret_cast<const signed char*>(codes)[d];
  const int c = (int)((codes[d >> 1] >> (4 * (d & 1))) & 15u) - 8;
  return (float)(c * (int)block[(is_v ? g.vsub : g.ksub) + slot * (g.hd / 16) + d / 16]);
}

template <int BITS>
__global__ void __launch_bounds__(256) attn_paged_kernel(const WvKvGeom g, const WvKvBatch b, const float* __restrict__ q, int ldq,
                                                         float* __restrict__ out, int ldo, int heads, float scale, int window, int* __restrict__ err) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int row = (int)(w / heads), h = (int)(w % heads);
  if (row >= b.total_q) return;
  const int s = wv_seq_of_row(b, row);
  if (s >= b.num_seqs) return;
  const WvSeq sq = wv_seq(b, g.page, s, err);
  if (row < sq.q0 || row >= sq.q1) return;
  const int p = sq.kv - (sq.q1 - sq.q0) + (row - sq.q0);
  const int kvh = h / (heads / g.kvh);
  float qv[8], acc[8], m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int d = lane + 32 * i;
    qv[i] = d < g.hd ? q[(size_t)row * ldq + (size_t)h * g.hd + d] : 0.f;
    acc[i] = 0.f;
  }
  for (int j = window > 0 ? max(0, p - window + 1) : 0; j <= p; j++) {
    const int id = b.pages[(size_t)s * b.table_stride + j / g.page], slot = j % g.page;
    if (id < 0 || id >= g.num_pages) { wv_paged_report(err, WV_PAGED_PAGE); continue; }
    const unsigned char* block = g.pool + ((size_t)id * g.kvh + kvh) * g.block;
    float d_ = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) if (lane + 32 * i < g.hd) d_ += qv[i] * kv_code<BITS>(g, block, false, slot, lane + 32 * i);
#pragma unroll
    for (int o = 16; o; o >>= 1) d_ += __shfl_xor_sync(0xffffffffu, d_, o);
    const float x = d_ * *reinterpret_cast<const float*>(block + g.kscale + 4 * slot) * scale;
    const float mn = fmaxf(m, x), f = sum == 0.f ? 0.f : expf(m - mn), e = expf(x - mn);
    const float ev = e * *reinterpret_cast<const float*>(block + g.vscale + 4 * slot);
    sum = sum * f + e;
#pragma unroll
    for (int i = 0; i < 8; i++) if (lane + 32 * i < g.hd) acc[i] = acc[i] * f + ev * kv_code<BITS>(g, block, true, slot, lane + 32 * i);
    m = mn;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int d = lane + 32 * i;
    if (d < g.hd) out[(size_t)row * ldo + (size_t)h * g.hd + d] = sum == 0.f ? 0.f : acc[i] / sum;
  }
}

int wv_launch_attn_paged(const WvKvPages& kv, const WvKvBatch& b, const float* dq, int ldq, float* dout, int ldo, int heads, float scale,
                         int window, cudaStream_t st) {
  const WvKvGeom g = wv_kv_geom(kv);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  const long long warps = (long long)b.total_q * heads;
  cfg.gridDim = dim3((unsigned)((warps + 7) / 8)); cfg.blockDim = dim3(256); cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  auto go = [&](auto kern) { return cudaLaunchKernelEx(&cfg, kern, g, b, dq, ldq, dout, ldo, heads, scale, window, wv_paged_err_ptr()); };
  const cudaError_t e = kv.bits == 16 ? go(attn_paged_kernel<16>) : kv.bits == 8 ? go(attn_paged_kernel<8>) : go(attn_paged_kernel<4>);
  if (e != cudaSuccess) { wv_set_error("wv_attn_paged_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA; }
  return WV_OK;
}
