// Low-rank adapters of many requests beside a shared projection (include/welvet_cuda.h, WvAdapters): y_r = base_r + scale_s B_s (A_s x_r).
//
// A plan sorts the rows by adapter into tiles of 16 (or 64) rows of one adapter. A cluster of eight CTAs takes a tile and a target: each CTA
// multiplies its part of the columns of x with A, the partial sums meet in distributed shared memory, and each CTA then has its part of the
// outputs, so that A and B are read once a tile, t = A x never leaves the SMs and one launch does both products and the addition.
//
// Bound: HBM and latency for few rows (a tile reads all of A_s and B_s, 256 KB at rank 16 of 4096 x 4096, and a row of x has 16 KB), the
// reading of x and y for prompts. The products run on mma.sync m16n8k16: rank 16 gives tiles of 16 x 16, where a tcgen05 tile of 128
// would be mostly padding. x, t and float32 weights are split exactly into three bfloat16 pieces (8 bits each, by truncation), float16 weights
// into two, so the products carry float32's 24 bits; bfloat16 weights are one piece. The tensor core cuts instead of rounding as it
// adds, so a chain is 64 columns of x long at most (24 products) and the chains are added in float32.
//
// In memory a lane's four (or eight) values of the summed index are neighbours; which places of a fragment they take does not matter as long as
// both operands agree.
#include "wv_paged.cuh"
#include <algorithm>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <limits.h>
namespace cg = cooperative_groups;

int wv_api_bind_device();

#define AD_CTAS 8               // of a cluster
#define AD_THREADS 256
#define AD_WARPS 8
#define AD_TARGETS 4
#define AD_RANK 256             // the largest max_rank
#define AD_SLOTS 8192

// A plan: {tiles, rows of a tile, rows, slots}, then a tile's {adapter (slots: none), first place, rows, 0}, then the rows in their places.
static int ad_tile(int rows, int slots) { return rows > 16LL * std::min(rows, slots) ? 64 : 16; }
static long long ad_tiles(int rows, int slots) { return (long long)rows / ad_tile(rows, slots) + std::min(rows, slots + 1); }

__global__ void __launch_bounds__(1024) adapter_plan_kernel(const int* __restrict__ slot, int rows, int slots, int size, int4* __restrict__ plan, int* __restrict__ place, int* err) {
  __shared__ int s_n[AD_SLOTS + 1];
  __shared__ int s_rows[32], s_tiles[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= slots; i += 1024) s_n[i] = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __syncthreads();
  auto at = [&](int r) {
    const int s = slot[r];
    if (s < -1 || s >= slots) wv_paged_report(err, WV_PAGED_ADAPTER);
    return s < 0 || s >= slots ? slots : s;
  };
  for (int r = tid; r < rows; r += 1024) atomicAdd(&s_n[at(r)], 1);
  __syncthreads();
  int row0 = 0, tile0 = 0;
  for (int i0 = 0; i0 <= slots; i0 += 1024) {
    const int i = i0 + tid, n = i <= slots ? s_n[i] : 0, t = (n + size - 1) / size;
    int nr = n, nt = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, nr, o), b = __shfl_up_sync(0xffffffffu, nt, o);
      if (lane >= o) { nr += a; nt += b; }
    }
    if (lane == 31) { s_rows[warp] = nr; s_tiles[warp] = nt; }
    __syncthreads();
    int r = row0 + nr - n, k = tile0 + nt - t;
#pragma unroll
    for (int w = 0; w < 32; w++) {
      if (w < warp) { r += s_rows[w]; k += s_tiles[w]; }
      row0 += s_rows[w]; tile0 += s_tiles[w];
    }
    if (i <= slots) {
      s_n[i] = r;                                        // from now on the next free place of the adapter's rows
      for (int j = 0; j < t; j++) plan[1 + k + j] = make_int4(i, r + j * size, min(size, n - j * size), 0);
    }
    __syncthreads();
  }
  if (tid == 0) plan[0] = make_int4(tile0, size, rows, slots);
  // A row's result does not depend on its place in a tile, so the order that the atomics give does not show.
  for (int r = tid; r < rows; r += 1024) place[atomicAdd(&s_n[at(r)], 1)] = r;
}

struct AdTarget {
  const void *a, *b;
  const int* rank;
  const float* scale;
  const float* base;
  float* y;
  int max_rank, out, ldb, ldy;
};
struct AdCall {
  AdTarget t[AD_TARGETS];
  const float* x;
  const int4* plan;
  const int* place;
  int* err;
  int in, ldx, rows, slots, size;
  long long tiles;
};

__device__ __forceinline__ void ad_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// a and b as three pairs of bfloat16 whose sums they are: the upper 8, the next 8 and the last 8 bits.
__device__ __forceinline__ void ad_split(float a, float b, unsigned& p0, unsigned& p1, unsigned& p2) {
  const unsigned ua = __float_as_uint(a), ub = __float_as_uint(b);
  p0 = __byte_perm(ua, ub, 0x7632);
  const float a1 = a - __uint_as_float(ua & 0xffff0000u), b1 = b - __uint_as_float(ub & 0xffff0000u);
  const unsigned va = __float_as_uint(a1), vb = __float_as_uint(b1);
  p1 = __byte_perm(va, vb, 0x7632);
  p2 = __byte_perm(__float_as_uint(a1 - __uint_as_float(va & 0xffff0000u)), __float_as_uint(b1 - __uint_as_float(vb & 0xffff0000u)), 0x7632);
}
// Weights: four neighbouring values of the summed index are a fragment's two words. DT: 1 float32, 2 float16, 3 bfloat16.
template <int DT> struct AdW {
  static constexpr int PIECES = DT == 1 ? 3 : DT == 2 ? 2 : 1;
  static constexpr int WORDS = DT == 1 ? 4 : 2;          // of four values
  static constexpr int SIZE = DT == 1 ? 4 : 2;
  __device__ static __forceinline__ void pieces(const unsigned* w, unsigned (&p)[PIECES][2]) {
    if constexpr (DT == 3) { p[0][0] = w[0]; p[0][1] = w[1]; }
    if constexpr (DT == 2) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        unsigned none;
        ad_split(f.x, f.y, p[0][i], p[PIECES - 1][i], none);
      }
    }
    if constexpr (DT == 1) {
#pragma unroll
      for (int i = 0; i < 2; i++) ad_split(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]), p[0][i], p[PIECES > 1 ? 1 : 0][i], p[PIECES - 1][i]);
    }
  }
  // x (three pieces) times w, the small products first; what is left out is below 2^-24 of the whole
  __device__ static __forceinline__ void mma(float (&d)[4], const unsigned (&x)[3][4], const unsigned (&w)[PIECES][2]) {
#pragma unroll
    for (int s = 2; s >= 0; s--)
#pragma unroll
      for (int i = s; i >= 0; i--)
        if (s - i < PIECES) ad_mma(d, x[i], w[s - i][0], w[s - i][1]);
  }
};
template <int N> __device__ __forceinline__ void ad_load(unsigned (&w)[N], const void* p, bool on) {      // 8, 16 or 32 bytes
  if constexpr (N == 2) { const uint2 v = on ? *static_cast<const uint2*>(p) : make_uint2(0u, 0u); w[0] = v.x; w[1] = v.y; }
  else {
#pragma unroll
    for (int i = 0; i < N / 4; i++) {
      const uint4 v = on ? static_cast<const uint4*>(p)[i] : make_uint4(0u, 0u, 0u, 0u);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
}

// Shared memory: partial sums of a pass [warps of the columns][MT][8 NT] (later t's fragments [16 ranks][MT / 16][piece][lane]), then t [MT][ranks].
__host__ __device__ constexpr size_t ad_part(int nt) { return (size_t)AD_WARPS * 16 * 8 * nt * 4; }
__host__ __device__ constexpr size_t ad_front(int mt, int nt, int ranks) {
  const size_t frag = (size_t)((ranks + 15) / 16) * (mt / 16) * 3 * 512;
  return ad_part(nt) > frag ? ad_part(nt) : frag;
}
// MT: rows of a tile; NT: tiles of 8 ranks of a pass over x.
template <int DT, int MT, int NT>
__global__ void __launch_bounds__(AD_THREADS, NT == 8 ? 2 : 3) __cluster_dims__(AD_CTAS, 1, 1) adapter_kernel(const __grid_constant__ AdCall c) {
  using W = AdW<DT>;
  constexpr int WM = MT / 16, WK = AD_WARPS / WM, RP = 8 * NT;
  extern __shared__ __align__(16) unsigned char ad_smem[];
  __shared__ int s_row[MT];
  cg::cluster_group cluster = cg::this_cluster();
  const AdTarget& T = c.t[blockIdx.y];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3, rank_ = (int)cluster.block_rank();
  const long long tile = blockIdx.x / AD_CTAS;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int4 head = c.plan[0];
  if (head.y != c.size || head.z != c.rows || head.w != c.slots || head.x > c.tiles) { if (tid == 0) wv_paged_report(c.err, WV_PAGED_ADAPTER); return; }
  if (tile >= head.x) return;
  const int4 me = c.plan[1 + tile];
  const int slot = me.x, count = me.z;
  if (tid < MT) s_row[tid] = tid < count ? c.place[me.y + tid] : -1;
  if (slot == c.slots) {                                 // rows without an adapter
    if (T.base == T.y) return;
    __syncthreads();
    for (int r = 0; r < count; r++) {
      const float* from = T.base + (size_t)s_row[r] * T.ldb;
      float* to = T.y + (size_t)s_row[r] * T.ldy;
      for (int i = rank_ * AD_THREADS + tid; i < T.out; i += AD_CTAS * AD_THREADS) to[i] = from[i];
    }
    return;
  }
  int rank = T.rank ? T.rank[slot] : T.max_rank;
  const float scale = T.scale ? T.scale[slot] : 1.f;
  if (rank < 0 || rank > T.max_rank) { if (tid == 0) wv_paged_report(c.err, WV_PAGED_ADAPTER); rank = min(max(rank, 0), T.max_rank); }
  float* part = reinterpret_cast<float*>(ad_smem);
  float* t = reinterpret_cast<float*>(ad_smem + ad_front(MT, NT, T.max_rank));
  const int ranks = (rank + 15) & ~15;                   // t's columns
  __syncthreads();

  // ---------------------------------------------------------------- t = A x: this CTA's columns, a warp every eighth (or second) 64 of them
  {
    const int m = warp % WM, wk = warp / WM;
    const int r0 = s_row[16 * m + g], r1 = s_row[16 * m + g + 8];
    const float *x0 = c.x + (size_t)max(r0, 0) * c.ldx + 8 * q, *x1 = c.x + (size_t)max(r1, 0) * c.ldx + 8 * q;
    const unsigned char* a = static_cast<const unsigned char*>(T.a) + ((size_t)slot * T.max_rank * c.in + 8 * q) * W::SIZE;
    const bool idle = 16 * m >= count;
    for (int j0 = 0; j0 < rank; j0 += RP) {
      float sum[NT][4];
#pragma unroll
      for (int n = 0; n < NT; n++) sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
#pragma unroll 1
      for (int k0 = 64 * (rank_ * WK + wk); k0 < c.in && !idle; k0 += 64 * WK * AD_CTAS) {
        unsigned w[NT][2][2 * W::WORDS];
        float4 xv[2][2][2];                              // [half][row][4 values]
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int k = k0 + 32 * h;
          const bool on = k + 8 * q < c.in;
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
            xv[h][0][e] = on && r0 >= 0 ? *reinterpret_cast<const float4*>(x0 + k + 4 * e) : z;
            xv[h][1][e] = on && r1 >= 0 ? *reinterpret_cast<const float4*>(x1 + k + 4 * e) : z;
          }
#pragma unroll
          for (int n = 0; n < NT; n++) ad_load(w[n][h], a + ((size_t)(j0 + 8 * n + g) * c.in + k) * W::SIZE, on && j0 + 8 * n + g < rank);
        }
        float d[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            unsigned p[3][4];
            const float4 u = xv[h][0][e], v = xv[h][1][e];
            ad_split(u.x, u.y, p[0][0], p[1][0], p[2][0]); ad_split(v.x, v.y, p[0][1], p[1][1], p[2][1]);
            ad_split(u.z, u.w, p[0][2], p[1][2], p[2][2]); ad_split(v.z, v.w, p[0][3], p[1][3], p[2][3]);
#pragma unroll
            for (int n = 0; n < NT; n++) {
              if (NT > 2 && j0 + 8 * n >= rank) break;
              unsigned wp[W::PIECES][2];
              W::pieces(&w[n][h][e * W::WORDS], wp);
              W::mma(d[n], p, wp);
            }
          }
#pragma unroll
        for (int n = 0; n < NT; n++) { sum[n][0] += d[n][0]; sum[n][1] += d[n][1]; sum[n][2] += d[n][2]; sum[n][3] += d[n][3]; }
      }
      __syncthreads();                                   // the sums of the pass before have been read
      float* to = part + (size_t)(wk * MT + 16 * m) * RP + 2 * q;
#pragma unroll
      for (int n = 0; n < NT; n++) {
        *reinterpret_cast<float2*>(to + g * RP + 8 * n) = make_float2(sum[n][0], sum[n][1]);
        *reinterpret_cast<float2*>(to + (g + 8) * RP + 8 * n) = make_float2(sum[n][2], sum[n][3]);
      }
      __syncthreads();
      for (int i = tid; i < MT * RP; i += AD_THREADS) {
        const int j = j0 + i % RP;
        if (j >= ranks) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WK; w++) v += part[w * MT * RP + i];
        t[i / RP * ranks + j] = v;
      }
    }
  }
  cluster.sync();

  // ---------------------------------------------------------------- the CTAs' sums of t, scaled, as fragments
  uint4* frag = reinterpret_cast<uint4*>(ad_smem);
  const int nk = ranks / 16;
  for (int i = tid; i < nk * WM * 32; i += AD_THREADS) { // a lane of a fragment: two rows of four neighbouring ranks
    const int l = i & 31, m = i / 32 % WM, k = i / 32 / WM, row = 16 * m + (l >> 2), j = 16 * k + 4 * (l & 3);
    float4 u = make_float4(0.f, 0.f, 0.f, 0.f), v = u;
#pragma unroll
    for (int r = 0; r < AD_CTAS; r++) {
      const float* o = cluster.map_shared_rank(t, r);
      const float4 a = *reinterpret_cast<const float4*>(o + row * ranks + j), b = *reinterpret_cast<const float4*>(o + (row + 8) * ranks + j);
      u.x += a.x; u.y += a.y; u.z += a.z; u.w += a.w;
      v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
    }
    unsigned p[3][4];
    ad_split(u.x * scale, u.y * scale, p[0][0], p[1][0], p[2][0]); ad_split(v.x * scale, v.y * scale, p[0][1], p[1][1], p[2][1]);
    ad_split(u.z * scale, u.w * scale, p[0][2], p[1][2], p[2][2]); ad_split(v.z * scale, v.w * scale, p[0][3], p[1][3], p[2][3]);
#pragma unroll
    for (int s = 0; s < 3; s++) frag[((k * WM + m) * 3 + s) * 32 + l] = make_uint4(p[s][0], p[s][1], p[s][2], p[s][3]);
  }
  cluster.barrier_arrive();                              // this CTA has read the others' sums
  __syncthreads();

  // ---------------------------------------------------------------- y = base + B t: 16 outputs a warp at a time
  const unsigned char* b = static_cast<const unsigned char*>(T.b) + ((size_t)slot * T.out * T.max_rank + 4 * q) * W::SIZE;
  for (int n0 = 16 * (rank_ * AD_WARPS + warp); n0 < T.out; n0 += 16 * AD_CTAS * AD_WARPS) {
    float d[WM][2][4];
#pragma unroll
    for (int m = 0; m < WM; m++)
#pragma unroll
      for (int n = 0; n < 2; n++) d[m][n][0] = d[m][n][1] = d[m][n][2] = d[m][n][3] = 0.f;
    for (int k0 = 0; k0 < nk; k0 += 4) {
      unsigned w[4][2][W::WORDS];
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const int o = n0 + 8 * n + g, j = 16 * (k0 + k) + 4 * q;
          ad_load(w[k][n], b + ((size_t)o * T.max_rank + 16 * (k0 + k)) * W::SIZE, o < T.out && j < rank);
          if (j < rank && j + 4 > rank) {                // what stands behind the adapter's rank does not count
            const int have = rank - j;
#pragma unroll
            for (int i = 0; i < W::WORDS; i++) {
              if (DT == 1) { if (i >= have) w[k][n][i] = 0u; }
              else if (2 * i >= have) w[k][n][i] = 0u;
              else if (2 * i + 1 >= have) w[k][n][i] &= 0xffffu;
            }
          }
        }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (k0 + k >= nk) break;
        unsigned wp[2][W::PIECES][2];
#pragma unroll
        for (int n = 0; n < 2; n++) W::pieces(w[k][n], wp[n]);
#pragma unroll
        for (int m = 0; m < WM; m++) {
          if (WM > 1 && 16 * m >= count) break;
          unsigned p[3][4];
#pragma unroll
          for (int s = 0; s < 3; s++) {
            const uint4 v = frag[(((k0 + k) * WM + m) * 3 + s) * 32 + lane];
            p[s][0] = v.x; p[s][1] = v.y; p[s][2] = v.z; p[s][3] = v.w;
          }
#pragma unroll
          for (int n = 0; n < 2; n++) W::mma(d[m][n], p, wp[n]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < WM; m++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = s_row[16 * m + g + 8 * h];
        if (row < 0) continue;
#pragma unroll
        for (int n = 0; n < 2; n++) {
          const int o = n0 + 8 * n + 2 * q;
          const float* from = T.base + (size_t)row * T.ldb + o;
          float* to = T.y + (size_t)row * T.ldy + o;
          if (o + 1 < T.out) {
            const float2 v = *reinterpret_cast<const float2*>(from);
            *reinterpret_cast<float2*>(to) = make_float2(v.x + d[m][n][2 * h], v.y + d[m][n][2 * h + 1]);
          } else if (o < T.out) {
            *to = *from + d[m][n][2 * h];
          }
        }
      }
  }
  cluster.barrier_wait();                                // nobody leaves while another reads its sums
}

// ------------------------------------------------------------------ host
template <int DT, int MT, int NT> static cudaError_t ad_go(const AdCall& c, int n, int ranks, cudaStream_t st) {
  auto kern = adapter_kernel<DT, MT, NT>;
  const size_t smem = ad_front(MT, NT, ranks) + (size_t)MT * ((ranks + 15) & ~15) * 4;
  static unsigned long long attr_mask = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !(attr_mask & (1ull << dev))) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(ad_front(MT, NT, AD_RANK) + (size_t)MT * AD_RANK * 4));
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_mask |= 1ull << dev;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  cfg.gridDim = dim3((unsigned)(c.tiles * AD_CTAS), (unsigned)n); cfg.blockDim = dim3(AD_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, c);
}
template <int DT, int MT> static cudaError_t ad_pick(const AdCall& c, int n, int ranks, cudaStream_t st) {
  return ranks <= 16 ? ad_go<DT, MT, 2>(c, n, ranks, st) : ranks <= 32 ? ad_go<DT, MT, 4>(c, n, ranks, st) : ad_go<DT, MT, 8>(c, n, ranks, st);
}
template <int DT> static cudaError_t ad_any(const AdCall& c, int n, int ranks, cudaStream_t st) {
  return c.size == 64 ? ad_pick<DT, 64>(c, n, ranks, st) : ad_pick<DT, 16>(c, n, ranks, st);
}
static int ad_counts(const char* who, int rows, int slots) {
  if (rows < 0 || rows > 1 << 24 || slots < 1 || slots > AD_SLOTS) { wv_set_error("%s: %d rows, %d adapters (1 to %d)", who, rows, slots, AD_SLOTS); return WV_ESHAPE; }
  return WV_OK;
}

extern "C" int wv_adapter_plan_bytes(int rows, int slots, uint64_t* bytes) {
  const char* who = "wv_adapter_plan_bytes";
  if (!bytes) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  if (const int rc = ad_counts(who, rows, slots)) return rc;
  *bytes = 16 + 16 * (uint64_t)ad_tiles(rows, slots) + 4 * (((uint64_t)rows + 3) & ~3ull);
  return WV_OK;
}

extern "C" int wv_adapter_plan_dev(const int* d_slot, int rows, int slots, void* d_plan, void* stream) {
  const char* who = "wv_adapter_plan_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = ad_counts(who, rows, slots))) return rc;
  if (!d_plan || (!d_slot && rows > 0)) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  if (reinterpret_cast<uintptr_t>(d_plan) & 15) { wv_set_error("%s: the plan is not 16-byte aligned", who); return WV_EARG; }
  if (rows == 0) return WV_OK;
  int4* plan = static_cast<int4*>(d_plan);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  cfg.gridDim = dim3(1); cfg.blockDim = dim3(1024); cfg.stream = static_cast<cudaStream_t>(stream);
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, adapter_plan_kernel, d_slot, rows, slots, ad_tile(rows, slots), plan, reinterpret_cast<int*>(plan + 1 + ad_tiles(rows, slots)), wv_paged_err_ptr());
  if (e != cudaSuccess) { cudaGetLastError(); wv_set_error("%s: launch: %s", who, cudaGetErrorString(e)); return WV_ECUDA; }
  return WV_OK;
}

extern "C" int wv_adapter_apply_dev(const WvAdapters* targets, int n, const void* d_plan, int rows, const float* dx, int ldx, const float* const* dbase, const int* ldb,
                                    float* const* dy, const int* ldy, void* stream) {
  const char* who = "wv_adapter_apply_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if (!targets || !dy || !d_plan || !dx) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  if (n < 1 || n > AD_TARGETS) { wv_set_error("%s: %d targets (1 to %d)", who, n, AD_TARGETS); return WV_EARG; }
  const WvAdapters& f = targets[0];
  if ((rc = ad_counts(who, rows, f.slots))) return rc;
  if (f.dtype < 1 || f.dtype > 3) { wv_set_error("%s: dtype %d (1 float32, 2 float16, 3 bfloat16)", who, f.dtype); return WV_EFORMAT; }
  if (f.in < 8 || f.in % 8) { wv_set_error("%s: %d columns (a multiple of 8)", who, f.in); return WV_ESHAPE; }
  if (ldx == 0) ldx = f.in;
  if (ldx < f.in || (ldx & 3)) { wv_set_error("%s: the row stride of x is %d for %d values (a multiple of 4)", who, ldx, f.in); return WV_ESHAPE; }
  if ((reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(d_plan)) & 15) { wv_set_error("%s: x or the plan is not 16-byte aligned", who); return WV_EARG; }
  AdCall c = {};
  int ranks = 0;
  for (int i = 0; i < n; i++) {
    const WvAdapters& w = targets[i];
    AdTarget& t = c.t[i];
    if (!w.a || !w.b || !dy[i]) { wv_set_error("%s: target %d: null pointer", who, i); return WV_EARG; }
    if (w.slots != f.slots || w.in != f.in || w.dtype != f.dtype) { wv_set_error("%s: target %d has other adapters, columns or another type than the first", who, i); return WV_ESHAPE; }
    if (w.max_rank < 8 || w.max_rank % 8 || w.max_rank > AD_RANK || w.out < 1) {
      wv_set_error("%s: target %d: %d outputs, rank %d (a multiple of 8, at most %d)", who, i, w.out, w.max_rank, AD_RANK); return WV_ESHAPE;
    }
    t.a = w.a; t.b = w.b; t.rank = w.rank; t.scale = w.scale; t.max_rank = w.max_rank; t.out = w.out;
    t.y = dy[i]; t.base = dbase ? dbase[i] : dy[i];
    if (!t.base) { wv_set_error("%s: target %d: null pointer", who, i); return WV_EARG; }
    t.ldy = ldy && ldy[i] ? ldy[i] : w.out;
    t.ldb = dbase ? (ldb && ldb[i] ? ldb[i] : w.out) : t.ldy;
    if (t.ldy < w.out || t.ldb < w.out || ((t.ldy | t.ldb) & 3)) {
      wv_set_error("%s: target %d: row strides %d and %d for %d outputs (multiples of 4)", who, i, t.ldb, t.ldy, w.out); return WV_ESHAPE;
    }
    if (t.base == t.y && t.ldb != t.ldy) { wv_set_error("%s: target %d in place with two strides", who, i); return WV_EARG; }
    if ((reinterpret_cast<uintptr_t>(w.a) | reinterpret_cast<uintptr_t>(w.b) | reinterpret_cast<uintptr_t>(t.y) | reinterpret_cast<uintptr_t>(t.base)) & 15) {
      wv_set_error("%s: target %d: a pointer is not 16-byte aligned", who, i); return WV_EARG;
    }
    ranks = std::max(ranks, w.max_rank);
  }
  if (rows == 0) return WV_OK;
  c.x = dx; c.ldx = ldx; c.in = f.in; c.rows = rows; c.slots = f.slots;
  c.size = ad_tile(rows, f.slots); c.tiles = ad_tiles(rows, f.slots);
  c.plan = static_cast<const int4*>(d_plan);
  c.place = reinterpret_cast<const int*>(c.plan + 1 + c.tiles);
  c.err = wv_paged_err_ptr();
  if (c.tiles * AD_CTAS > INT_MAX) { wv_set_error("%s: %d rows are too many", who, rows); return WV_ESHAPE; }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = f.dtype == 1 ? ad_any<1>(c, n, ranks, st) : f.dtype == 2 ? ad_any<2>(c, n, ranks, st) : ad_any<3>(c, n, ranks, st);
  if (e != cudaSuccess) { cudaGetLastError(); wv_set_error("%s: launch: %s", who, cudaGetErrorString(e)); return WV_ECUDA; }
  return WV_OK;
}
