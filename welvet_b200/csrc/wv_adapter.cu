// Low-rank adapters of many requests beside a shared projection (include/welvet_cuda.h, WvAdapters): y_r = base_r + scale_s B_s (A_s x_r).
//
// A plan sorts the rows by adapter into tiles of 8 (or 32) rows of one adapter. A cluster of CTAs takes a tile and a target: each CTA
// multiplies its part of the columns of x with A, the partial sums meet in distributed shared memory, and each CTA then has its part of the
// outputs, so that A and B are read once a tile, t = A x never leaves the SMs and one launch does both products and the addition.
//
// Bound: HBM and latency for few rows (a tile reads all of A_s and B_s, 256 KB at rank 16 of 4096 x 4096, and a row of x has 16 KB), the
// reading of x and y for prompts. A warp works alone: 16 columns of A and x, or 16 or 32 outputs' rows of B and their values of base, at a time through a
// ring of its own (cp.async, no barrier but its own), and the first outputs' copies are under way while t is being added up. The products run on mma.sync m16n8k16 with
// the weights as the side of 16 and the rows of x as the side of 8: of a step of decoding an adapter has a row or two, and a tcgen05 tile of 128 would be nearly
// all padding.
//
// With 16-bit weights x and t go through as three pieces of the weights' type: of bfloat16 (8 bits each by truncation, exactly x), or of float16, behind a
// power of two for each row: the third piece ends 2^-32 below the row's largest value so far, so a value 2^-8 of that keeps 24 bits and one 2^-16 of it 16. (float16 weights
// as two bfloat16 pieces would keep them all, for five products in place of three.) Float32 weights are split into three bfloat16 pieces themselves, and the
// six products that matter are taken. These products carry float32's 24 bits. The tensor core cuts instead of rounding as it adds, so chains of products are
// short: what a warp has of the columns (3 in 128 of a CTA's: 42 at most up to 28672 columns, and 3 in 2048 of wider matrices), or 24 products where registers allow
// a second sum.
//
// 16-bit weights come out of shared memory by ldmatrix, which puts a fragment's words where the product wants them (put together from
// vector loads they took a move each).
//
// Measured, plan and targets, us from a graph (floor): a row, rank 16 of 4096 beside 4096 + 1024 + 1024 in bf16 7.2 (0.1); 64 rows of 32 such adapters 17 (3.4); 48
// rows of 16, rank 64 of 4096 beside 2 x 14336 in f16 36 (13); 2048 rows of 6, rank 64 of 4096 beside 4096 in bf16 53 (16); 333 rows of 9, rank 24 of 14336
// beside 4096 in f32 50 (7). Ranks beyond 64 go in pieces; with rank 128 the first
// takes 13 (0.4), the second 65 (13), the third 75 (22), the fourth 98 (17). The plan is 2 of them, 4 for 2048 rows. What bounds the rest is a cluster's chain: its ring
// fills, t is made, added up and spread, and only then do the outputs run; clusters of up to 16 CTAs shorten both parts (with 8 at most the last one took 54), and are kept from running in turns by the rule below.
#include "wv_paged.cuh"
#include "wv_tma_common.cuh"      // lds64, smem_u32
#include <algorithm>
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <type_traits>
#include <limits.h>
namespace cg = cooperative_groups;

int wv_api_bind_device();
int wv_sm_count();

#define AD_WARPS 8
#define AD_THREADS (32 * AD_WARPS)
#define AD_CTAS 16              // of a cluster at most
#define AD_TARGETS 4
#define AD_RANK 256             // the largest max_rank
#define AD_SLOTS 8192
#define AD_WIDE (1 << 30)       // columns and outputs: a CTA's offsets, in bytes of at most half the columns, and the units' ends stay in 32 bits

// A plan: {tiles, rows of a tile, rows, slots}, then a tile's {adapter (slots: none), first place, rows, 0}, then the rows in their places.
// Tiles of 32 where an adapter has more than 8 rows on average.
static int ad_tile(int rows, int slots) { return rows > 8LL * std::min(rows, slots) ? 32 : 8; }
static long long ad_tiles(int rows, int slots) { return (long long)rows / ad_tile(rows, slots) + std::min(rows, slots + 1); }

__global__ void __launch_bounds__(1024) adapter_plan_kernel(const int* __restrict__ slot, int rows, int slots, int size, int4* __restrict__ plan, int* __restrict__ place, int* err) {
  __shared__ int s_n[AD_SLOTS + 1];
  __shared__ int2 s_sum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= slots; i += 1024) s_n[i] = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  auto at = [&](int r) {
    const int s = slot[r];
    if (s < -1 || s >= slots) wv_paged_report(err, WV_PAGED_ADAPTER);
    return s < 0 || s >= slots ? slots : s;
  };
  const int mine = tid < rows ? at(tid) : 0;             // a thread's first row
  __syncthreads();
  const int nth = tid < rows ? atomicAdd(&s_n[mine], 1) : 0;
  for (int r = tid + 1024; r < rows; r += 1024) atomicAdd(&s_n[at(r)], 1);
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
    if (lane == 31) s_sum[warp] = make_int2(nr, nt);
    __syncthreads();
    const int2 v = s_sum[lane];                          // a lane each for the warps before this one
    const int r = row0 + __reduce_add_sync(0xffffffffu, lane < warp ? v.x : 0) + nr - n, k = tile0 + __reduce_add_sync(0xffffffffu, lane < warp ? v.y : 0) + nt - t;
    row0 += __reduce_add_sync(0xffffffffu, v.x);
    tile0 += __reduce_add_sync(0xffffffffu, v.y);
    if (i <= slots) {
      s_n[i] = r;                                        // from now on the first place of the adapter's rows
      for (int j = 0; j < t; j++) plan[1 + k + j] = make_int4(i, r + j * size, min(size, n - j * size), 0);
    }
    __syncthreads();
  }
  if (tid == 0) plan[0] = make_int4(tile0, size, rows, slots);
  // A row's result does not depend on its place in a tile, so the order that the atomics give does not show.
  if (rows <= 1024) {
    if (tid < rows) place[s_n[mine] + nth] = tid;
  } else {
    for (int r = tid; r < rows; r += 1024) place[atomicAdd(&s_n[at(r)], 1)] = r;
  }
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
  int slab;                       // bytes of a warp's ring
  long long tiles;
};

// 16 bytes of which the first `bytes` exist (0 to 16); the others become zeros
__device__ __forceinline__ void ad_copy(unsigned dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Not volatile: the compiler may put independent ones between those that wait for one another. ZERO: the sum begins here.
template <bool HALF, bool ZERO> __device__ __forceinline__ void ad_mma(float (&d)[4], const unsigned (&a)[4], const unsigned (&b)[2]) {
  if constexpr (ZERO && HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
  else if constexpr (ZERO)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
  else if constexpr (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
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
// The same in float16, for values up to 2^15.
__device__ __forceinline__ void ad_split16(float a, float b, unsigned& p0, unsigned& p1, unsigned& p2) {
  unsigned* p[3] = {&p0, &p1, &p2};
#pragma unroll
  for (int i = 0; i < 3; i++) {
    const __half2 h = __floats2half2_rn(a, b);
    *p[i] = *reinterpret_cast<const unsigned*>(&h);
    const float2 f = __half22float2(h);
    a -= f.x; b -= f.y;
  }
}
// A power of two that brings values of up to m (as bits; an infinity or NaN stays one) below 2^8: they may grow by 2^7 before it has to change.
__device__ __forceinline__ float ad_up(unsigned m, float& down) {
  const unsigned k = min(max(m >> 23, 8u), 254u);
  down = __uint_as_float((k - 7u) << 23);
  return __uint_as_float((261u - k) << 23);
}
__device__ __forceinline__ void ad_ldmatrix(unsigned (&r)[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
// Weights (DT: 1 float32, 2 float16, 3 bfloat16) as a product's side of 16. A lane's places of the summed index are 2 q, 2 q + 1 and those 8 further on.
template <int DT> struct AdW {
  static constexpr int PIECES = DT == 1 ? 3 : 1, SIZE = DT == 1 ? 4 : 2;
  // where a lane reads in rows of `pitch` bytes
  __device__ static __forceinline__ unsigned place(int pitch) {
    const int lane = threadIdx.x & 31;
    return DT == 1 ? (lane >> 2) * pitch + 8 * (lane & 3) : (lane & 15) * pitch + 16 * (lane >> 4);
  }
  // 16 rows of 16 values, `at` with place(pitch) in it. CUT: places from `left` on are zeros.
  template <bool CUT> __device__ static __forceinline__ void load(unsigned (&p)[PIECES][4], unsigned at, int pitch, int left) {
    const int q = threadIdx.x & 3;
    if constexpr (DT == 1) {
#pragma unroll
      for (int r = 0; r < 2; r++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          uint2 v = lds64(at + 8 * r * pitch + 32 * i);
          if constexpr (CUT) {
            if (2 * q + 8 * i >= left) v.x = 0u;
            if (2 * q + 8 * i + 1 >= left) v.y = 0u;
          }
          const int o = r + 2 * i;
          ad_split(__uint_as_float(v.x), __uint_as_float(v.y), p[0][o], p[PIECES > 1 ? 1 : 0][o], p[PIECES - 1][o]);
        }
    } else {
      ad_ldmatrix(p[0], at);
      if constexpr (CUT) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int have = left - 2 * q - 8 * i;
          const unsigned mask = have >= 2 ? ~0u : have == 1 ? 0xffffu : 0u;
          p[0][2 * i] &= mask; p[0][2 * i + 1] &= mask;
        }
      }
    }
  }
  // x's pieces: places 2 q, 2 q + 1, 2 q + 8, 2 q + 9
  __device__ static __forceinline__ void values(const float4& v, unsigned (&p)[3][2]) {
    if constexpr (DT == 2) { ad_split16(v.x, v.y, p[0][0], p[1][0], p[2][0]); ad_split16(v.z, v.w, p[0][1], p[1][1], p[2][1]); }
    else { ad_split(v.x, v.y, p[0][0], p[1][0], p[2][0]); ad_split(v.z, v.w, p[0][1], p[1][1], p[2][1]); }
  }
  // piece J of the weights times piece I of x; what is left out is below 2^-24 of the whole
  template <int I, int J, bool ZERO> __device__ static __forceinline__ void mma(float (&d)[4], const unsigned (&w)[PIECES][4], const unsigned (&x)[3][2]) {
    if constexpr (J < PIECES) ad_mma<DT == 2, ZERO>(d, w[J < PIECES ? J : 0], x[I]);
  }
};
__device__ __forceinline__ float4 ad_four(const float* p, int q) {      // places 2 q, 2 q + 1, 2 q + 8, 2 q + 9
  const float2 a = *reinterpret_cast<const float2*>(p + 2 * q), b = *reinterpret_cast<const float2*>(p + 2 * q + 8);
  return make_float4(a.x, a.y, b.x, b.y);
}

// NR: rows of a tile, in NB blocks of 8; MR: tiles of 16 ranks of a pass over x, and of a piece of B.
template <int DT, int NR, int MR> struct AdShape {
  using W = AdW<DT>;
  static constexpr int NB = NR / 8, RP = 16 * MR;
  static constexpr bool WIDE = DT == 1 && MR == 4;                       // one CTA an SM, and its registers
  static constexpr bool SUMS = WIDE || MR * NB < 16;                     // room for a second set of sums
  static constexpr int Z = NB == 1 && DT != 1 ? 2 : 1;                   // a unit is 16 Z outputs
  // a step: 16 columns of A and of x, rows shifted against one another so that reads meet few banks twice
  static constexpr int PA = 16 * W::SIZE + (DT == 1 ? 32 : 16), PX = NB == 1 ? 96 : 64, XO = RP * PA, STEP = XO + NR * PX;
  static constexpr int STEPS = NB == 1 && !WIDE ? 3 : 2;
  // a unit's rows of B (a piece of RP ranks at most), an odd number of 16 bytes from one another, and base
  static constexpr int PB = 16 * Z + 4;                                  // floats
  static __host__ __device__ constexpr int prow(int ranks) { return ((ranks < RP ? ranks : RP) * W::SIZE / 16 | 1) * 16; }
  static __host__ __device__ constexpr int unit(int ranks) { return 16 * Z * prow(ranks) + NR * PB * 4; }
  static __host__ __device__ constexpr int slab(int ranks) { return STEPS * STEP > 2 * unit(ranks) ? STEPS * STEP : 2 * unit(ranks); }
  // the warps' sums of a pass, a few warps at a time
  static constexpr int PP = RP + 4;                                      // floats of a row: rows 2 q of a warp's stores meet no bank twice
  static constexpr int ROUND = NR * RP * 4 * AD_WARPS <= 16384 ? AD_WARPS : 16384 / (NR * RP * 4);
  static constexpr size_t PART = (size_t)ROUND * NR * PP * 4;
  static __host__ __device__ constexpr int row(int ranks) { return (ranks + 15) / 16 * 16 + 4; }      // of t
  static __host__ __device__ constexpr size_t frags(int ranks) { return (size_t)((ranks + 15) / 16) * NB * 3 * 256; }
  // [front: the warps' sums, later the whole t][back: this CTA's t, later t's fragments]
  static __host__ __device__ constexpr size_t front(int ranks) { return PART > (size_t)NR * row(ranks) * 4 ? PART : (size_t)NR * row(ranks) * 4; }
  static __host__ __device__ constexpr size_t back(int ranks) { return frags(ranks) > (size_t)NR * row(ranks) * 4 ? frags(ranks) : (size_t)NR * row(ranks) * 4; }
  static __host__ __device__ constexpr size_t smem(int ranks, int slab_) { return (size_t)AD_WARPS * slab_ + front(ranks) + back(ranks); }
};
template <int N> __device__ __forceinline__ void ad_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ad_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int DT, int NR, int MR>
__global__ void __launch_bounds__(AD_THREADS, AdShape<DT, NR, MR>::WIDE ? 1 : 2) adapter_kernel(const __grid_constant__ AdCall c) {
  using S = AdShape<DT, NR, MR>;
  using W = AdW<DT>;
  constexpr int NB = S::NB, RP = S::RP, Z = S::Z;
  extern __shared__ __align__(128) unsigned char ad_smem[];
  __shared__ int s_row[NR];
  __shared__ float s_down[NR];
  cg::cluster_group cluster = cg::this_cluster();
  const AdTarget& T = c.t[blockIdx.y];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3, ctas = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
  const long long tile = blockIdx.x / ctas;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int4 head = c.plan[0];
  if (head.y != c.size || head.z != c.rows || head.w != c.slots || head.x > c.tiles) { if (tid == 0) wv_paged_report(c.err, WV_PAGED_ADAPTER); return; }
  if (tile >= head.x) return;
  const int4 my = c.plan[1 + tile];
  const int slot = my.x, count = my.z;
  if (tid < NR) s_row[tid] = tid < count ? c.place[my.y + tid] : -1;
  if (slot == c.slots) {                                 // rows without an adapter
    if (T.base == T.y) return;
    __syncthreads();
    for (int r = 0; r < count; r++) {
      const float* from = T.base + (size_t)s_row[r] * T.ldb;
      float* to = T.y + (size_t)s_row[r] * T.ldy;
      for (int i = me * AD_THREADS + tid; i < T.out; i += ctas * AD_THREADS) to[i] = from[i];
    }
    return;
  }
  int rank = T.rank ? T.rank[slot] : T.max_rank;
  const float scale = T.scale ? T.scale[slot] : 1.f;
  if (rank < 0 || rank > T.max_rank) { if (tid == 0) wv_paged_report(c.err, WV_PAGED_ADAPTER); rank = min(max(rank, 0), T.max_rank); }
  const int nk = (rank + 15) / 16, passes = (rank + RP - 1) / RP;
  unsigned char* slab = ad_smem + warp * c.slab;
  unsigned char* front = ad_smem + AD_WARPS * c.slab;
  float* t = reinterpret_cast<float*>(front + S::front(T.max_rank));      // [NR][tr]
  const int tr = S::row(T.max_rank);
  const unsigned sl = smem_u32(slab);
  __syncthreads();

  // ---------------------------------------------------------------- a warp's outputs: units of 16 Z of this CTA's, in pieces of RP ranks, through its ring
  const int outs = T.out, units = (outs + 16 * Z - 1) / (16 * Z), per = (units + ctas - 1) / ctas, u0 = min(me * per, units) + warp, u1 = min((me + 1) * per, units);
  const int prow = S::prow(T.max_rank), unit = S::unit(T.max_rank), bo = 16 * Z * prow, pieces = max(passes, 1);
  const int items = u0 < u1 ? (u1 - u0 + AD_WARPS - 1) / AD_WARPS * pieces : 0;
  // What a lane copies of a unit is the same in each: from where in B and to where in the stage (16-byte pieces of a row; of the last ranks there may be
  // fewer), and which rows of base.
  constexpr int NC = Z * RP * W::SIZE / 32, PR = 4 * Z, NP = NR * PR / 32;
  const int rowb = T.max_rank * W::SIZE, wide = min(T.max_rank, RP) * W::SIZE / 16;
  int cf[NC];
  unsigned ct[NC];
#pragma unroll
  for (int z = 0; z < NC; z++) {
    const int e = lane + 32 * z, r = e / wide, x = e - r * wide;
    cf[z] = r < 16 * Z && rank ? r * rowb + 16 * x : -1;
    ct[z] = (unsigned)((r % (2 * Z) * 8 + r / (2 * Z)) * prow + 16 * x);              // row 2 Z g + i of a unit is its row 8 i + g
  }
  const float* pb[NP];                                   // null: no such row
#pragma unroll
  for (int z = 0; z < NP; z++) {
    const int r = s_row[lane / PR + 32 / PR * z];
    pb[z] = r < 0 ? nullptr : T.base + (size_t)r * T.ldb + lane % PR * 4 + 16 * Z * u0;
  }
  const unsigned pt = sl + bo + 4 * (lane / PR * S::PB + lane % PR * 4);
  const unsigned char* b0 = static_cast<const unsigned char*>(T.b) + ((size_t)slot * outs + 16 * Z * u0) * rowb;
  auto ask = [&](int i, int p, int v) {                  // item i, piece p of the warp's unit number v
    if (i < items) {
      const unsigned st = (i & 1) * unit;
      const unsigned char* from = b0 + (size_t)v * (AD_WARPS * 16 * Z) * rowb + p * (RP * W::SIZE);
      const int left = outs - 16 * Z * (u0 + v * AD_WARPS);              // outputs from here on
      if (left >= 16 * Z && (p + 1) * RP <= T.max_rank) {
#pragma unroll
        for (int z = 0; z < NC; z++) if (cf[z] >= 0) ad_copy(sl + st + ct[z], from + cf[z], 16);
      } else {
        const int end = min(left, 16 * Z) * rowb, have = rowb - p * RP * W::SIZE;      // bytes of B in the unit, of a row from here on
#pragma unroll
        for (int z = 0; z < NC; z++) if (cf[z] >= 0 && cf[z] < end && cf[z] % rowb < have) ad_copy(sl + st + ct[z], from + cf[z], 16);
      }
      if (p == pieces - 1) {
        const int bytes = 4 * min(4, left - lane % PR * 4);
#pragma unroll
        for (int z = 0; z < NP; z++) if (pb[z] && bytes > 0) ad_copy(pt + st + z * (32 / PR * S::PB * 4), pb[z] + v * (AD_WARPS * 16 * Z), bytes);
      }
    }
    ad_commit();
  };

  // ---------------------------------------------------------------- t = A x over this CTA's columns, every eighth 16 of them a warp's
  {
    const int each = (((c.in + ctas - 1) / ctas) + 63) & ~63, kbegin = min(me * each, c.in), kend = min(kbegin + each, c.in);
    const int steps = (kend - kbegin + 15) / 16, mine = warp < steps ? (steps - warp + AD_WARPS - 1) / AD_WARPS : 0;
    float* part = reinterpret_cast<float*>(front);
    constexpr int APR = W::SIZE, ARI = 32 / APR, NA = RP / ARI;      // 16-byte pieces of a row of A in a step, rows that a copy of the warp takes, copies
    const int rest = kend - kbegin - 16 * warp;          // columns from the warp's first step on
    const size_t arow = (size_t)ARI * c.in * W::SIZE;
    const unsigned char* a0 = static_cast<const unsigned char*>(T.a) + ((size_t)(slot * (long long)T.max_rank + lane / APR) * c.in + kbegin + 16 * warp) * W::SIZE + lane % APR * 16;
    const float* xr[NB];                                 // null: no such row
#pragma unroll
    for (int z = 0; z < NB; z++) {
      const int r = s_row[lane / 4 + 8 * z];
      xr[z] = r < 0 ? nullptr : c.x + (size_t)r * c.ldx + kbegin + 16 * warp + lane % 4 * 4;
    }
    const unsigned at_a = sl + lane / APR * S::PA + lane % APR * 16, at_x = sl + S::XO + lane / 4 * S::PX + lane % 4 * 16, wl = sl + W::place(S::PA);
    const float* xl = reinterpret_cast<const float*>(slab + S::XO + g * S::PX) + 2 * q;
    for (int p = 0; p < passes; p++) {
      const int ranks = min(RP, rank - p * RP);
      const unsigned char* ap = a0 + (size_t)p * RP * c.in * W::SIZE;
      int in = 0;                                        // the stage that is filled next, as an offset
      auto get = [&](int i) {                            // the copies of the warp's step i
        if (i < mine) {
          const int k = 16 * AD_WARPS * i, n = rest - k; // columns that there are from here on: 8, or 16 and more
          if (n >= 16 || lane % APR * (16 / W::SIZE) < n) {
#pragma unroll
            for (int z = 0; z < NA; z++) if (lane / APR + ARI * z < ranks) ad_copy(at_a + in + z * (ARI * S::PA), ap + z * arow + k * W::SIZE, 16);
          }
          if (n >= 16 || lane % 4 < 2) {
#pragma unroll
            for (int z = 0; z < NB; z++) if (xr[z]) ad_copy(at_x + in + z * (8 * S::PX), xr[z] + k, 16);
          }
        }
        in = in == (S::STEPS - 1) * S::STEP ? 0 : in + S::STEP;
        ad_commit();
      };
      float d[MR][NB][4], sum[S::SUMS ? MR : 1][NB][4];
#pragma unroll
      for (int m = 0; m < MR; m++)
#pragma unroll
        for (int n = 0; n < NB; n++) {
          d[m][n][0] = d[m][n][1] = d[m][n][2] = d[m][n][3] = 0.f;
          if (S::SUMS) sum[S::SUMS ? m : 0][n][0] = sum[S::SUMS ? m : 0][n][1] = sum[S::SUMS ? m : 0][n][2] = sum[S::SUMS ? m : 0][n][3] = 0.f;
        }
      float up[NB], d0[NB], d1[NB];                      // float16: the powers of two of rows g, and the inverses of rows 2 q and 2 q + 1
      unsigned lim[NB];
#pragma unroll
      for (int n = 0; n < NB; n++) { up[n] = d0[n] = d1[n] = 1.f; lim[n] = 0u; }
#pragma unroll
      for (int i = 0; i < S::STEPS - 1; i++) get(i);
      int out = 0;
      auto step = [&](auto cut) {                        // the step at `out`; cut: it has 8 columns
        constexpr bool CUT = decltype(cut)::value;
        unsigned xp[NB][3][2];
#pragma unroll
        for (int n = 0; n < NB; n++) {
          const float2* src = reinterpret_cast<const float2*>(reinterpret_cast<const unsigned char*>(xl) + out + n * (8 * S::PX));
          const float2 lo = src[0], hi = src[4];
          float4 v = make_float4(lo.x, lo.y, hi.x, hi.y);
          if (CUT) v.z = v.w = 0.f;                      // behind the last column
          if constexpr (DT == 2) {
            if (8 * n + g >= count) v = make_float4(0.f, 0.f, 0.f, 0.f);           // nothing was copied here
            unsigned top = max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu), max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
            if (__any_sync(0xffffffffu, top >= lim[n])) {
              top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
              top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
              float down = 0.f;
              if (top >= lim[n]) { up[n] = ad_up(top, down); lim[n] = (min(max(top >> 23, 8u), 254u) + 7u) << 23; }
              // the rows whose power changed: what their sums held is put down to it
              const float n0 = __shfl_sync(0xffffffffu, down, 8 * q), n1 = __shfl_sync(0xffffffffu, down, 8 * q + 4);
              const float f0 = n0 != 0.f ? d0[n] / n0 : 1.f, f1 = n1 != 0.f ? d1[n] / n1 : 1.f;
              if (n0 != 0.f) d0[n] = n0;
              if (n1 != 0.f) d1[n] = n1;
#pragma unroll
              for (int m = 0; m < MR; m++) {
                d[m][n][0] *= f0; d[m][n][1] *= f1; d[m][n][2] *= f0; d[m][n][3] *= f1;
                if (S::SUMS) { float* w = sum[S::SUMS ? m : 0][n]; w[0] *= f0; w[1] *= f1; w[2] *= f0; w[3] *= f1; }
              }
            }
            v.x *= up[n]; v.y *= up[n]; v.z *= up[n]; v.w *= up[n];
          }
          W::values(v, xp[n]);
        }
#pragma unroll
        for (int m = 0; m < MR; m++) {
          if (MR > 1 && 16 * m >= ranks) break;
          unsigned wp[W::PIECES][4];
          W::template load<CUT>(wp, wl + out + m * (16 * S::PA), S::PA, 8);
#define AD_MMA(I, J) { _Pragma("unroll") for (int n = 0; n < NB; n++) W::template mma<I, J, false>(d[m][n], wp, xp[n]); }
          AD_MMA(2, 0) AD_MMA(1, 1) AD_MMA(0, 2) AD_MMA(1, 0) AD_MMA(0, 1) AD_MMA(0, 0)
#undef AD_MMA
        }
        out = out == (S::STEPS - 1) * S::STEP ? 0 : out + S::STEP;
      };
      for (int i = 0; i < mine; i++) {
        get(i + S::STEPS - 1);
        ad_wait<S::STEPS - 1>();
        __syncwarp();
        if (rest - 16 * AD_WARPS * i >= 16) step(std::false_type());
        else step(std::true_type());
        if (S::SUMS && ((i & (DT == 1 ? 3 : 7)) == (DT == 1 ? 3 : 7) || i == mine - 1)) {      // 24 products
#pragma unroll
          for (int m = 0; m < MR; m++)
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
              for (int z = 0; z < 4; z++) { sum[S::SUMS ? m : 0][n][z] += d[m][n][z]; d[m][n][z] = 0.f; }
        }
        __syncwarp();                                    // every lane has read the step that is filled next
      }
      ad_wait<0>();
      __syncwarp();
      if (p == passes - 1) ask(0, 0, 0);
      // [warp][row][rank]: rows 2 q and 2 q + 1 of ranks g and g + 8; more warps than there is room for add to the first ones' sums
      if (p) __syncthreads();                            // the sums of the pass before have been read
#pragma unroll
      for (int h = 0; h < AD_WARPS / S::ROUND; h++) {
        if (warp / S::ROUND == h) {
#pragma unroll
          for (int n = 0; n < NB; n++) {
            float* to = part + (size_t)(warp % S::ROUND * NR + 8 * n + 2 * q) * S::PP + g;
#pragma unroll
            for (int m = 0; m < MR; m++)
#pragma unroll
              for (int z = 0; z < 4; z++) {
                float* at = to + (z & 1) * S::PP + 16 * m + 8 * (z >> 1);
                float v = S::SUMS ? sum[S::SUMS ? m : 0][n][z] : d[m][n][z];
                if (DT == 2) v *= z & 1 ? d1[n] : d0[n];
                *at = h ? *at + v : v;
              }
          }
        }
        __syncthreads();
      }
      for (int e = tid; e < NR * RP; e += AD_THREADS) {
        const int j = p * RP + e % RP;
        if (j >= rank) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < S::ROUND; w++) v += part[(w * NR + e / RP) * S::PP + e % RP];
        t[e / RP * tr + j] = v;
      }
    }
    if (passes == 0) ask(0, 0, 0);
  }
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");

  // ---------------------------------------------------------------- the CTAs' sums of t, scaled: each CTA adds up its share of it and hands that to all
  // (with every CTA reading all of the others' sums, distributed shared memory took 3 us with 8 CTAs and 12 with 16). An item is what a lane has of a
  // fragment: four ranks of a row.
  float4* whole = reinterpret_cast<float4*>(front);      // [16 ranks][8 rows][lane]
  uint2* frag = reinterpret_cast<uint2*>(t);             // [16 ranks][8 rows][piece][lane]
  const int all = nk * NB * 32, share = (all + ctas - 1) / ctas;
  for (int e = me * share + tid; e < min((me + 1) * share, all); e += AD_THREADS) {
    const int l = e & 31, n = e / 32 % NB, k = e / 32 / NB, at = (8 * n + (l >> 2)) * tr + 16 * k, j = 16 * k + 2 * (l & 3);
    float4 a[8], v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r0 = 0; r0 < ctas; r0 += 8) {               // eight under way at once
#pragma unroll
      for (int r = 0; r < 8; r++) if (r0 + r < ctas) a[r] = ad_four(cluster.map_shared_rank(t, r0 + r) + at, l & 3);
#pragma unroll
      for (int r = 0; r < 8; r++) if (r0 + r < ctas) { v.x += a[r].x; v.y += a[r].y; v.z += a[r].z; v.w += a[r].w; }
    }
    v.x = j < rank ? v.x * scale : 0.f; v.y = j + 1 < rank ? v.y * scale : 0.f; v.z = j + 8 < rank ? v.z * scale : 0.f; v.w = j + 9 < rank ? v.w * scale : 0.f;
    for (int r = 0; r < ctas; r++) cluster.map_shared_rank(whole, r)[e] = v;
  }
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");          // from here on nobody touches another CTA's shared memory
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  if constexpr (DT == 2) {
    for (int r = warp; r < NR; r += AD_WARPS) {          // a power of two for each row
      unsigned top = 0u;
      for (int e = lane; e < nk * 4; e += 32) {
        const float4 v = whole[((e >> 2) * NB + (r >> 3)) * 32 + (r & 7) * 4 + (e & 3)];
        top = max(top, max(max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu), max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu)));
      }
      top = __reduce_max_sync(0xffffffffu, top);
      float down;
      const float up = ad_up(top, down);
      if (lane == 0) s_down[r] = down;
      for (int e = lane; e < nk * 4; e += 32) {          // the row's fragments: eight steps at a time
        const int at = ((e >> 2) * NB + (r >> 3)) * 32 + (r & 7) * 4 + (e & 3);
        float4 v = whole[at];
        v.x *= up; v.y *= up; v.z *= up; v.w *= up;
        unsigned f[3][2];
        W::values(v, f);
#pragma unroll
        for (int s = 0; s < 3; s++) frag[(at / 32 * 3 + s) * 32 + at % 32] = make_uint2(f[s][0], f[s][1]);
      }
    }
  } else {
    for (int e = tid; e < all; e += AD_THREADS) {
      unsigned f[3][2];
      W::values(whole[e], f);
#pragma unroll
      for (int s = 0; s < 3; s++) frag[(e / 32 * 3 + s) * 32 + e % 32] = make_uint2(f[s][0], f[s][1]);
    }
  }
  __syncthreads();

  // ---------------------------------------------------------------- y = base + B t
  // A unit's products have the outputs 2 Z g + 2 z and 2 Z g + 2 z + 1 in their rows g and g + 8: a lane's outputs of a row are neighbours.
  float* to[NB][2];                                      // the lane's rows 2 q and 2 q + 1 at its outputs of the warp's first unit
  float down[NB][2];
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int r = s_row[8 * n + 2 * q + h];
      to[n][h] = r < 0 ? nullptr : T.y + (size_t)r * T.ldy + 16 * Z * u0 + 2 * Z * g;
      down[n][h] = DT == 2 ? s_down[8 * n + 2 * q + h] : 1.f;
    }
  const unsigned fr = smem_u32(frag) + 8 * lane, wl = sl + W::place(prow);
  const float* bl = reinterpret_cast<const float*>(slab + bo) + 2 * q * S::PB + 2 * Z * g;
  // t's fragments of a warp's one block of rows stay in registers where they are one piece
  constexpr int HELD = NB == 1 ? MR : 1;
  unsigned xh[HELD][3][2];
  auto fetch = [&](unsigned at, unsigned (&x)[3][2]) {
#pragma unroll
    for (int s = 0; s < 3; s++) { const uint2 v = lds64(at + s * 256); x[s][0] = v.x; x[s][1] = v.y; }
  };
  if (NB == 1 && pieces == 1) {
#pragma unroll
    for (int k = 0; k < HELD; k++) if (k < nk) fetch(fr + k * 768, xh[k]);
  }
  float d[Z][NB][4];
  int p = 0, v = 0;                                      // piece and number of the unit
  for (int i = 0; i < items; i++) {
    const bool last = p == pieces - 1;
    ask(i + 1, last ? 0 : p + 1, last ? v + 1 : v);
    ad_wait<1>();
    __syncwarp();
    const int st = (i & 1) * unit;
    if (p == 0) {
#pragma unroll
      for (int z = 0; z < Z; z++)
#pragma unroll
        for (int n = 0; n < NB; n++) d[z][n][0] = d[z][n][1] = d[z][n][2] = d[z][n][3] = 0.f;
    }
    if (NB == 1 && pieces > 1) {                         // each unit goes through all pieces anew
#pragma unroll
      for (int k = 0; k < HELD; k++) if (p * MR + k < nk) fetch(fr + (p * MR + k) * 768, xh[k]);
    }
    auto step = [&](auto cut, int k, int left) {         // 16 ranks; cut: what stands behind the adapter's rank does not count
      constexpr bool CUT = decltype(cut)::value;
      unsigned wp[Z][W::PIECES][4];
#pragma unroll
      for (int z = 0; z < Z; z++) W::template load<CUT>(wp[z], wl + st + 16 * z * prow + 16 * k * W::SIZE, prow, left);
#pragma unroll
      for (int n = 0; n < NB; n++) {
        unsigned xp[3][2];
        if constexpr (NB > 1) fetch(fr + ((p * MR + k) * NB + n) * 768, xp);
#define AD_MMA(I, J) { _Pragma("unroll") for (int z = 0; z < Z; z++) W::template mma<I, J, false>(d[z][n], wp[z], NB > 1 ? xp : xh[NB > 1 ? 0 : k]); }
        AD_MMA(2, 0) AD_MMA(1, 1) AD_MMA(0, 2) AD_MMA(1, 0) AD_MMA(0, 1) AD_MMA(0, 0)
#undef AD_MMA
      }
    };
    const int left = rank - p * RP;
    if (left >= RP) {
#pragma unroll
      for (int k = 0; k < MR; k++) step(std::false_type(), k, 16);
    } else {
#pragma unroll
      for (int k = 0; k < MR; k++) if (16 * k < left) step(std::true_type(), k, left - 16 * k);
    }
    if (last) {
      const int there = outs - 16 * Z * (u0 + v * AD_WARPS) - 2 * Z * g;
      const float* base = reinterpret_cast<const float*>(reinterpret_cast<const unsigned char*>(bl) + st);
#pragma unroll
      for (int n = 0; n < NB; n++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const float* from = base + (8 * n + h) * S::PB;
          float y[2 * Z];
          if constexpr (Z == 2) { const float4 b = *reinterpret_cast<const float4*>(from); y[0] = b.x; y[1] = b.y; y[2 * Z - 2] = b.z; y[2 * Z - 1] = b.w; }
          else { const float2 b = *reinterpret_cast<const float2*>(from); y[0] = b.x; y[1] = b.y; }
#pragma unroll
          for (int o = 0; o < 2 * Z; o++) {
            const float w = d[o >> 1][n][2 * (o & 1) + h];
            y[o] = DT == 2 ? fmaf(w, down[n][h], y[o]) : y[o] + w;
          }
          if (!to[n][h]) continue;
          float* at = to[n][h] + v * (AD_WARPS * 16 * Z);
          if (there >= 2 * Z) {
            if constexpr (Z == 2) *reinterpret_cast<float4*>(at) = make_float4(y[0], y[1], y[2 * Z - 2], y[2 * Z - 1]);
            else *reinterpret_cast<float2*>(at) = make_float2(y[0], y[1]);
          } else {
#pragma unroll
            for (int o = 0; o < 2 * Z - 1; o++) if (o < there) at[o] = y[o];
          }
        }
    }
    __syncwarp();                                        // every lane has read the item that is replaced next
    p = last ? 0 : p + 1;
    v += last;
  }
  ad_wait<0>();
}

// ------------------------------------------------------------------ host
template <int DT, int NR, int MR> static cudaError_t ad_go(AdCall c, int n, int ranks, int ctas, cudaStream_t st) {
  using S = AdShape<DT, NR, MR>;
  auto kern = adapter_kernel<DT, NR, MR>;
  static unsigned long long attr_mask = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !(attr_mask & (1ull << dev))) {
    constexpr int most = MR == 4 ? AD_RANK : 16 * MR;
    static_assert(S::smem(most, S::slab(most)) <= 227 * 1024 - 1024, "shared memory");
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::smem(most, S::slab(most)));
    if (e != cudaSuccess) return e;
    const cudaError_t f = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (f != cudaSuccess) return f;
    if (dev < 64) attr_mask |= 1ull << dev;
  }
  c.slab = S::slab(ranks);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.gridDim = dim3((unsigned)(c.tiles * ctas), (unsigned)n); cfg.blockDim = dim3(AD_THREADS); cfg.dynamicSmemBytes = S::smem(ranks, c.slab); cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)ctas; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at; cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, c);
}
template <int DT, int NR> static cudaError_t ad_pick(const AdCall& c, int n, int ranks, int ctas, cudaStream_t st) {
  return ranks <= 16 ? ad_go<DT, NR, 1>(c, n, ranks, ctas, st) : ranks <= 32 ? ad_go<DT, NR, 2>(c, n, ranks, ctas, st) : ad_go<DT, NR, 4>(c, n, ranks, ctas, st);
}
template <int DT> static cudaError_t ad_any(const AdCall& c, int n, int ranks, int ctas, cudaStream_t st) {
  return c.size == 32 ? ad_pick<DT, 32>(c, n, ranks, ctas, st) : ad_pick<DT, 8>(c, n, ranks, ctas, st);
}
static int ad_counts(const char* who, int rows, int slots) {
  if (rows < 0 || rows > 1 << 24 || slots < 1 || slots > AD_SLOTS) { wv_set_error("%s: %d rows, %d adapters (1 to %d)", who, rows, slots, AD_SLOTS); return WV_ESHAPE; }
  return WV_OK;
}

// Whether two matrices of `rows` rows, wp of each ldp values and wq of each ldq, have a value in common. Columns of one matrix with the same stride may lie
// beside one another.
static bool ad_meets(const float* p, int ldp, int wp, const float* q, int ldq, int wq, int rows) {
  const long long d = (static_cast<long long>(reinterpret_cast<uintptr_t>(q)) - static_cast<long long>(reinterpret_cast<uintptr_t>(p))) / 4;      // both 16-byte aligned
  const long long endp = (rows - 1LL) * ldp + wp, endq = (rows - 1LL) * ldq + wq;
  if (d >= endp || -d >= endq) return false;
  if (ldp == ldq) {
    const long long o = (d % ldp + ldp) % ldp;           // q's columns begin o behind p's
    return o < wp || o + wq > ldp;
  }
  for (long long r = 0; r < rows; r++) {                 // the first of q's rows that ends behind the beginning of p's
    const long long a = r * ldp - d, j = a < wq ? 0 : (a - wq) / ldq + 1;
    if (j < rows && j * ldq < a + wp) return true;
  }
  return false;
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
  if (f.in > AD_WIDE) { wv_set_error("%s: %d columns (at most %d)", who, f.in, AD_WIDE); return WV_ESHAPE; }
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
    if (w.max_rank < 8 || w.max_rank % 8 || w.max_rank > AD_RANK || w.out < 1 || w.out > AD_WIDE) {
      wv_set_error("%s: target %d: %d outputs (at most %d), rank %d (a multiple of 8, at most %d)", who, i, w.out, AD_WIDE, w.max_rank, AD_RANK); return WV_ESHAPE;
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
  // targets run side by side, all of them read x, and clusters read base while others write
  for (int i = 0; i < n; i++) {
    const AdTarget& t = c.t[i];
    if (ad_meets(t.y, t.ldy, t.out, dx, ldx, f.in, rows)) { wv_set_error("%s: target %d writes into x", who, i); return WV_EARG; }
    for (int j = 0; j < n; j++) {
      const AdTarget& o = c.t[j];
      if ((i != j && ad_meets(t.y, t.ldy, t.out, o.y, o.ldy, o.out, rows)) || ((i != j || t.y != t.base) && ad_meets(t.y, t.ldy, t.out, o.base, o.ldb, o.out, rows))) {
        wv_set_error("%s: target %d writes what target %d reads or writes", who, i, j); return WV_EARG;
      }
    }
  }
  c.x = dx; c.ldx = ldx; c.in = f.in; c.rows = rows; c.slots = f.slots;
  c.size = ad_tile(rows, f.slots); c.tiles = ad_tiles(rows, f.slots);
  c.plan = static_cast<const int4*>(d_plan);
  c.place = reinterpret_cast<const int*>(c.plan + 1 + c.tiles);
  c.err = wv_paged_err_ptr();
  if (c.tiles * AD_CTAS > INT_MAX) { wv_set_error("%s: %d rows are too many", who, rows); return WV_ESHAPE; }
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // CTAs of a cluster: as many as let the tiles that are expected (half of the adapters' last ones beside the full ones) run at once, two CTAs an SM: a row
  // beside Q, K and V takes 10.0, 8.0 and 7.5 us with 4, 8 and 16, 64 rows of 32 adapters 17 with 4 and 22 with 8, 2048 rows of six 53 and 69. Where sums are
  // one chain (32 rows, ranks beyond 32), no more than 1792 columns each. Shared memory leaves an SM one CTA where ranks are wide (16-bit weights from some 80
  // in tiles of 32 rows and 128 in tiles of 8, float32 ones beyond 32): such calls may run their clusters in two turns where one would do.
  const long long likely = n * std::max(1LL, (long long)rows / c.size + (std::min(rows, f.slots) + 1) / 2), room = 2LL * wv_sm_count();
  int ctas = 2;
  while (ctas < AD_CTAS && likely * ctas * 2 <= room) ctas *= 2;
  while (c.size == 32 && ranks > 32 && f.in > 1792 * ctas && ctas < AD_CTAS) ctas *= 2;
  const cudaError_t e = f.dtype == 1 ? ad_any<1>(c, n, ranks, ctas, st) : f.dtype == 2 ? ad_any<2>(c, n, ranks, ctas, st) : ad_any<3>(c, n, ranks, ctas, st);
  if (e != cudaSuccess) { cudaGetLastError(); wv_set_error("%s: launch: %s", who, cudaGetErrorString(e)); return WV_ECUDA; }
  return WV_OK;
}
