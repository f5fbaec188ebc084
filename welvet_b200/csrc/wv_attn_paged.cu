// Attention of the new tokens of a batch over the paged cache (include/welvet_cuda.h, wv_attn_paged_dev): few rows against many keys.
//
// The rows of a block are the query heads of one kv head, for one token or a few: up to 8 of them (or 16) against all keys, so
// that a cached row is read once for all of them. Bound: HBM, one pass over the pages; arithmetic intensity is 2 x 8 products a
// code. The products run on mma.sync m16n8k16 (float16 operands, float32 sums): with so few rows a tcgen05 tile of 128 would be nine
// tenths padding. Codes are exact in float16; q and the weights go through it as two pieces each, hi + lo (22 bits). With up to 8 rows
// the pieces share one instruction, hi in the fragment's rows 0-7 and lo in rows 8-15, and a lane finds both sums in its own
// registers; with 9 to 16 rows there is an instruction for each.
//
// A warp works alone: it takes 16 keys at a time, copies their K and V rows, scales and sub-scales into its own ring of shared memory
// (cp.async, 20 to 25 KB in flight a warp, no barrier but its own), turns codes into float16 as it reads them, and keeps maximum,
// divisor and the weighted sum in registers. Which 8 or 16 values of a row a lane reads is chosen so that they are neighbours in
// memory: the order of the products does not matter for K, and for V it only decides which output a lane holds. Rows lie in the
// ring with their 16-byte pieces permuted so that both reading patterns are free of bank conflicts.
//
// Four warps a block, two blocks an SM, so that one block's start (three dependent loads: lengths, page numbers, rows) runs beside
// another's keys. The keys of a sequence are split over blocks; the splits leave {M, divisor, sums} and a second kernel joins them
// in order, so results do not depend on who ran first.
#include "wv_attn_paged.cuh"
#include "wv_lease.h"
#include <cuda_pipeline.h>

int wv_sm_count();

#define PR_WARPS 4

template <int BITS, int DP> struct PrShape {
  static constexpr int RB = DP * BITS / 8;                               // bytes of a row in the ring
  static constexpr int SUB = BITS == 4 ? DP : 0;                         // bytes of the sub-scales of 16 keys
  static constexpr int STAGE = 32 * RB + 128 + 2 * SUB;                  // K rows, V rows, 2 x 16 scales, sub-scales
  static constexpr int FIT = 25 * 1024 / STAGE;
  static constexpr int NST = FIT < 2 ? 2 : (FIT > 8 ? 8 : FIT);
  static constexpr int CH = BITS == 4 ? 8 : 16;                          // bytes of a copy: 4-bit rows are multiples of 8
  static constexpr int NCP = (16 * RB / CH + 31) / 32;                   // copies a lane makes for K (and for V)
};

// Where the 16-byte piece j of row r lies in a ring of rows of RB bytes.
template <int RB> __device__ __forceinline__ unsigned pr_at(int r, int j) {
  if constexpr (RB >= 128) {
    const int sw = ((r >> 1) & 3) << 1 ^ (r & 1) << 2;
    return (unsigned)(r * RB + ((j & ~7) | ((j ^ sw) & 7)) * 16);
  } else {
    constexpr int PER = 128 / RB;                                        // rows in 128 bytes
    const int line = r / PER, sw = (RB == 64 ? line & 3 : line & 1) << 1;
    return (unsigned)(line * 128 + ((((r % PER) * (RB / 16) + j) ^ sw) & 7) * 16);
  }
}
__device__ __forceinline__ void pr_mma(float (&d)[4], const uint4& a, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// The value index within a row of element e (0..3: k = 2c, 2c+1, 2c+8, 2c+9 of the fragment) of QK step s in lane column c.
template <int BITS, int DP> __device__ __forceinline__ int pr_kdim(int s, int c, int e) {
  if constexpr (BITS == 16) return (c + 4 * (s >> 1)) * 8 + 4 * (s & 1) + e;
  if constexpr (BITS == 8) return (c + 4 * (s >> 2)) * 16 + 4 * (s & 3) + e;
  if constexpr (DP == 64) return c * 16 + 8 * (s >> 1) + 2 * (s & 1) + (e >> 1) + 4 * (e & 1);
  return (c + 4 * (s >> 3)) * 32 + 8 * ((s >> 1) & 3) + 2 * (s & 1) + (e >> 1) + 4 * (e & 1);
}
// One value's code out of a ring of V rows, times its sub-scale.
template <int BITS, int DP> __device__ __forceinline__ float pr_code(const unsigned char* rows, const unsigned char* sub, int r, int d, int hd) {
  constexpr int RB = PrShape<BITS, DP>::RB;
  const int at = d * BITS / 8;
  const unsigned char* p = rows + pr_at<RB>(r, at >> 4) + (at & 15);
  if constexpr (BITS == 16) return __half2float(*reinterpret_cast<const __half*>(p));
  if constexpr (BITS == 8) return (float)(int)*reinterpret_cast<const signed char*>(p);
  return (float)(((int)((*p >> (4 * (d & 1))) & 15u) - 8) * (int)sub[r * (hd / 16) + min(d, hd - 1) / 16]);
}
// The value index of column n of PV's n-tile t.
template <int BITS, int DP> __device__ __forceinline__ int pr_vdim(int t, int n) {
  if constexpr (BITS == 16) return (n + 8 * (t >> 3)) * 8 + (t & 7);
  if constexpr (BITS == 8 && DP >= 128) return (n + 8 * (t >> 4)) * 16 + (t & 15);
  if constexpr (BITS == 4 && DP == 256) return n * 32 + t;
  return n * (DP / 8) + t;
}

template <int BITS, int DP, bool R16>
__global__ void __launch_bounds__(32 * PR_WARPS, (BITS == 16 && DP == 256) || (DP == 256 && R16) ? 1 : 2) attn_rows_kernel(const __grid_constant__ PaCall c) {
  using S = PrShape<BITS, DP>;
  constexpr int RB = S::RB, KS = DP / 16, NT = DP / 8, NROW = R16 ? 16 : 8, NST = S::NST;
  constexpr bool QREG = KS * (R16 ? 8 : 4) <= 32;                        // q fragments in registers, or read from shared memory each time
  extern __shared__ __align__(128) unsigned char pr_smem[];
  __shared__ uint4 s_qf[(R16 ? 2 : 1) * KS * 32];
  __shared__ float2 s_ml[PR_WARPS][NROW];
  __shared__ unsigned s_qmax;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, cl = lane & 3;
  unsigned char* ring = pr_smem + warp * NST * S::STAGE;
  if (tid == 0) s_qmax = 0;
  if (c.g.hd < DP) {                                                     // what lies beyond the head stays zero
    for (int i = tid * 16; i < PR_WARPS * NST * S::STAGE; i += 32 * PR_WARPS * 16) *reinterpret_cast<uint4*>(pr_smem + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int tiles = gridDim.x / (c.b.num_seqs * c.g.kvh);
  const int kvh = blockIdx.x % c.g.kvh, tile = blockIdx.x / c.g.kvh % tiles, seq = blockIdx.x / c.g.kvh / tiles, sp = blockIdx.y;
  const WvSeq sq = wv_seq(c.b, c.g.page, seq, sp == 0 && kvh == 0 && tile == 0 ? c.err : nullptr);
  const int nrows = (sq.q1 - sq.q0) * c.group, r0 = tile * NROW;
  if (r0 >= nrows || nrows > c.rows_most) return;
  const int rn = min(NROW, nrows - r0);
  int lo, hi;
  pa_range(sq, r0 / c.group, (r0 + rn - 1) / c.group, c.window, lo, hi);
  const int k0 = lo + sp * c.per, k1 = min(hi, k0 + c.per);              // this block's keys; k0 is a multiple of 16
  auto rec = [&](int r) { return (((size_t)seq * c.g.kvh + kvh) * (tiles * NROW) + r0 + r) * c.nsplit + sp; };      // a row's split result
  if (k0 >= k1) {
    if (c.nsplit > 1) { if (tid < rn) c.ml[rec(tid)] = make_float2(-INFINITY, 0.f); }
    else for (int i = tid; i < rn * c.g.hd; i += 32 * PR_WARPS) {        // rows that see nothing
      const int r = i / c.g.hd, t = sq.q0 + (r0 + r) / c.group, h = kvh * c.group + (r0 + r) % c.group;
      c.out[(size_t)t * c.ldo + (size_t)h * c.g.hd + i % c.g.hd] = 0.f;
    }
    return;
  }

  // ---------------------------------------------------------------- the warp's groups of 16 keys: k0 / 16 + warp, + PR_WARPS, ...
  const int g0 = k0 / 16 + warp, ng = ((k1 + 15) / 16 - g0 + PR_WARPS - 1) / PR_WARPS;
  const int code = c.g.code;
  // a lane's copies of a group's K (or V) rows: the source is contiguous, the place in the ring the same in every stage
  const int ncp = 16 * code / S::CH;
  unsigned dst[S::NCP];
#pragma unroll
  for (int i = 0; i < S::NCP; i++) {
    const int at = (lane + 32 * i) * S::CH, r = at / code, o = at - r * code;
    dst[i] = lane + 32 * i < ncp ? pr_at<RB>(r, o / 16) + (o & 15) : 0u;
  }
  int ids = 0;                                                           // page numbers of 32 of the warp's groups, a lane each
  auto issue = [&](int it) {
    if ((it & 31) == 0) {
      const int gi = g0 + (it + lane) * PR_WARPS;
      int id = it + lane < ng ? c.b.pages[(size_t)seq * c.b.table_stride + gi * 16 / c.g.page] : 0;
      if (id < 0 || id >= c.g.num_pages) { wv_paged_report(c.err, WV_PAGED_PAGE); id = -1; }
      ids = id;
    }
    const int id = __shfl_sync(0xffffffffu, ids, it & 31);
    if (it < ng) {
      unsigned char* st = ring + (it % NST) * S::STAGE;
      const int key = (g0 + it * PR_WARPS) * 16, slot = key % c.g.page;
      const int have = id < 0 ? 0 : min(16, k1 - key);                   // keys of the group that exist; the rest is zeros
      const unsigned char* block = c.g.pool + ((size_t)max(id, 0) * c.g.kvh + kvh) * c.g.block;
      const unsigned char* ks = block + (size_t)slot * code;
      const unsigned char* vs = ks + (size_t)c.g.page * code;
      const int bytes = have * code;
#pragma unroll
      for (int i = 0; i < S::NCP; i++) {
        const int at = (lane + 32 * i) * S::CH;
        if (at < 16 * code) {
          const int z = at < bytes ? 0 : S::CH;
          __pipeline_memcpy_async(st + dst[i], ks + (z ? 0 : at), S::CH, z);
          __pipeline_memcpy_async(st + 16 * RB + dst[i], vs + (z ? 0 : at), S::CH, z);
        }
      }
      // scales (64 bytes each) and sub-scales
      unsigned char* sc = st + 32 * RB;
      if (lane < 8) __pipeline_memcpy_async(sc + 16 * lane, block + (lane < 4 ? c.g.kscale : c.g.vscale) + 4 * slot + 16 * (lane & 3), 16, have ? 0 : 16);
      if (BITS == 4) {
        const int n16 = c.g.hd / 16;                                     // 16-byte pieces of the 16 keys' sub-scales
        for (int i = lane; i < 2 * n16; i += 32) {
          const bool v = i >= n16;
          const int j = v ? i - n16 : i;
          __pipeline_memcpy_async(sc + 128 + (v ? S::SUB : 0) + 16 * j, block + (v ? c.g.vsub : c.g.ksub) + slot * n16 + 16 * j, 16, have ? 0 : 16);
        }
      }
    }
    __pipeline_commit();
    return id;
  };
  unsigned bad = 0;                                                      // bit it & 31: the group's page is outside the pool
  auto start = [&](int it) { const int id = issue(it); if (it < ng) bad = (bad & ~(1u << (it & 31))) | (unsigned)(id < 0) << (it & 31); };
#pragma unroll
  for (int i = 0; i < NST - 1; i++) start(i);

  // ---------------------------------------------------------------- q: a common power of two, then two float16 pieces, as fragments
  const int hd = c.g.hd;
  {
    unsigned m = 0;
    for (int i = tid; i < rn * hd / 4; i += 32 * PR_WARPS) {
      const int r = i * 4 / hd, d = i * 4 % hd, t = sq.q0 + (r0 + r) / c.group, h = kvh * c.group + (r0 + r) % c.group;
      const float4 v = *reinterpret_cast<const float4*>(c.q + (size_t)t * c.ldq + (size_t)h * hd + d);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; e++) { const unsigned u = __float_as_uint(x[e]) & 0x7fffffffu; if (u < 0x7f800000u) m = max(m, u); }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    __syncthreads();
    if (lane == 0) atomicMax(&s_qmax, m);
    __syncthreads();
  }
  const int qe = min(max((int)(s_qmax >> 23) - 127 - 13, -100), 114);    // max |q| 2^-qe in [2^13, 2^14)
  const float qinv = __uint_as_float((unsigned)(127 - qe) << 23);
  const float qf = c.scale * __uint_as_float((unsigned)(127 + qe) << 23);
  for (int i = tid; i < KS * 32; i += 32 * PR_WARPS) {
    const int s = i >> 5, g = (i & 31) >> 2, cc = i & 3;
    unsigned h_[2][2], l_[2][2];                                         // [row g, row g + 8][k half]
#pragma unroll
    for (int rr = 0; rr < (R16 ? 2 : 1); rr++) {
      const int r = g + 8 * rr;
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int d = pr_kdim<BITS, DP>(s, cc, e);
        x[e] = 0.f;
        if (r < rn && d < hd) {
          const int t = sq.q0 + (r0 + r) / c.group, h = kvh * c.group + (r0 + r) % c.group;
          const float v = c.q[(size_t)t * c.ldq + (size_t)h * hd + d];
          x[e] = v - v == 0.f ? v * qinv : NAN;                          // not finite: the row's sums are NaN
        }
      }
#pragma unroll
      for (int p = 0; p < 2; p++) {
        h_[rr][p] = pa_pack(x[2 * p], x[2 * p + 1]);
        const float2 b = pa_unpack(h_[rr][p]);
        l_[rr][p] = pa_pack(x[2 * p] - b.x, x[2 * p + 1] - b.y);
      }
    }
    if (R16) {
      s_qf[i] = make_uint4(h_[0][0], h_[1][0], h_[0][1], h_[1][1]);
      s_qf[KS * 32 + i] = make_uint4(l_[0][0], l_[1][0], l_[0][1], l_[1][1]);
    } else {
      s_qf[i] = make_uint4(h_[0][0], l_[0][0], h_[0][1], l_[0][1]);
    }
  }
  __syncthreads();
  uint4 qr[QREG ? (R16 ? 2 : 1) * KS : 1];
  if constexpr (QREG) {
#pragma unroll
    for (int i = 0; i < (R16 ? 2 : 1) * KS; i++) qr[i] = s_qf[i * 32 + lane];
  }
  auto qfrag = [&](int i) -> uint4 { if constexpr (QREG) return qr[i]; else return s_qf[i * 32 + lane]; };

  // the last position that a lane's rows see, and how far back
  constexpr int NR = R16 ? 2 : 1;
  int plast[NR];
#pragma unroll
  for (int i = 0; i < NR; i++) plast[i] = sq.kv - (sq.q1 - sq.q0) + (r0 + min(gl + 8 * i, rn - 1)) / c.group;
  const int pmin = sq.kv - (sq.q1 - sq.q0) + r0 / c.group, pmax = sq.kv - (sq.q1 - sq.q0) + (r0 + rn - 1) / c.group;

  float o[NT][4], m[NR], l[NR];
#pragma unroll
  for (int t = 0; t < NT; t++) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
#pragma unroll
  for (int i = 0; i < NR; i++) { m[i] = -INFINITY; l[i] = 0.f; }

  for (int it = 0; it < ng; it++) {
    __pipeline_wait_prior(NST - 2);
    __syncwarp();                                                        // every lane has read the stage that is filled next
    start(it + NST - 1);
    const unsigned char* st = ring + (it % NST) * S::STAGE;
    const unsigned char* sc = st + 32 * RB;
    const int key = (g0 + it * PR_WARPS) * 16;
    // -------------------------------------------------------------- logits of two n-tiles of 8 keys, two chains of sums each
    float s[2][2][4];
#pragma unroll
    for (int n = 0; n < 2; n++) {
#pragma unroll
      for (int ch = 0; ch < 2; ch++) s[n][ch][0] = s[n][ch][1] = s[n][ch][2] = s[n][ch][3] = 0.f;
      const int r = gl + 8 * n;
      auto step = [&](int k, unsigned b0, unsigned b1) {
        if (R16) pr_mma(s[n][k & 1], qfrag(KS + k), b0, b1);             // the small pieces first
        pr_mma(s[n][k & 1], qfrag(k), b0, b1);
      };
      if constexpr (BITS == 4 && DP == 64) {
        const uint2 w = *reinterpret_cast<const uint2*>(st + pr_at<RB>(r, cl >> 1) + 8 * (cl & 1));
        const unsigned t1 = sc[128 + r * (hd / 16) + min(cl, hd / 16 - 1)], t = pa_pair(t1, t1);
        step(0, pa_nibbles(w.x, 0, t), pa_nibbles(w.x, 1, t)); step(1, pa_nibbles(w.x, 2, t), pa_nibbles(w.x, 3, t));
        step(2, pa_nibbles(w.y, 0, t), pa_nibbles(w.y, 1, t)); step(3, pa_nibbles(w.y, 2, t), pa_nibbles(w.y, 3, t));
      } else {
#pragma unroll
        for (int i = 0; i < RB / 64; i++) {
          const uint4 v = *reinterpret_cast<const uint4*>(st + pr_at<RB>(r, cl + 4 * i));
          const unsigned w[4] = {v.x, v.y, v.z, v.w};
          if constexpr (BITS == 16) { step(2 * i, w[0], w[1]); step(2 * i + 1, w[2], w[3]); }
          if constexpr (BITS == 8) {
#pragma unroll
            for (int j = 0; j < 4; j++) { const unsigned x = w[j] ^ 0x80808080u; step(4 * i + j, pa_bytes<0x4140>(x), pa_bytes<0x4342>(x)); }
          }
          if constexpr (BITS == 4) {
            const int at = 2 * (cl + 4 * i), n16 = hd / 16;
            const unsigned ta = at < n16 ? sc[128 + r * n16 + at] : 0u, tb = at + 1 < n16 ? sc[128 + r * n16 + at + 1] : 0u;
            const unsigned t2[2] = {pa_pair(ta, ta), pa_pair(tb, tb)};
#pragma unroll
            for (int j = 0; j < 4; j++) {
              step(8 * i + 2 * j, pa_nibbles(w[j], 0, t2[j >> 1]), pa_nibbles(w[j], 1, t2[j >> 1]));
              step(8 * i + 2 * j + 1, pa_nibbles(w[j], 2, t2[j >> 1]), pa_nibbles(w[j], 3, t2[j >> 1]));
            }
          }
        }
      }
    }
    // -------------------------------------------------------------- weights of the lane's four keys 2c, 2c + 1, 2c + 8, 2c + 9
    const bool whole = key >= lo && key + 15 <= pmin && (c.window == 0 || key > pmax - c.window) && !((bad >> (it & 31)) & 1u);
    float y[NR][4], f[4], inv[4], emin = 1000.f, emax = -1000.f;
#pragma unroll
    for (int n = 0; n < 2; n++) {
      const float2 ks = *reinterpret_cast<const float2*>(sc + 4 * (8 * n + 2 * cl)), vs = *reinterpret_cast<const float2*>(sc + 64 + 4 * (8 * n + 2 * cl));
      const float kk[2] = {ks.x * qf, ks.y * qf}, vv[2] = {vs.x, vs.y};
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const float e = pa_split_scale(vv[j], f[2 * n + j], inv[2 * n + j]);
        if (e > -90.f && vv[j] == vv[j] && key + 8 * n + 2 * cl + j < k1) { emin = fminf(emin, e); emax = fmaxf(emax, e); }
        if (R16) {
          y[0][2 * n + j] = fmaf(s[n][0][j] + s[n][1][j], kk[j], e);
          y[NR - 1][2 * n + j] = fmaf(s[n][0][2 + j] + s[n][1][2 + j], kk[j], e);
        } else {
          y[0][2 * n + j] = fmaf((s[n][0][2 + j] + s[n][1][2 + j]) + (s[n][0][j] + s[n][1][j]), kk[j], e);
        }
      }
    }
    bool seen[NR][4];
    if (!whole) {
#pragma unroll
      for (int i = 0; i < NR; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int p = key + 8 * (j >> 1) + 2 * cl + (j & 1);
          seen[i][j] = p <= plast[i] && p < k1 && (c.window == 0 || p > plast[i] - c.window) && !((bad >> (it & 31)) & 1u);
          if (!seen[i][j]) y[i][j] = -INFINITY;
        }
    }
    uint4 ph, pl;
    unsigned* hh = reinterpret_cast<unsigned*>(&ph);
    unsigned* ll = reinterpret_cast<unsigned*>(&pl);
    // The 16 keys' value scales are all within 2^18 of one another, or (rows of zeros apart) the pieces' range may not hold them.
    const bool far = __any_sync(0xffffffffu, __reduce_max_sync(0xffffffffu, (int)emax + 1000) + __reduce_max_sync(0xffffffffu, 1000 - (int)emin) > 2018);
    float pw[NR][4];
    bool moved = false;
    float fac[NR], ref[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) {
      float mx = fmaxf(fmaxf(y[i][0], y[i][1]), fmaxf(y[i][2], y[i][3]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      mx = fmaxf(mx, m[i]);
      ref[i] = mx == -INFINITY ? 0.f : mx;
      fac[i] = pa_ex2(m[i] - ref[i]);
      moved |= mx != m[i];
      m[i] = mx;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int i = 0; i < NR; i++) l[i] *= fac[i];
#pragma unroll
      for (int t = 0; t < NT; t++) { o[t][0] *= fac[0]; o[t][1] *= fac[0]; o[t][2] *= fac[NR - 1]; o[t][3] *= fac[NR - 1]; }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
      float (&p)[4] = pw[i];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float e = pa_ex2(y[i][j] - (ref[i] - PA_LIFT));
        p[j] = e * f[j];
        const float w = e * inv[j];
        if (whole) l[i] += w;
        else { l[i] += seen[i][j] ? w : 0.f; p[j] = seen[i][j] ? p[j] : 0.f; }
      }
#pragma unroll
      for (int n = 0; n < 2; n++) {                                      // keys' halves: fragment registers 0, 2 of row g and 1, 3 of row g + 8
        const unsigned h = pa_pack(p[2 * n], p[2 * n + 1]);
        const float2 b = pa_unpack(h);
        const unsigned lw = pa_pack(p[2 * n] - b.x, p[2 * n + 1] - b.y);
        if (R16) { hh[2 * n + i] = h; ll[2 * n + i] = lw; }
        else { hh[2 * n] = h; hh[2 * n + 1] = lw; }
      }
    }
    // -------------------------------------------------------------- weighted sum of the V rows
    const unsigned char* vb = st + 16 * RB;
    auto put = [&](int t, unsigned b0, unsigned b1) {
      if (R16) pr_mma(o[t], pl, b0, b1);
      pr_mma(o[t], ph, b0, b1);
    };
    const int rows4[4] = {2 * cl, 2 * cl + 1, 2 * cl + 8, 2 * cl + 9};
    if (far) {                                                           // value by value in float32
#pragma unroll 1
      for (int j = 0; j < 16; j++) {
        const int mine = 2 * (j >> 3) + (j & 1), from = (lane & ~3) | ((j & 7) >> 1);
        float w[NR];
#pragma unroll
        for (int i = 0; i < NR; i++) {
          const float x = mine == 0 ? pw[i][0] : mine == 1 ? pw[i][1] : mine == 2 ? pw[i][2] : pw[i][3];
          w[i] = __shfl_sync(0xffffffffu, x, from);
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int n = 0; n < 2; n++) {
            const float x = pr_code<BITS, DP>(vb, sc + 128 + S::SUB, j, pr_vdim<BITS, DP>(t, 2 * cl + n), hd);
            o[t][n] += w[0] * x;
            if (R16) o[t][2 + n] += w[NR - 1] * x;
          }
      }
      continue;
    }
    if constexpr (BITS == 16) {
#pragma unroll
      for (int i = 0; i < NT / 8; i++) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = *reinterpret_cast<const uint4*>(vb + pr_at<RB>(rows4[j], gl + 8 * i));
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const unsigned a = (&v[0].x)[w], b = (&v[1].x)[w], d = (&v[2].x)[w], e = (&v[3].x)[w];
          put(8 * i + 2 * w, __byte_perm(a, b, 0x5410), __byte_perm(d, e, 0x5410));
          put(8 * i + 2 * w + 1, __byte_perm(a, b, 0x7632), __byte_perm(d, e, 0x7632));
        }
      }
    } else if constexpr (BITS == 8) {
      constexpr int NW = DP >= 128 ? 4 : 2;                              // words of a piece
#pragma unroll
      for (int i = 0; i < NT / (4 * NW); i++) {
        unsigned v[4][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if constexpr (NW == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(vb + pr_at<RB>(rows4[j], gl + 8 * i));
            v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(vb + pr_at<RB>(rows4[j], gl >> 1) + 8 * (gl & 1));
            v[j][0] = x.x; v[j][1] = x.y;
          }
        }
#pragma unroll
        for (int w = 0; w < NW; w++) {
          const unsigned x0 = __byte_perm(v[0][w], v[1][w], 0x5140) ^ 0x80808080u, x1 = __byte_perm(v[0][w], v[1][w], 0x7362) ^ 0x80808080u;
          const unsigned z0 = __byte_perm(v[2][w], v[3][w], 0x5140) ^ 0x80808080u, z1 = __byte_perm(v[2][w], v[3][w], 0x7362) ^ 0x80808080u;
          const int t = 4 * (NW * i + w);
          put(t, pa_bytes<0x4140>(x0), pa_bytes<0x4140>(z0)); put(t + 1, pa_bytes<0x4342>(x0), pa_bytes<0x4342>(z0));
          put(t + 2, pa_bytes<0x4140>(x1), pa_bytes<0x4140>(z1)); put(t + 3, pa_bytes<0x4342>(x1), pa_bytes<0x4342>(z1));
        }
      }
    } else {
      constexpr int NW = DP / 64;                                        // words of a lane's piece: 8 values each
      unsigned v[4][NW];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if constexpr (NW == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(vb + pr_at<RB>(rows4[j], gl));
          v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
        } else if constexpr (NW == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(vb + pr_at<RB>(rows4[j], gl >> 1) + 8 * (gl & 1));
          v[j][0] = x.x; v[j][1] = x.y;
        } else {
          v[j][0] = *reinterpret_cast<const unsigned*>(vb + pr_at<RB>(rows4[j], gl >> 2) + 4 * (gl & 3));
        }
      }
#pragma unroll
      for (int w = 0; w < NW; w++) {
        const int n16 = hd / 16, at = min((gl * NW + w) >> 1, n16 - 1);  // beyond the head the codes' columns are dropped
        unsigned t4[4];
#pragma unroll
        for (int j = 0; j < 4; j++) t4[j] = sc[128 + S::SUB + rows4[j] * n16 + at];
        const unsigned ta = pa_pair(t4[0], t4[1]), tb = pa_pair(t4[2], t4[3]);
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
          const unsigned x = __byte_perm(v[0][w], v[1][w], hf ? 0x7632 : 0x5410), z = __byte_perm(v[2][w], v[3][w], hf ? 0x7632 : 0x5410);
#pragma unroll
          for (int j = 0; j < 4; j++) put(8 * w + 4 * hf + j, pa_nibbles(x, j, ta), pa_nibbles(z, j, tb));
        }
      }
    }
  }

  // ---------------------------------------------------------------- the warps' results joined, in the warps' order
  __pipeline_wait_prior(0);
#pragma unroll
  for (int i = 0; i < NR; i++) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (cl == 0) s_ml[warp][gl + 8 * i] = make_float2(m[i], l[i]);
  }
  __syncthreads();                                                       // the rings are free: sums [warp][row][value]
  float* sums = reinterpret_cast<float*>(pr_smem);
#pragma unroll
  for (int t = 0; t < NT; t++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int d = pr_vdim<BITS, DP>(t, 2 * cl + j);
      if (R16) {
        sums[(warp * NROW + gl) * DP + d] = o[t][j];
        sums[(warp * NROW + gl + 8) * DP + d] = o[t][2 + j];
      } else {
        sums[(warp * NROW + gl) * DP + d] = o[t][j] + o[t][2 + j];
      }
    }
  __syncthreads();
  for (int i = tid; i < rn * hd; i += 32 * PR_WARPS) {
    const int r = i / hd, d = i % hd;
    float M = -INFINITY, L = 0.f, a = 0.f;
#pragma unroll
    for (int w = 0; w < PR_WARPS; w++) M = fmaxf(M, s_ml[w][r].x);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < PR_WARPS; w++) {
      const float2 x = s_ml[w][r];
      const float fw = pa_ex2(x.x - ref);
      L += x.y * (x.x == -INFINITY ? (x.y == x.y ? 0.f : 1.f) : fw);     // a warp that saw nothing has a zero, or a NaN that counts
      a += sums[(w * NROW + r) * DP + d] * (x.x == -INFINITY ? 1.f : fw);
    }
    if (c.nsplit > 1) {
      c.acc[rec(r) * hd + d] = a;
      if (d == 0) c.ml[rec(r)] = make_float2(M, L);
    } else {
      const int t = sq.q0 + (r0 + r) / c.group, h = kvh * c.group + (r0 + r) % c.group;
      c.out[(size_t)t * c.ldo + (size_t)h * hd + d] = L == 0.f ? 0.f : a / L;
    }
  }
}

// The splits' results joined in their order: a block per (sequence, kv head, row), a thread per value.
__global__ void __launch_bounds__(256) rows_join_kernel(const __grid_constant__ PaCall c, int per_head) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int r = blockIdx.x % per_head, kvh = blockIdx.x / per_head % c.g.kvh, seq = blockIdx.x / per_head / c.g.kvh, d = threadIdx.x;
  const WvSeq sq = wv_seq(c.b, c.g.page, seq, nullptr);
  const int nrows = (sq.q1 - sq.q0) * c.group;
  if (r >= nrows || nrows > c.rows_most || d >= c.g.hd) return;
  pa_join(c, blockIdx.x, sq.q0 + r / c.group, kvh * c.group + r % c.group, d);
}

template <int BITS, int DP, bool R16>
static cudaError_t rows_go(const PaCall& c, int tiles, cudaStream_t st) {
  using S = PrShape<BITS, DP>;
  constexpr size_t sums = (size_t)PR_WARPS * (R16 ? 16 : 8) * DP * 4, ring = (size_t)PR_WARPS * S::NST * S::STAGE;
  constexpr size_t smem = sums > ring ? sums : ring;
  auto kern = attn_rows_kernel<BITS, DP, R16>;
  static unsigned long long attr_mask = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !(attr_mask & (1ull << dev))) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    if (dev < 64) attr_mask |= 1ull << dev;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  cfg.gridDim = dim3((unsigned)(c.b.num_seqs * tiles * c.g.kvh), (unsigned)c.nsplit); cfg.blockDim = dim3(32 * PR_WARPS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, c);
}
template <int BITS>
static cudaError_t rows_pick(const PaCall& c, bool r16, int tiles, cudaStream_t st) {
  if (c.g.hd <= 64) return r16 ? rows_go<BITS, 64, true>(c, tiles, st) : rows_go<BITS, 64, false>(c, tiles, st);
  if (c.g.hd <= 128) return r16 ? rows_go<BITS, 128, true>(c, tiles, st) : rows_go<BITS, 128, false>(c, tiles, st);
  return r16 ? rows_go<BITS, 256, true>(c, tiles, st) : rows_go<BITS, 256, false>(c, tiles, st);
}

int wv_launch_attn_paged(const WvKvPages& kv, const WvKvBatch& b, const float* dq, int ldq, float* dout, int ldo, int heads, float scale,
                         int window, cudaStream_t st) {
  PaCall c = {};
  c.g = wv_kv_geom(kv);
  c.b = b;
  c.q = dq; c.ldq = ldq; c.out = dout; c.ldo = ldo;
  c.heads = heads; c.group = heads / c.g.kvh;
  c.scale = scale * 1.4426950408889634f;
  c.window = window;
  c.err = wv_paged_err_ptr();
  // Up to 32 rows (tokens x query heads of a kv head) a sequence is taken 8 or 16 rows at a time, beyond in tiles of 128.
  const long long most = (long long)b.max_q * c.group;
  c.rows_most = c.g.hd <= 128 ? 32 : INT_MAX;
  const bool alike = (long long)b.num_seqs * b.max_q == b.total_q;       // every sequence has max_q new tokens
  const bool chunk = most > c.rows_most, rows = !chunk || !alike;
  if ((long long)b.total_q * heads > INT_MAX) { wv_set_error("wv_attn_paged_dev: %d rows of %d heads are too many", b.total_q, heads); return WV_ESHAPE; }
  // what a sequence's new tokens can see together
  const long long keys = window > 0 && (long long)window + b.max_q + 16 < b.max_kv ? (long long)window + b.max_q + 16 : b.max_kv;
  const int sms = wv_sm_count();
  if (rows) {
    const long long top = chunk ? c.rows_most : most;
    const bool r16 = top > 8;
    const long long tiles = (top + (r16 ? 15 : 7)) / (r16 ? 16 : 8), per_head = tiles * (r16 ? 16 : 8);
    const long long blocks = (long long)b.num_seqs * tiles * c.g.kvh, want = 2LL * sms;
    if (blocks * (r16 ? 16 : 8) > INT_MAX) { wv_set_error("wv_attn_paged_dev: %d sequences are too many", b.num_seqs); return WV_ESHAPE; }
    long long per = (keys * blocks + want - 1) / want;
    per = (per + 63) & ~63LL;
    if (per < 64) per = 64;
    if (per > 1024) per = 1024;
    if (per < keys / 8192) per = (keys / 8192 + 63) & ~63LL;
    const long long ns = keys > per ? (keys + per - 1) / per : 1;
    PaCall r = c;
    r.per = (int)per; r.nsplit = (int)ns;
    WvLease lease;
    if (ns > 1) {
      const size_t n = (size_t)(b.num_seqs * c.g.kvh) * per_head * ns;
      if (const int rc = wv_lease(lease, n * (2 + c.g.hd), st, "wv_attn_paged_dev: the splits' results")) return rc;
      r.ml = reinterpret_cast<float2*>(lease.p);
      r.acc = lease.p + 2 * n;
    }
    cudaError_t e = kv.bits == 16 ? rows_pick<16>(r, r16, (int)tiles, st) : kv.bits == 8 ? rows_pick<8>(r, r16, (int)tiles, st) : rows_pick<4>(r, r16, (int)tiles, st);
    if (e == cudaSuccess && ns > 1) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at[1];
      cfg.gridDim = dim3((unsigned)(b.num_seqs * c.g.kvh * per_head)); cfg.blockDim = dim3((c.g.hd + 31) & ~31); cfg.stream = st;
      at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = at; cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, rows_join_kernel, r, (int)per_head);
    }
    if (e != cudaSuccess) { wv_set_error("wv_attn_paged_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA; }
  }
  return chunk ? wv_launch_attn_chunk(c, kv.bits, keys, alike, st) : WV_OK;
}
