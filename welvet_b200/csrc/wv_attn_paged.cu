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
// (cp.async, 9 to 17 KB in flight a warp, no barrier but its own), turns codes into float16 as it reads them, and keeps maximum,
// divisor and the weighted sum in registers. Which 8 or 16 values of a row a lane reads is chosen so that they are neighbours in
// memory: the order of the products does not matter for K, and for V it only decides which output a lane holds. Rows lie in the
// ring with their 16-byte pieces permuted so that both reading patterns are free of bank conflicts.
//
// Four warps a block and three blocks an SM (two with 16-bit rows of 128 or 16 query rows, see pr_blocks), so that one block's start (three
// dependent loads: lengths, page numbers, rows) runs beside another's keys. The keys of a sequence are split over blocks; the splits
// leave {M, divisor, sums} and a second kernel joins them in order, so results do not depend on who ran first.
//
// Measured: one token over 2049 positions (32 heads, 8 kv heads of 128, 16 bits) 10 us; over 131000 positions in 4 bits (64 heads) 72 us,
// 2.3 TB/s of codes and scales; 64 tokens over up to 8192 positions in 8 bits 130 us, 4.3 TB/s; 16 x 5 tokens over 3000, heads of 64 in
// 16 bits, 29 us. Neither DRAM (32 and 54 %) nor issue (0.55 a cycle and scheduler) is full in the long ones: what bounds them is latency
// within a warp, one dependent chain a group of 16 keys (535 instructions in 4 bits, 460 in 8 bits) with 2.8 warps a scheduler to
// hide it. A fourth block (q's fragments out of shared memory, 128 registers) issued no more and took 79 and 191 us.
#include "wv_attn_paged.cuh"
#include "wv_tma_common.cuh"
#include "wv_lease.h"
#include "wv_dev_hooks.h"
#include <algorithm>
#include <type_traits>

int wv_sm_count();

#define PR_WARPS 4
#define PR_CHAIN 40           // products that a warp adds to its sums at most, see rows_per_split
// The running maximum is raised only when a logit is 2^7 above it (the sums, 64 registers a lane, are multiplied each time), so weights
// reach 2^7 and carry 2^6 instead of 2^13: at most 2^14, and 2^-30 of that is still there.
#define PR_LIFT 6.f
#define PR_SLACK 7.f
#define PR_FAR 10u            // value scales up to 2^10 apart keep 20 bits

template <int BITS, int DP> struct PrShape {
  static constexpr int RB = DP * BITS / 8;                               // bytes of a row in the ring
  static constexpr int SUB = BITS == 4 ? DP : 0;                         // bytes of the sub-scales of 16 keys
  static constexpr int STAGE = 32 * RB + 128 + 2 * SUB;                  // K rows, V rows, 2 x 16 scales, sub-scales
  static constexpr int NCP = (RB + 31) / 32;                             // copies of 16 bytes that a lane makes for K's 16 rows (and for V's)
};

// Blocks an SM: three where the registers allow it (up to 8 rows of 128 values). wv_launch_attn_paged splits the keys over as many.
__host__ __device__ constexpr int pr_blocks(int bits, int dp, bool r16) {
  return dp == 256 && (bits == 16 || r16) ? 1 : !r16 && (dp == 64 || (dp == 128 && bits < 16)) ? 3 : 2;
}
// The keys that make a warp's chains of products PR_CHAIN long.
__host__ __device__ constexpr int pr_stretch(bool r16) { return 16 * PR_WARPS * (r16 ? PR_CHAIN / 2 : PR_CHAIN); }
// And the stages of a warp's ring in what they leave.
template <int BITS, int DP, bool R16> struct PrFit {
  static constexpr int STAGE = PrShape<BITS, DP>::STAGE;
  static constexpr int BLOCKS = pr_blocks(BITS, DP, R16);
  static constexpr int FIT = (BLOCKS == 3 ? 35 * 512 : 25 * 1024) / STAGE;
  static constexpr int NST = FIT < 2 ? 2 : (FIT > 8 ? 8 : FIT);
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
__device__ __forceinline__ void pr_copy(unsigned dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
template <int N> __device__ __forceinline__ void pr_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void pr_mma(float (&d)[4], const uint4& a, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pr_mma0(float (&d)[4], const uint4& a, unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
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

// EXACT: head_dim is DP, known at compile time; otherwise it is smaller and what lies beyond it is zero. SHARED: a part of wv_attn_shared_dev.
template <int BITS, int DP, bool R16, bool EXACT, bool SHARED>
__global__ void __launch_bounds__(32 * PR_WARPS, PrFit<BITS, DP, R16>::BLOCKS) attn_rows_kernel(const __grid_constant__ PaCall c) {
  using S = PrShape<BITS, DP>;
  constexpr int RB = S::RB, KS = DP / 16, NT = DP / 8, NROW = R16 ? 16 : 8, NST = PrFit<BITS, DP, R16>::NST;
  constexpr bool QREG = KS * (R16 ? 8 : 4) <= 32;                        // q fragments in registers, or read from shared memory each time
  extern __shared__ __align__(128) unsigned char pr_smem[];
  __shared__ uint4 s_qf[(R16 ? 2 : 1) * KS * 32];
  __shared__ float2 s_ml[PR_WARPS][NROW];
  __shared__ unsigned s_qmax[NROW];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, cl = lane & 3;
  unsigned char* ring = pr_smem + warp * NST * S::STAGE;
  if (tid < NROW) s_qmax[tid] = 0;
  const unsigned one = c.one;
  const int hd = EXACT ? DP : c.g.hd, n16 = hd / 16, code = EXACT ? RB : c.g.code;
  if (!EXACT) {                                                          // what lies beyond the head stays zero
    for (int i = tid * 16; i < PR_WARPS * NST * S::STAGE; i += 32 * PR_WARPS * 16) *reinterpret_cast<uint4*>(pr_smem + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // SHARED: blocks in one row, a part's splits one after the other
  const bool own = SHARED && blockIdx.x >= c.split;
  const int nsplit = SHARED && own ? c.own_nsplit : c.nsplit, slot0 = SHARED && own ? c.own_slot0 : c.slot0;
  const unsigned mine = SHARED ? (own ? gridDim.x - c.split : c.split) / (unsigned)nsplit : 0u, at = SHARED ? blockIdx.x - (own ? c.split : 0u) : 0u;
  const int sp = SHARED ? (int)(at / mine) : blockIdx.y;
  const unsigned flat = SHARED ? at - sp * mine : c.first + blockIdx.x, of_head = flat / (unsigned)c.g.kvh;
  const int kvh = flat - of_head * c.g.kvh;
  int seq, tile, table, shared = 0;                                      // table: the sequence whose pages are read
  WvSeq sq;
  if (SHARED && !own) {                                                  // the rows of a group's sequences, all behind its shared keys
    PaGroup g;
    int q0, q1;
    if (!pa_find_group(c, of_head, NROW, flat == 0 && sp == 0 && warp == 0 ? c.err : nullptr, g, q0, q1, tile)) return;
    shared = pa_shared_keys(c, g, table);
    if (shared == 0) return;
    sq = WvSeq{q0, q1, shared, shared};
  } else {
    if (DP == 256 && !SHARED && c.tiles == 0) {                          // see wv_launch_attn_paged
      __shared__ int s_at[2];
      if (warp == 0) {
        pa_find(c, of_head, NROW, 0, flat == 0 && sp == 0 ? c.err : nullptr, seq, tile);
        if (lane == 0) { s_at[0] = seq; s_at[1] = tile; }
      }
      __syncthreads();
      seq = s_at[0]; tile = s_at[1];
      if (seq < 0) return;
    } else {
      const unsigned tiles = SHARED ? c.own_tiles : c.tiles;
      seq = of_head / tiles; tile = of_head - seq * tiles;
    }
    sq = wv_seq(c.b, c.g.page, seq, sp == 0 && kvh == 0 && tile == 0 ? c.err : nullptr);
    table = seq;
  }
  const int nrows = (sq.q1 - sq.q0) * c.group, r0 = tile * NROW;
  if (r0 >= nrows || nrows > c.rows_most) return;
  const int rn = min(NROW, nrows - r0);
  if (SHARED && own) shared = pa_shared_of(c, seq);
  int lo, hi, per = SHARED && own ? c.own_per : c.per;
  pa_range(sq, r0 / c.group, (r0 + rn - 1) / c.group, c.window, lo, hi);
  auto rec = [&](int r) {                                                // a row's split result
    if (SHARED) return ((size_t)(sq.q0 + (r0 + r) / c.group) * (c.group * c.g.kvh) + kvh * c.group + (r0 + r) % c.group) * c.nslots + slot0 + sp;
    return ((size_t)blockIdx.x * c.kept + r) * c.nsplit + sp;
  };
  if (SHARED) {
    if (!own) {
      hi = min(hi, shared);
    } else {
      lo = max(lo, shared);
      // planned for what lies behind the longest prefix; where less is shared the splits are longer (and go in stretches, below)
      if (hi > lo) per = max(per, ((hi - lo + nsplit - 1) / nsplit + 63) & ~63);
      if (shared == 0 && sp == 0)                                        // nobody else writes these rows' results of part 1
        for (int i = tid; i < rn * slot0; i += 32 * PR_WARPS) c.ml[rec(i / slot0) - slot0 + i % slot0] = make_float2(-INFINITY, 0.f);
    }
  }
  const unsigned first = (unsigned)lo + (unsigned)sp * (unsigned)per;
  const int k0 = (int)min(first, (unsigned)hi);
  int k1 = min(hi, k0 + per);                                            // this block's keys; k0 is a multiple of 16 if there are any
  if (k0 >= k1) {
    if (SHARED || c.nsplit > 1) { if (tid < rn) c.ml[rec(tid)] = make_float2(-INFINITY, 0.f); }
    else for (int i = tid; i < rn * hd; i += 32 * PR_WARPS) {            // rows that see nothing
      const int r = i / hd, t = sq.q0 + (r0 + r) / c.group, h = kvh * c.group + (r0 + r) % c.group;
      c.out[(size_t)t * c.ldo + (size_t)h * hd + i % hd] = 0.f;
    }
    return;
  }

  // SHARED: a split that is longer than was planned, or that the scratch made long, goes in stretches, whose sums are joined in float32: its chains of products
  // are as short as any other's. 16 sequences of 131072 keys (64 heads over 8 of 128, 8 bits) of which all could be shared and nothing is take 2180 us so, 2010 in one
  // chain, whose sums were off by up to 7 times as much; a second set of sums beside the first would take 64 registers.
  __shared__ float2 s_all[SHARED ? 2 : 1][NROW];                         // {M, divisor} of the stretches before; read while the next turn's are written
  __shared__ int s_end;
  int turn = 0;
  if (SHARED) {
    if (tid == 0) s_end = k1;
    k1 = min(k1, k0 + pr_stretch(R16));
  }
  // ---------------------------------------------------------------- the warp's groups of 16 keys: k0 / 16 + warp, + PR_WARPS, ...
  int g0 = k0 / 16 + warp, ng = ((k1 + 15) / 16 - g0 + PR_WARPS - 1) / PR_WARPS;
  // A lane's copies of a group's K (or V) rows: the source is contiguous, the place in the ring the same in every stage.
  unsigned dst[S::NCP];
#pragma unroll
  for (int i = 0; i < S::NCP; i++) { const int at = (lane + 32 * i) * 16; dst[i] = smem_u32(ring) + pr_at<RB>(at / RB, at % RB / 16); }
  // Scales (lanes 0-3 of K, 4-7 of V) and sub-scales (the next n16 lanes of K, then of V): offset in the block, bytes a slot, place.
  int xo = 0, xm = 4;
  unsigned xd = 0xffffffffu;
  if (lane < 8) { xo = (lane < 4 ? c.g.kscale : c.g.vscale) + 16 * (lane & 3); xd = smem_u32(ring) + 32 * RB + 16 * lane; }
  else if (BITS == 4 && DP <= 128 && lane < 8 + 2 * n16) {
    const int j = lane - 8, v = j >= n16;
    xo = (v ? c.g.vsub : c.g.ksub) + 16 * (v ? j - n16 : j); xm = n16; xd = smem_u32(ring) + 32 * RB + 128 + (v ? S::SUB : 0) + 16 * (v ? j - n16 : j);
  }
  // 32 of the warp's groups at a time, a lane each: where the block is (-1: not in the pool), and the slot in it
  long long blk = 0;
  int slots = 0;
  unsigned bad = 0;                                                      // bit it & 31: the group's page is outside the pool
  int stage_in = 0;                                                      // of the next group to be copied
  auto start = [&](int it) {
    if ((it & 31) == 0) {
      const int key = (g0 + (it + lane) * PR_WARPS) * 16, at = key / c.g.page;
      int id = it + lane < ng ? c.b.pages[(size_t)table * c.b.table_stride + at] : 0;
      if (id < 0 || id >= c.g.num_pages) { wv_paged_report(c.err, WV_PAGED_PAGE); id = -1; }
      blk = id < 0 ? -1LL : ((long long)id * c.g.kvh + kvh) * c.g.block;
      slots = key - at * c.g.page;
    }
    const long long at = __shfl_sync(0xffffffffu, blk, it & 31);
    const int slot = __shfl_sync(0xffffffffu, slots, it & 31);
    if (it < ng) {
      const unsigned so = (unsigned)(stage_in * S::STAGE);
      const int have = at < 0 ? 0 : min(16, k1 - (g0 + it * PR_WARPS) * 16);      // keys of the group that exist; the rest is zeros
      bad = (bad & ~(1u << (it & 31))) | (unsigned)(at < 0) << (it & 31);
      const unsigned char* block = c.g.pool + (at < 0 ? 0 : at);
      const unsigned char* ks = block + slot * code;
      const unsigned char* vs = ks + (size_t)c.g.page * code;
      if (EXACT && have == 16) {
#pragma unroll
        for (int i = 0; i < S::NCP; i++) {
          if (16 * RB / 16 % 32 == 0 || lane + 32 * i < 16 * RB / 16) {
            pr_copy(dst[i] + so, ks + 16 * lane + 512 * i);
            pr_copy(dst[i] + so + 16 * RB, vs + 16 * lane + 512 * i);
          }
        }
      } else {
        constexpr int CH = BITS == 4 ? 8 : 16;                           // 4-bit rows are multiples of 8 bytes
        for (int a = lane * CH; a < 16 * code; a += 32 * CH) {
          const int r = a / code, o = a - r * code;
          const unsigned d = smem_u32(ring) + so + pr_at<RB>(r, o / 16) + (o & 15);
          const int n = r < have ? CH : 0;
          if (CH == 16) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(ks + (n ? a : 0)), "r"(n) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + 16 * RB), "l"(vs + (n ? a : 0)), "r"(n) : "memory");
          } else {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(d), "l"(ks + (n ? a : 0)), "r"(n) : "memory");
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(d + 16 * RB), "l"(vs + (n ? a : 0)), "r"(n) : "memory");
          }
        }
      }
      if (xd != 0xffffffffu) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(xd + so), "l"(block + xo + slot * xm), "r"(have ? 16 : 0) : "memory");
      if (BITS == 4 && DP == 256)
        for (int i = lane; i < 2 * n16; i += 32) {
          const int v = i >= n16, j = v ? i - n16 : i;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(ring) + so + 32 * RB + 128 + (v ? S::SUB : 0) + 16 * j),
                       "l"(block + (v ? c.g.vsub : c.g.ksub) + slot * n16 + 16 * j), "r"(have ? 16 : 0) : "memory");
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_in = stage_in + 1 == NST ? 0 : stage_in + 1;
  };
#pragma unroll
  for (int i = 0; i < NST - 1; i++) start(i);

  // ---------------------------------------------------------------- q: a power of two for each row, then two float16 pieces, as fragments
  constexpr int NR = R16 ? 2 : 1;
  const float* qrow[NR];                                                 // of the lane's rows
  int plast[NR], where[NR];                                              // the last position that they see; token and head as an offset in out
#pragma unroll
  for (int i = 0; i < NR; i++) {
    const int r = r0 + min(gl + 8 * i, rn - 1), tok = r / c.group, h = kvh * c.group + r - tok * c.group;
    qrow[i] = c.q + (size_t)(sq.q0 + tok) * c.ldq + (size_t)h * hd;
    plast[i] = sq.p0 + tok;
    where[i] = h * hd;
  }
  float qv[NR][KS / PR_WARPS][4];                                        // the lane's fragment values of steps warp, warp + 4, ...
  {
    unsigned m[NR] = {};
#pragma unroll
    for (int k = 0; k < KS / PR_WARPS; k++)
#pragma unroll
      for (int i = 0; i < NR; i++) {
        const bool on = gl + 8 * i < rn;
        if constexpr (BITS == 4) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int d = pr_kdim<BITS, DP>(warp + PR_WARPS * k, cl, e);
            qv[i][k][e] = on && d < hd ? qrow[i][d] : 0.f;
          }
        } else {
          const int d = pr_kdim<BITS, DP>(warp + PR_WARPS * k, cl, 0);   // four neighbours
          const float4 v = on && d < hd ? *reinterpret_cast<const float4*>(qrow[i] + d) : make_float4(0.f, 0.f, 0.f, 0.f);
          qv[i][k][0] = v.x; qv[i][k][1] = v.y; qv[i][k][2] = v.z; qv[i][k][3] = v.w;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) { const unsigned u = __float_as_uint(qv[i][k][e]) & 0x7fffffffu; if (u < 0x7f800000u) m[i] = max(m[i], u); }
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NR; i++) {
      m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], 1));
      m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], 2));
      if (cl == 0) atomicMax(&s_qmax[gl + 8 * i], m[i]);
    }
    __syncthreads();
  }
  float qinv[NR], qf[NR];
#pragma unroll
  for (int i = 0; i < NR; i++) {
    const int qe = min(max((int)(s_qmax[gl + 8 * i] >> 23) - 127 - 13, -100), 114);      // max |q| 2^-qe in [2^13, 2^14)
    qinv[i] = __uint_as_float((unsigned)(127 - qe) << 23);
    qf[i] = c.scale * __uint_as_float((unsigned)(127 + qe) << 23);
  }
#pragma unroll
  for (int k = 0; k < KS / PR_WARPS; k++) {
    unsigned h_[NR][2], l_[NR][2];                                       // [row g, row g + 8][k half]
#pragma unroll
    for (int i = 0; i < NR; i++)
#pragma unroll
      for (int p = 0; p < 2; p++) {
        float x = qv[i][k][2 * p], z = qv[i][k][2 * p + 1];
        x = x - x == 0.f ? x * qinv[i] : NAN;                            // not finite: the row's sums are NaN
        z = z - z == 0.f ? z * qinv[i] : NAN;
        h_[i][p] = pa_pack(x, z);
        const float2 b = pa_unpack(h_[i][p]);
        l_[i][p] = pa_pack(x - b.x, z - b.y);
      }
    const int at = (warp + PR_WARPS * k) * 32 + lane;
    if constexpr (R16) {
      s_qf[at] = make_uint4(h_[0][0], h_[1][0], h_[0][1], h_[1][1]);
      s_qf[KS * 32 + at] = make_uint4(l_[0][0], l_[1][0], l_[0][1], l_[1][1]);
    } else {
      s_qf[at] = make_uint4(h_[0][0], l_[0][0], h_[0][1], l_[0][1]);
    }
  }
  __syncthreads();
  const int pmin = sq.p0 + r0 / c.group, pmax = sq.p0 + (r0 + rn - 1) / c.group;
  for (;;) {
  uint4 qr[QREG ? (R16 ? 2 : 1) * KS : 1];
  if constexpr (QREG) {
#pragma unroll
    for (int i = 0; i < (R16 ? 2 : 1) * KS; i++) qr[i] = s_qf[i * 32 + lane];
  }
  auto qfrag = [&](int i) -> uint4 { if constexpr (QREG) return qr[i]; else return s_qf[i * 32 + lane]; };

  float o[NT][4], m[NR], l[NR];
#pragma unroll
  for (int t = 0; t < NT; t++) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
#pragma unroll
  for (int i = 0; i < NR; i++) { m[i] = -INFINITY; l[i] = 0.f; }
  // where the lane reads K (row gl) and V (rows 2 cl, 2 cl + 1) in a stage; 8 rows further on lie 8 RB bytes further
  constexpr int NKO = RB >= 64 ? RB / 64 : 1;
  unsigned kofs[NKO], vofs[2];
#pragma unroll
  for (int i = 0; i < NKO; i++) kofs[i] = RB == 32 ? pr_at<RB>(gl, cl >> 1) + 8 * (cl & 1) : pr_at<RB>(gl, cl + 4 * i);
#pragma unroll
  for (int i = 0; i < 2; i++)
    vofs[i] = 16 * RB + (RB >= 128 ? pr_at<RB>(2 * cl + i, gl) : RB == 64 ? pr_at<RB>(2 * cl + i, gl >> 1) + 8 * (gl & 1) : pr_at<RB>(2 * cl + i, gl >> 2) + 4 * (gl & 3));
  unsigned erun = 37;                                                    // exponent field of the largest value scale so far, at least 2^-90's
  int stage_out = 0;

  // One group of 16 keys out of a stage of the ring. PLAIN: every row sees all of them, and their value scales are near one another.
  auto group = [&](auto plain, unsigned sa, const unsigned char* st, int key, const unsigned (&vv)[4], bool far, bool there) {
    constexpr bool PLAIN = decltype(plain)::value;
    const unsigned char* sc = st + 32 * RB;
    // -------------------------------------------------------------- logits of two n-tiles of 8 keys, two chains of sums each
    float s[2][2][4];
#pragma unroll
    for (int n = 0; n < 2; n++) {
      [[maybe_unused]] const int r = gl + 8 * n;
      auto step = [&](int k, unsigned b0, unsigned b1) {
        if (k < 2) pr_mma0(s[n][k & 1], qfrag(R16 ? KS + k : k), b0, b1);
        else pr_mma(s[n][k & 1], qfrag(R16 ? KS + k : k), b0, b1);
        if (R16) pr_mma(s[n][k & 1], qfrag(k), b0, b1);                  // the small pieces first
      };
      if constexpr (BITS == 4 && DP == 64) {
        const uint2 w = lds64(sa + kofs[0] + n * 8 * RB);
        const unsigned t1 = sc[128 + r * n16 + min(cl, n16 - 1)];
        const PaSub t = pa_pair(t1, t1);
        step(0, pa_nibbles(w.x, 0, t, one), pa_nibbles(w.x, 1, t, one)); step(1, pa_nibbles(w.x, 2, t, one), pa_nibbles(w.x, 3, t, one));
        step(2, pa_nibbles(w.y, 0, t, one), pa_nibbles(w.y, 1, t, one)); step(3, pa_nibbles(w.y, 2, t, one), pa_nibbles(w.y, 3, t, one));
      } else {
#pragma unroll
        for (int i = 0; i < RB / 64; i++) {
          const uint4 v = lds128(sa + kofs[i] + n * 8 * RB);
          const unsigned w[4] = {v.x, v.y, v.z, v.w};
          if constexpr (BITS == 16) { step(2 * i, w[0], w[1]); step(2 * i + 1, w[2], w[3]); }
          if constexpr (BITS == 8) {
#pragma unroll
            for (int j = 0; j < 4; j++) { const unsigned x = w[j] ^ 0x80808080u; step(4 * i + j, pa_bytes<0x4140>(x), pa_bytes<0x4342>(x)); }
          }
          if constexpr (BITS == 4) {
            const int at = 2 * (cl + 4 * i);
            unsigned ta, tb;
            if constexpr (EXACT) {
              const unsigned both = *reinterpret_cast<const unsigned short*>(sc + 128 + r * n16 + at);
              ta = both & 255u; tb = both >> 8;
            } else {
              ta = at < n16 ? sc[128 + r * n16 + at] : 0u; tb = at + 1 < n16 ? sc[128 + r * n16 + at + 1] : 0u;
            }
            const PaSub t2[2] = {pa_pair(ta, ta), pa_pair(tb, tb)};
#pragma unroll
            for (int j = 0; j < 4; j++) {
              step(8 * i + 2 * j, pa_nibbles(w[j], 0, t2[j >> 1], one), pa_nibbles(w[j], 1, t2[j >> 1], one));
              step(8 * i + 2 * j + 1, pa_nibbles(w[j], 2, t2[j >> 1], one), pa_nibbles(w[j], 3, t2[j >> 1], one));
            }
          }
        }
      }
    }
    // -------------------------------------------------------------- weights of the lane's four keys 2c, 2c + 1, 2c + 8, 2c + 9
    const float2 k0_ = *reinterpret_cast<const float2*>(sc + 8 * cl), k1_ = *reinterpret_cast<const float2*>(sc + 32 + 8 * cl);
    float kk[NR][4];
#pragma unroll
    for (int i = 0; i < NR; i++) { kk[i][0] = k0_.x * qf[i]; kk[i][1] = k0_.y * qf[i]; kk[i][2] = k1_.x * qf[i]; kk[i][3] = k1_.y * qf[i]; }
    const float inv = __uint_as_float((254u - erun) << 23);
    float y[NR][4], f[4];
    bool seen[NR][4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int n = j >> 1, e = j & 1;
      f[j] = __uint_as_float(vv[j]) * inv;
      if (R16) {
        y[0][j] = (s[n][0][e] + s[n][1][e]) * kk[0][j];
        y[NR - 1][j] = (s[n][0][2 + e] + s[n][1][2 + e]) * kk[NR - 1][j];
      } else {
        y[0][j] = ((s[n][0][2 + e] + s[n][1][2 + e]) + (s[n][0][e] + s[n][1][e])) * kk[0][j];
      }
      if (!PLAIN) {
        const int p = key + 8 * n + 2 * cl + e;
#pragma unroll
        for (int i = 0; i < NR; i++) {
          seen[i][j] = there && p <= plast[i] && p < k1 && (c.window == 0 || p > plast[i] - c.window);
          if (!seen[i][j]) y[i][j] = -INFINITY;
        }
      }
    }
    float mx[NR];
    bool up = false;
#pragma unroll
    for (int i = 0; i < NR; i++) {
      mx[i] = fmaxf(fmaxf(y[i][0], y[i][1]), fmaxf(y[i][2], y[i][3]));
      up |= mx[i] > m[i] + PR_SLACK;
    }
    if (__any_sync(0xffffffffu, up)) {
      float fac[NR];
#pragma unroll
      for (int i = 0; i < NR; i++) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        fac[i] = mx[i] > m[i] ? pa_ex2(m[i] - mx[i]) : 1.f;              // 0 while there was nothing
        m[i] = fmaxf(m[i], mx[i]);
        l[i] *= fac[i];
      }
#pragma unroll
      for (int t = 0; t < NT; t++) { o[t][0] *= fac[0]; o[t][1] *= fac[0]; o[t][2] *= fac[NR - 1]; o[t][3] *= fac[NR - 1]; }
    }
    uint4 ph, pl;
    unsigned* hh = reinterpret_cast<unsigned*>(&ph);
    unsigned* ll = reinterpret_cast<unsigned*>(&pl);
    float pw[NR][4];
#pragma unroll
    for (int i = 0; i < NR; i++) {
      float (&p)[4] = pw[i];
      const float off = !PLAIN && m[i] == -INFINITY ? 0.f : PR_LIFT - m[i];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        float e = pa_ex2(y[i][j] + off);
        p[j] = e * f[j];
        if (!PLAIN && !seen[i][j]) e = p[j] = 0.f;
        l[i] += e;
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
    [[maybe_unused]] const int rows4[4] = {2 * cl, 2 * cl + 1, 2 * cl + 8, 2 * cl + 9};
    if (!PLAIN && far) {                                                 // value by value in float32
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
      return;
    }
    if constexpr (BITS == 16) {
#pragma unroll
      for (int i = 0; i < NT / 8; i++) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = lds128(sa + vofs[j & 1] + (j >> 1) * 8 * RB + 128 * i);
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
            const uint4 x = lds128(sa + vofs[j & 1] + (j >> 1) * 8 * RB + 128 * i);
            v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
          } else {
            const uint2 x = lds64(sa + vofs[j & 1] + (j >> 1) * 8 * RB);
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
          const uint4 x = lds128(sa + vofs[j & 1] + (j >> 1) * 8 * RB);
          v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
        } else if constexpr (NW == 2) {
          const uint2 x = lds64(sa + vofs[j & 1] + (j >> 1) * 8 * RB);
          v[j][0] = x.x; v[j][1] = x.y;
        } else {
          v[j][0] = lds32(sa + vofs[j & 1] + (j >> 1) * 8 * RB);
        }
      }
      PaSub ta, tb;
#pragma unroll
      for (int w = 0; w < NW; w++) {
        if (w % 2 == 0) {                                                // a sub-scale serves two words
          const int at = EXACT ? (gl * NW + w) >> 1 : min((gl * NW + w) >> 1, n16 - 1);      // beyond the head the codes' columns are dropped
          unsigned t4[4];
#pragma unroll
          for (int j = 0; j < 4; j++) t4[j] = sc[128 + S::SUB + rows4[j] * n16 + at];
          ta = pa_pair(t4[0], t4[1]); tb = pa_pair(t4[2], t4[3]);
        }
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
          const unsigned x = __byte_perm(v[0][w], v[1][w], hf ? 0x7632 : 0x5410), z = __byte_perm(v[2][w], v[3][w], hf ? 0x7632 : 0x5410);
#pragma unroll
          for (int j = 0; j < 4; j++) put(8 * w + 4 * hf + j, pa_nibbles(x, j, ta, one), pa_nibbles(z, j, tb, one));
        }
      }
    }
  };
  const int seen_lo = c.window == 0 ? lo : max(lo, pmax - c.window + 1), seen_hi = min(pmin + 1, k1);         // what every row sees
  for (int it = 0; it < ng; it++) {
    pr_wait<NST - 2>();
    __syncwarp();                                                        // every lane has read the stage that is filled next
    start(it + NST - 1);
    const unsigned char* st = ring + stage_out * S::STAGE;
    const unsigned sa = smem_u32(ring) + stage_out * S::STAGE;
    stage_out = stage_out + 1 == NST ? 0 : stage_out + 1;
    const int key = (g0 + it * PR_WARPS) * 16;
    const bool there = !((bad >> (it & 31)) & 1u);
    const bool whole = key >= seen_lo && key + 16 <= seen_hi && there;
    const uint2 v0 = *reinterpret_cast<const uint2*>(st + 32 * RB + 64 + 8 * cl), v1 = *reinterpret_cast<const uint2*>(st + 32 * RB + 96 + 8 * cl);
    unsigned vv[4] = {v0.x, v0.y, v1.x, v1.y};
    // Most groups: all 16 value scales within PR_FAR powers of two below the largest so far, by one difference a scale and one vote.
    const unsigned least = (max(erun, PR_FAR + 37u) - PR_FAR) << 23, span = ((erun + 1u) << 23) - least;
    const bool near = max(max(vv[0] - least, vv[1] - least), max(vv[2] - least, vv[3] - least)) < span;
    bool easy = whole && __all_sync(0xffffffffu, near), far = false;
    if (!easy) {
      // the largest and smallest exponent among the 16 value scales; a scale of NaN has none, one below 2^-90 is nothing
      unsigned top = 0u, low = 255u << 23;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (!whole && key + 8 * (j >> 1) + 2 * cl + (j & 1) >= k1) vv[j] = 0u;
        const unsigned u = vv[j] < 0x7f800000u ? vv[j] : 0u;
        top = max(top, u);
        low = min(low, u < (37u << 23) ? 255u << 23 : u);
      }
      top = __reduce_max_sync(0xffffffffu, top) >> 23;
      low = __reduce_min_sync(0xffffffffu, low) >> 23;
      if (top > erun) {
        const float down = __uint_as_float((unsigned)max(127 - (int)(top - erun), 0) << 23);
        erun = top;
#pragma unroll
        for (int t = 0; t < NT; t++) { o[t][0] *= down; o[t][1] *= down; o[t][2] *= down; o[t][3] *= down; }
      }
      far = low + PR_FAR < erun;
      easy = whole && !far;
    }
    if (easy) group(std::true_type(), sa, st, key, vv, false, true);
    else group(std::false_type(), sa, st, key, vv, far, there);
  }

  // ---------------------------------------------------------------- the warps' results joined, in the warps' order
  pr_wait<0>();
  const float beta = __uint_as_float(erun << 23);
#pragma unroll
  for (int i = 0; i < NR; i++) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (cl == 0) s_ml[warp][gl + 8 * i] = make_float2(m[i], l[i]);
  }
  __syncthreads();                                                       // the rings are free: sums [warp][row half][n-tile][lane], two values each
  float2* sums = reinterpret_cast<float2*>(pr_smem);
#pragma unroll
  for (int t = 0; t < NT; t++) {
    if (R16) {
      sums[((warp * NR + 0) * NT + t) * 32 + lane] = make_float2(o[t][0] * beta, o[t][1] * beta);
      sums[((warp * NR + NR - 1) * NT + t) * 32 + lane] = make_float2(o[t][2] * beta, o[t][3] * beta);
    } else {
      sums[(warp * NT + t) * 32 + lane] = make_float2((o[t][0] + o[t][2]) * beta, (o[t][1] + o[t][3]) * beta);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NR; i++) {
    const int r = gl + 8 * i;
    if (r >= rn) break;
    float M = -INFINITY, L = 0.f, fw[PR_WARPS];
#pragma unroll
    for (int w = 0; w < PR_WARPS; w++) M = fmaxf(M, s_ml[w][r].x);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < PR_WARPS; w++) {
      const float2 x = s_ml[w][r];
      fw[w] = x.x == -INFINITY ? (x.y == x.y ? 0.f : 1.f) : pa_ex2(x.x - ref);      // a warp that saw nothing has zeros, or NaN, which counts
      L += x.y * fw[w];
    }
    float* to;
    float scale = 1.f, before = 0.f;
    const bool more = SHARED && turn > 0;
    if (SHARED || c.nsplit > 1) {
      to = c.acc + rec(r) * hd;
      if (more) {                                                        // a lane's values of the stretches before are its own
        const float2 all = s_all[turn & 1][r];
        const float top = fmaxf(M, all.x), t0 = top == -INFINITY ? 0.f : top;
        before = all.x == -INFINITY ? (all.y == all.y ? 0.f : 1.f) : pa_ex2(all.x - t0);
        scale = M == -INFINITY ? (L == L ? 0.f : 1.f) : pa_ex2(M - t0);
        L = all.y * before + L * scale;
        M = top;
      }
      if (warp == 0 && cl == 0) {
        c.ml[rec(r)] = make_float2(M, L);
        if (SHARED) s_all[(turn + 1) & 1][r] = make_float2(M, L);
      }
    } else {
      to = c.out + (size_t)(sq.q0 + plast[i] - sq.p0) * c.ldo + where[i];
      scale = L == 0.f ? 0.f : 1.f / L;
    }
    for (int t4 = warp; t4 < NT / 4; t4 += PR_WARPS) {                   // four neighbouring values at a time, twice
      float v[2][4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        float x = 0.f, z = 0.f;
#pragma unroll
        for (int w = 0; w < PR_WARPS; w++) {
          const float2 s = sums[((w * NR + i) * NT + 4 * t4 + k) * 32 + lane];
          x += s.x * fw[w]; z += s.y * fw[w];
        }
        v[0][k] = x * scale; v[1][k] = z * scale;
      }
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const int d = pr_vdim<BITS, DP>(4 * t4, 2 * cl + j);
        if (d < hd) {
          float4 y = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
          if (more) {
            const float4 x = *reinterpret_cast<const float4*>(to + d);
            y.x += x.x * before; y.y += x.y * before; y.z += x.z * before; y.w += x.w * before;
          }
          *reinterpret_cast<float4*>(to + d) = y;
        }
      }
    }
  }
  if (!SHARED || k1 == s_end) break;
  turn++;
  g0 = k1 / 16 + warp; k1 = min(s_end, k1 + pr_stretch(R16)); ng = ((k1 + 15) / 16 - g0 + PR_WARPS - 1) / PR_WARPS;
  stage_in = 0;
  __syncthreads();                                                       // every warp has read the sums: the rings again
  if (!EXACT) {
    for (int i = tid * 16; i < PR_WARPS * NST * S::STAGE; i += 32 * PR_WARPS * 16) *reinterpret_cast<uint4*>(pr_smem + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < NST - 1; i++) start(i);
  }
}

// The splits' results joined in their order: a block per row (tokens x query heads) of the blocks of attn_rows_kernel, which took `nrow` each.
__global__ void __launch_bounds__(128) rows_join_kernel(const __grid_constant__ PaCall c, int nrow) {
  extern __shared__ float pr_w[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const unsigned block = blockIdx.x / c.kept, flat = c.first + block, of_head = flat / (unsigned)c.g.kvh;
  const int kvh = flat - of_head * c.g.kvh;
  int seq, tile;
  if (c.tiles == 0) {                                                    // each of the warps for itself
    pa_find(c, of_head, nrow, 0, nullptr, seq, tile);
    if (seq < 0) return;
  } else {
    seq = of_head / c.tiles; tile = of_head - seq * c.tiles;
  }
  const int r = tile * nrow + blockIdx.x - block * c.kept;
  const WvSeq sq = wv_seq(c.b, c.g.page, seq, nullptr);
  const int nrows = (sq.q1 - sq.q0) * c.group;
  if (r >= nrows || nrows > c.rows_most) return;
  const float inv = pa_join_weights(c, blockIdx.x, c.nsplit, pr_w);
  __syncthreads();
  pa_join_sums(c, blockIdx.x, c.nsplit, sq.q0 + r / c.group, kvh * c.group + r % c.group, pr_w, inv, threadIdx.x, 128);
}

// The same for the rows of wv_attn_shared_dev: a block for eight heads of a token, a warp each, four values a lane.
__global__ void __launch_bounds__(256) shared_join_kernel(const __grid_constant__ PaCall c) {
  extern __shared__ float pr_w[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int token = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.y * 8 + warp, heads = c.group * c.g.kvh;
  if (head >= heads) return;
  const size_t rec = (size_t)token * heads + head;
  float* w = pr_w + warp * c.nslots;
  const float inv = pa_join_weights(c, rec, c.nslots, w);                // of a row that belongs to nobody, too: its results are not used
  const int s = wv_seq_of_row(c.b, token);
  if (s >= c.b.num_seqs) return;
  const WvSeq q = wv_seq(c.b, c.g.page, s, nullptr);
  if (token < q.q0 || token >= q.q1) return;
  __syncwarp();
  const float* acc = c.acc + rec * c.nslots * c.g.hd;
  float* out = c.out + (size_t)token * c.ldo + (size_t)head * c.g.hd;
  for (int d = 4 * lane; d < c.g.hd; d += 128) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < c.nslots; s0 += 8) {
      float4 v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) v[u] = s0 + u < c.nslots && w[s0 + u] != 0.f ? *reinterpret_cast<const float4*>(acc + (size_t)(s0 + u) * c.g.hd + d) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < 8; u++) if (s0 + u < c.nslots) { const float f = w[s0 + u]; a.x += v[u].x * f; a.y += v[u].y * f; a.z += v[u].z * f; a.w += v[u].w * f; }
    }
    *reinterpret_cast<float4*>(out + d) = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  }
}

template <int BITS, int DP, bool R16, bool EXACT, bool SHARED>
static cudaError_t rows_go(const PaCall& c, int blocks, cudaStream_t st) {
  using S = PrShape<BITS, DP>;
  constexpr size_t sums = (size_t)PR_WARPS * (R16 ? 16 : 8) * DP * 4, ring = (size_t)PR_WARPS * PrFit<BITS, DP, R16>::NST * S::STAGE;
  constexpr size_t smem = sums > ring ? sums : ring;
  auto kern = attn_rows_kernel<BITS, DP, R16, EXACT, SHARED>;
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
  cfg.gridDim = SHARED ? dim3((unsigned)blocks) : dim3((unsigned)blocks, (unsigned)c.nsplit); cfg.blockDim = dim3(32 * PR_WARPS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, c);
}
template <int BITS, bool R16, bool SHARED>
static cudaError_t rows_pick(const PaCall& c, int blocks, cudaStream_t st) {
  if (c.g.hd == 64) return rows_go<BITS, 64, R16, true, SHARED>(c, blocks, st);
  if (c.g.hd == 128) return rows_go<BITS, 128, R16, true, SHARED>(c, blocks, st);
  if (c.g.hd < 64) return rows_go<BITS, 64, R16, false, SHARED>(c, blocks, st);
  if (c.g.hd < 128) return rows_go<BITS, 128, R16, false, SHARED>(c, blocks, st);
  return rows_go<BITS, 256, R16, false, SHARED>(c, blocks, st);
}
template <bool SHARED> static cudaError_t rows_any(const PaCall& c, int bits, bool r16, int blocks, cudaStream_t st) {
  return bits == 16 ? (r16 ? rows_pick<16, true, SHARED>(c, blocks, st) : rows_pick<16, false, SHARED>(c, blocks, st))
       : bits == 8 ? (r16 ? rows_pick<8, true, SHARED>(c, blocks, st) : rows_pick<8, false, SHARED>(c, blocks, st))
                   : (r16 ? rows_pick<4, true, SHARED>(c, blocks, st) : rows_pick<4, false, SHARED>(c, blocks, st));
}

// Splits of the keys: the number that fills 1, 2, .. 8 waves of the blocks that run at once and costs least, a wave being worth a
// warp's groups of 16 keys and some six more of start and end (2049 positions and eight blocks: 33 splits of 64; 131000: 55).
// The tensor core cuts instead of rounding as it adds, so the error grows with the products that a warp adds to its sums one
// after the other (two a group with 16 rows): 12 rows over 12000 keys in one chain of 376 were off by 6.7e-6, in chains of 40 by
// 7e-7; 131000 keys in chains of 38 by 9e-7. So no more than 40, at 2 us of 26 for the drafted tokens and 4 of 126 for the batch above.
static long long rows_per_split(long long keys, long long blocks, const WvKvGeom& g, int bits, bool r16) {
  const long long slots = (long long)wv_sm_count() * pr_blocks(bits, g.hd <= 64 ? 64 : g.hd <= 128 ? 128 : 256, r16);
  const long long longest = pr_stretch(r16);
  long long per = 64, cost = -1;
  for (long long w = 1; w <= 8; w++) {
    long long n = w * slots / blocks;
    if (n < 1) { if (w < 8) continue; n = 1; }
    long long p = std::min(((keys + n - 1) / n + 63) & ~63LL, longest);
    if (p < 64) p = 64;
    const long long m = keys > p ? (keys + p - 1) / p : 1, k = (blocks * m + slots - 1) / slots * (p / 64 + 6);
    if (cost < 0 || k < cost) { cost = k; per = p; }
  }
  return per;
}

int wv_launch_attn_paged(const WvKvPages& kv, const WvKvBatch& b, const float* dq, int ldq, float* dout, int ldo, int heads, float scale,
                         int window, cudaStream_t st) {
  PaCall c = {};
  c.g = wv_kv_geom(kv);
  c.b = b;
  c.q = dq; c.ldq = ldq; c.out = dout; c.ldo = ldo;
  c.group = heads / c.g.kvh;
  c.scale = scale * 1.4426950408889634f;
  c.window = window;
  c.one = 0x3c003c00u;
  c.err = wv_paged_err_ptr();
  // Up to 32 rows (tokens x query heads of a kv head) a sequence is taken 8 or 16 rows at a time, beyond in tiles of 128.
  const long long most = (long long)b.max_q * c.group;
  c.rows_most = c.g.hd <= 128 ? 32 : INT_MAX;
  // Where every sequence can have max_q new tokens they are expected to, and one kernel takes them all. They need not (the lengths are
  // the device's, and may be others in each replay of a graph): that kernel then takes the short ones too.
  const bool alike = (long long)b.num_seqs * b.max_q == b.total_q;
  const bool chunk = most > c.rows_most, rows = !chunk || !alike;
  if (!rows) c.rows_most = 0;
  if ((long long)b.total_q * heads > INT_MAX) { wv_set_error("wv_attn_paged_dev: %d rows of %d heads are too many", b.total_q, heads); return WV_ESHAPE; }
  // what a sequence's new tokens can see together
  const long long keys = window > 0 && (long long)window + b.max_q + 16 < b.max_kv ? (long long)window + b.max_q + 16 : b.max_kv;
  if (rows) {
    const long long top = chunk ? c.rows_most : most;
    const bool r16 = top > 8;
    const int nrow = r16 ? 16 : 8;
    const long long tiles = (top + nrow - 1) / nrow;
    // Heads beyond 128 come here with prompts as well. Beside short sequences most of the tiles that max_q allows for each are then empty
    // (and may be more than a grid holds): where total_q allows a quarter of them or less, a block looks its sequence up.
    const long long rows_tiles = (long long)b.num_seqs * tiles, full_tiles = (long long)b.total_q * c.group / nrow + b.num_seqs;
    const bool look = c.g.hd > 128 && full_tiles <= rows_tiles / 4;
    const long long blocks = (look ? full_tiles : rows_tiles) * c.g.kvh;
    if (blocks * nrow > INT_MAX) { wv_set_error("wv_attn_paged_dev: %d sequences are too many", b.num_seqs); return WV_ESHAPE; }
    long long per = rows_per_split(keys, blocks, c.g, kv.bits, r16);
    if (per < keys / 8192) per = (keys / 8192 + 63) & ~63LL;
    const long long ns = keys > per ? (keys + per - 1) / per : 1;
    PaCall r = c;
    r.per = (int)per; r.nsplit = (int)ns; r.tiles = look ? 0u : (unsigned)tiles; r.kept = (unsigned)(top < nrow ? top : nrow);
    // The splits' results of all rows may be more than a call should keep (a prompt of 8192 tokens and 16 heads of 256: 0.9 GB): the blocks
    // then go in parts of equal size, one after the other through the same scratch. A part holds 600 blocks of 16 rows or more up to 26
    // splits of the widest heads, so it still fills the chip.
    const long long bytes = (long long)r.kept * ns * (2 + c.g.hd) * 4, most_blocks = ns == 1 || bytes * blocks <= PA_SCRATCH ? blocks : std::max(PA_SCRATCH / bytes, 1LL);
    const long long parts = (blocks + most_blocks - 1) / most_blocks, part = (blocks + parts - 1) / parts;
    WvLease lease;
    if (ns > 1) {
      const size_t n = (size_t)part * r.kept * ns, sums = (2 * n + 3) & ~(size_t)3;      // the sums are stored 16 bytes at a time
      if (const int rc = wv_lease(lease, sums + n * c.g.hd, st, "wv_attn_paged_dev: the splits' results")) return rc;
      r.ml = reinterpret_cast<float2*>(lease.p);
      r.acc = lease.p + sums;
    }
    cudaError_t e = cudaSuccess;
    for (long long at0 = 0; at0 < blocks && e == cudaSuccess; at0 += part) {
      const int now = (int)std::min(part, blocks - at0);
      r.first = (unsigned)at0;
      e = rows_any<false>(r, kv.bits, r16, now, st);
      if (e != cudaSuccess || ns == 1) continue;
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute at[1];
      cfg.gridDim = dim3((unsigned)(now * r.kept)); cfg.blockDim = dim3(128); cfg.dynamicSmemBytes = (size_t)ns * 4; cfg.stream = st;
      at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[0].val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = at; cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, rows_join_kernel, r, nrow);
    }
    if (e != cudaSuccess) { wv_set_error("wv_attn_paged_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA; }
  }
  return chunk ? wv_launch_attn_chunk(c, kv.bits, keys, alike, st) : WV_OK;
}

// The shared keys of every group for all rows of its sequences (part 1), every sequence's own keys (part 2), and the two joined. Part 1
// runs on tcgen05 where a group has more than 32 rows of a kv head on average, part 2 where a sequence can have; otherwise 8 or 16 rows a pass.
#ifdef WV_DEV_HOOKS
static int g_sharing = 0;
extern "C" void wv_set_attn_sharing(int always) { g_sharing = always; }
#endif
// Splits of `tiles` key tiles for blocks of the chunk kernel: the number (up to `most`) that costs least in waves of blocks, each worth its key tiles and
// some four more of start and end.
static long long chunk_waves(long long blocks, long long tiles, long long n) {
  const long long sms = wv_sm_count();
  return (blocks * n + sms - 1) / sms * ((tiles + n - 1) / n + 4);
}
static long long chunk_splits(long long blocks, long long tiles, long long most) {
  long long best = 1, cost = -1;
  for (long long n = 1; n <= most && n <= tiles; n++) {
    const long long w = chunk_waves(blocks, tiles, n);
    if (cost < 0 || w < cost) { cost = w; best = n; }
  }
  return best;
}
// Does it pay to take the front keys apart? A pass of the kernel for few rows over a key costs 0.25 ps for each value of a kv head and eight query rows, 0.35 for sixteen
// (0.47 with heads beyond 128, which leave an SM half as many blocks).
//
// Up to 32 rows of a kv head a sequence, num_seqs - num_groups passes are saved. It costs two results a row written and joined (at 2 TB/s of their bytes: the
// join is short) and 6 us, or 12 where the front keys go to the chunk kernel, which takes that long to start. Of 186 shapes (2 to 48 sequences a group, 1 or 4 groups,
// 256 to 16384 shared tokens, 1 or 4 new ones, three layouts) this takes the faster way, or one within 5 %, in all but 6, and loses 27 % at most; e.g. us apart / not,
// 32 heads over 8 of 128 in 8 bits: 2 sequences x 16384 tokens 23.1 / 22.6, 48 x 1024 34.6 / 29.5, 48 x 4096 41.6 / 94.9, 48 x 16384 72 / 298.
//
// More rows fill tiles of their own, and reading the front once saves what the tiles of the sequences leave empty, no more: beside that rule both ways are then
// counted in waves of the chunk kernel's blocks, 4.5 us a key tile for 256 rows of a sequence (3.0 up to 128 of them) and 2.7 for 128 rows of a group or of one; a result
// of all rows at 3 TB/s (many of them are still in L2). Of 203 shapes (9 to 1024 new tokens, even, ragged, and beside single ones; 4 to 64 sequences) this takes
// the faster way, or one within 5 %, in all but 6, and loses 38 % at most; the rule above alone took the slower one in 82, by up to 2.2 times. Apart / not, as above: 16 x 16 tokens behind 16384
// 213 / 417, 16 x 32 behind 4096 139 / 126, 16 x 65 behind 16384 789 / 1143, 16 x 128 behind 1024 287 / 134.
// Wide heads likewise by tiles of sixteen rows: 64 x 1 token of 4 heads a kv head of 256 behind 8192 149 / 241, of 8 heads 253 / 244, 64 x 4 918 / 894; of 96 shapes none is
// slower by more than 5 % (43 by the first rule).
static bool sharing_pays(const WvKvBatch& b, int num_groups, long long front, const WvKvGeom& g, int group, long long each) {
#ifdef WV_DEV_HOOKS
  if (g_sharing) return true;
#endif
  const long long rows = (long long)b.max_q * group, first = each * group;           // of a sequence at most, of a group on average
  const bool wide = g.hd > 128, chunk = !wide && first > 32;
  const double result = (double)b.total_q * group * g.kvh * (g.hd + 2) * 2 * 4 / 2e6;  // of every row, written and read at 2 TB/s
  if (!wide) {
    const double saved = (double)(b.num_seqs - num_groups) * front * g.kvh * g.hd * (rows <= 8 ? 0.25e-6 : 0.35e-6 * ((rows + 15) / 16));
    const bool pays = saved > (chunk ? 12.0 : 6.0) + result;
    if (!pays || rows <= 32) return pays;
  }
  // as many sequences as total_q has room for have max_q new tokens, the others share what is left
  const long long many = std::max(1LL, std::min<long long>(b.num_seqs, b.total_q / b.max_q)), others = b.num_seqs - many;
  const long long rest = others > 0 ? (std::max(0LL, b.total_q - many * b.max_q) * group + others - 1) / others : 0;
  if (wide) {
    auto tiles = [](long long r) { return (double)((r + 15) / 16); };
    const double alone = rows <= 8 ? 0.25 * b.num_seqs : 0.47 * (many * tiles(rows) + others * tiles(rest));
    const double apart = rows <= 8 && first <= 8 ? 0.25 * num_groups : 0.47 * b.total_q * group / 16;
    return (alone - apart) * front * g.kvh * g.hd * 1e-6 > 8.0 + result;
  }
  const double narrow = 0.6 + 0.4 * g.hd / 128;
  auto few = [&](long long seqs, long long r, long long keys) { return (double)seqs * g.kvh * keys * g.hd * (r <= 8 ? 0.25e-6 : 0.35e-6 * ((r + 15) / 16)); };
  // wv_attn_paged_dev: planned for blocks that the bounds allow, and those that there are
  const bool alike = (long long)b.num_seqs * b.max_q == b.total_q;
  const long long blocks = (rows + 255) / 256, upto = (long long)b.total_q * group / 256 + b.num_seqs, all = (b.max_kv + 127LL) / 128;
  const long long n = chunk_splits((alike ? b.num_seqs * blocks : std::min(b.num_seqs * blocks, upto)) * g.kvh, all, 16);
  const long long there = (many * blocks + (rest > 32 ? others * ((rest + 255) / 256) : 0)) * g.kvh;
  double alone = 5 + chunk_waves(there, all, n) * (rows > 128 ? 4.5 : 3.0) * narrow;
  if (n > 1) alone += 2 + 0.65 * n * there * 256 * (g.hd + 2) * 2 * 4 / 2e6;
  if (others > 0 && rest <= 32) alone += 30 + few(others, rest, b.max_kv);
  // the front keys, and every sequence's own in tiles of 128 rows
  const long long fronts = (front + 127) / 128, owns = std::max((b.max_kv - front + 127) / 128, 1LL), sure = (rows + 127) / 128;
  const long long groups = num_groups * ((first + 127) / 128) * g.kvh, m = chunk_splits(groups, fronts, 64);
  const long long k = chunk_splits(std::min(b.num_seqs * sure, (long long)b.total_q * group / 128 + b.num_seqs) * g.kvh, owns, 64);
  const double apart = 8 + (chunk ? chunk_waves(groups, fronts, m) * 2.7 * narrow : few(num_groups, first, front)) +
                       chunk_waves((many * sure + others * ((rest + 127) / 128)) * g.kvh, owns, k) * 2.7 * narrow + 0.65 * result * ((chunk ? m : 1) + k);
  return apart < alone;
}
int wv_launch_attn_shared(const WvKvPages& kv, const WvKvBatch& b, const WvKvGroups& share, const float* dq, int ldq, float* dout, int ldo, int heads, float scale,
                          cudaStream_t st) {
  PaCall c = {};
  c.g = wv_kv_geom(kv);
  c.b = b;
  c.share = share;
  c.q = dq; c.ldq = ldq; c.out = dout; c.ldo = ldo;
  c.group = heads / c.g.kvh;
  c.scale = scale * 1.4426950408889634f;
  c.one = 0x3c003c00u;
  c.err = wv_paged_err_ptr();
  c.rows_most = INT_MAX;
  if (c.share.max_shared > b.max_kv) c.share.max_shared = b.max_kv;
  const long long rows = (long long)b.total_q * heads, each = ((long long)b.total_q + share.num_groups - 1) / std::max(share.num_groups, 1);      // tokens of a group
  const long long front = (long long)c.share.max_shared / c.g.page * c.g.page;
  // two results a row at least
  const long long most_slots = std::min(PA_SCRATCH / std::max(rows * (c.g.hd + 2) * 4, 1LL), 1024LL);
  // nothing is shared, so little that it gains nothing, or there are so many rows
  if (share.num_groups == 0 || front == 0 || most_slots < 2 || !sharing_pays(b, share.num_groups, front, c.g, c.group, each))
    return wv_launch_attn_paged(kv, b, dq, ldq, dout, ldo, heads, scale, 0, st);
  const long long top[2] = {each * c.group, (long long)b.max_q * c.group};                   // rows of a kv head: of a group on average, of a sequence at most
  struct Part { bool chunk, r16; long long grid, per, n; } part[2];
  for (int i = 0; i < 2; i++) { part[i].chunk = c.g.hd <= 128 && top[i] > 32; part[i].r16 = top[i] > 8; }
  const bool both = !part[0].chunk && !part[1].chunk;                    // one launch
  if (both) part[0].r16 = part[1].r16 = part[0].r16 || part[1].r16;
  for (int i = 0; i < 2; i++) {
    Part& p = part[i];
    const long long keys = i ? std::max((long long)b.max_kv - front, 1LL) : front;
    const int size = p.chunk ? 128 : p.r16 ? 16 : 8;
    const long long upto = (long long)b.total_q * c.group / size + (i ? b.num_seqs : share.num_groups), sure = (top[i] + size - 1) / size;
    const long long likely = i && p.chunk ? std::min(b.num_seqs * sure, upto) : (i ? b.num_seqs : share.num_groups) * sure;
    p.grid = i ? likely : upto;
    if (p.chunk) {
      const long long tiles = (keys + 127) / 128, n = chunk_splits(likely * c.g.kvh, tiles, 64);
      p.per = (tiles + n - 1) / n * 128;
    } else {
      p.per = rows_per_split(keys, likely * c.g.kvh, c.g, kv.bits, p.r16);
    }
    p.n = (keys + p.per - 1) / p.per;
  }
  if (part[0].n + part[1].n > most_slots) {                              // fewer and longer splits, which the kernel for few rows takes in stretches
    for (int i = 1; i >= 0; i--) {
      const long long n = std::min(part[i].n, i ? std::max(most_slots / 2, 1LL) : most_slots - part[1].n), keys = i ? std::max((long long)b.max_kv - front, 1LL) : front;
      part[i].per = ((keys + n - 1) / n + 127) & ~127LL;
      part[i].n = (keys + part[i].per - 1) / part[i].per;
    }
  }
  // Bounds so loose that most of the tiles which they allow are empty (wide heads alone: the chunk kernel's follow total_q), or that a grid cannot hold them: the
  // other call looks its sequences up.
  if (!part[1].chunk && part[1].grid / 4 > (long long)b.total_q * c.group / (part[1].r16 ? 16 : 8) + b.num_seqs) return wv_launch_attn_paged(kv, b, dq, ldq, dout, ldo, heads, scale, 0, st);
  if ((part[0].grid * part[0].n + part[1].grid * part[1].n) * c.g.kvh > INT_MAX) return wv_launch_attn_paged(kv, b, dq, ldq, dout, ldo, heads, scale, 0, st);
  c.nslots = (int)(part[0].n + part[1].n);
  WvLease lease;
  const size_t n = (size_t)rows * c.nslots, sums = (2 * n + 3) & ~(size_t)3;
  if (const int rc = wv_lease(lease, sums + n * c.g.hd, st, "wv_attn_shared_dev: the splits' results")) return rc;
  c.ml = reinterpret_cast<float2*>(lease.p);
  c.acc = lease.p + sums;
  cudaError_t e = cudaSuccess;
  const long long blocks[2] = {part[0].grid * c.g.kvh * part[0].n, part[1].grid * c.g.kvh * part[1].n};
  c.slot0 = 0; c.per = (int)part[0].per; c.nsplit = (int)part[0].n;
  c.own_slot0 = (int)part[0].n; c.own_per = (int)part[1].per; c.own_nsplit = (int)part[1].n;
  c.own_tiles = (unsigned)(((long long)b.max_q * c.group + (part[1].r16 ? 15 : 7)) / (part[1].r16 ? 16 : 8));
  if (both) {
    c.split = (unsigned)blocks[0];
    e = rows_any<true>(c, kv.bits, part[0].r16, (int)(blocks[0] + blocks[1]), st);
  } else {
    for (int i = 0; i < 2 && e == cudaSuccess; i++) {
      PaCall r = c;
      if (part[i].chunk) {
        r.part = i + 1;
        r.rows_most = 0;
        if (i) { r.slot0 = c.own_slot0; r.per = c.own_per; r.nsplit = c.own_nsplit; }
        e = wv_launch_chunk_part(r, kv.bits, part[i].grid, st);
      } else {
        r.split = i ? 0u : (unsigned)blocks[0];
        e = rows_any<true>(r, kv.bits, part[i].r16, (int)blocks[i], st);
      }
    }
  }
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    cfg.gridDim = dim3((unsigned)b.total_q, (unsigned)((heads + 7) / 8)); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = (size_t)8 * c.nslots * 4; cfg.stream = st;
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, shared_join_kernel, c);
  }
  if (e != cudaSuccess) { wv_set_error("wv_attn_shared_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA; }
  return WV_OK;
}
