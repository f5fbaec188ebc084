// Attention of many new tokens of a sequence over the paged cache (prompts and pieces of them) on tcgen05.
//
// A block takes 256 rows (tokens x query heads of one kv head, so that a cached row is read once for the group) as two tiles of 128
// and walks the keys, 128 at a time, with a running maximum:
//   S = Q K^T    Q (two float16 pieces, hi and lo) and K in shared memory, S in tensor memory       2 x 128 x 128 x head_dim products
//   P            weights in two float16 pieces, written over S, 16 keys a piece pair                 two threads a row
//   O_j = P V    P out of tensor memory, V in shared memory, keys being V's rows                     2 x 128 x head_dim x 128
// O is summed up over the key tiles in registers (128 float32 a row): the tensor core cuts instead of rounding as it adds, which over
// thousands of keys would show, a tile's 128 do not; and the maximum's correction is a factor in that sum instead of a pass over
// tensor memory. Codes are exact in float16, so with hi and lo the products carry 22 bits: float32's accuracy costs two products
// where 16-bit activations would take one: the tensor pipe runs 4096 cycles for 256 x 128 x head_dim 128. Such a pair of tiles takes some
// 8000 now: the weights alone 2600 of issue on every scheduler (ten cycles an element: ex2 eight, beside it the conversions and the
// packed products), the maxima, the sums in registers and the waits between the roles the rest.
//
// Measured, heads of 128: prompts of up to 4096 tokens, four together, 32 heads in 16 bits, 546 us (floor of the doubled products 238); 2048
// tokens of 10000 with a window of 4000, 64 heads in 4 bits, 669 us (323); 512 tokens over 4608 positions, 32 heads in 8 bits, 120 us (44).
//
// Roles: four warpgroups have a tile's half each (a thread a row: the weights of 64 of the 128 keys, the sums of half of the values),
// one warp issues the MMAs, three fill the ring, K and V tiles in turn. With one warpgroup a tile the weights of 128 keys were a
// chain of some 3500 cycles with nothing to issue beside it; with two the pairs hide one another's latencies. Rows of 16 bits are
// copied asynchronously into one of three stages; codes of 8 and 4 bits are copied as they are, two tiles ahead and each thread for
// itself, and turned into float16 on the way from there to one of two stages. Codes of 4 bits lie in the order in which they unpack two
// at a time (0 4 1 5 2 6 3 7); Q follows, and the outputs are put back.
//
// The running maximum is raised only where a logit may lie 2^10 above it, which a bound tells (the row's largest product times the
// tile's largest scale), so that most tiles are read once; a row's two threads agree on that, and exchange their maxima through tensor
// memory that the next tile's sums will overwrite.
//
// A logit is S times its key's scale, in one fused step with the subtraction of the reference. The reference is a rounded product, so from
// 2^24 on the two may lie further apart than a weight's range: where a warp's reference is 2^20 or more, and in tiles with a mask, the
// product is rounded first.
//
// A key's scale multiplies its column of S; a value row's, relative to the largest of its tile, its weight, and the tile's own power
// of two goes into the sum over tiles. Where the scales in a tile lie further apart than the pieces' range holds (2^8), the tile's
// weighted sum is taken value by value in float32 instead.
//
// Every wait is bounded: when one runs out the block records a code, all roles leave their loops, and tensor memory is released
// after the MMAs in flight (waited for, bounded again).
#include "wv_attn_paged.cuh"
#include "wv_tma_common.cuh"
#include "wv_lease.h"
#include <type_traits>

#define PC_THREADS 640
#define PC_MMA_WARP 19
#define PC_M 128                    // rows of a tile
#define PC_N 128                    // keys of a tile
#define PC_PRODUCERS 3              // warps 16 - 18
#define PC_LIFT 4.f                 // weights carry 2^4 and are at most 2^15 (2^10 over the reference, scales below 2)
#define PC_SLACK 10.f
#define PC_SPIN (1u << 20)          // polls of a wait

int wv_sm_count();

__device__ __forceinline__ void pc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool pc_elect() {
  unsigned p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Operands in shared memory, 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1024 bytes apart. As K-major operand (Q, K) a
// row is 64 values of the sum's index; as MN-major operand (V) a row is a step of the sum's index and the next 64 columns lie
// `lbo` bytes further.
__device__ __forceinline__ unsigned long long pc_desc(unsigned saddr, unsigned lbo) {
  return (unsigned long long)((saddr & 0x3FFFFu) >> 4) | ((unsigned long long)(lbo >> 4) << 16) | ((unsigned long long)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void pc_mma_ss(unsigned d, unsigned long long da, unsigned long long db, unsigned idesc, unsigned acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void pc_mma_ts(unsigned d, unsigned ta, unsigned long long db, unsigned idesc, unsigned acc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(ta), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void pc_commit(unsigned bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
#define PC_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define PC_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void pc_ld32(unsigned taddr, unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : PC_R8(r, 0), PC_R8(r, 8), PC_R8(r, 16), PC_R8(r, 24) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void pc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pc_ld16(unsigned taddr, unsigned (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : PC_R8(r, 0), PC_R8(r, 8) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void pc_st16(unsigned taddr, const unsigned (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), PC_W8(r, 0), PC_W8(r, 8) : "memory");
}
__device__ __forceinline__ unsigned pc_ld1(unsigned taddr) {
  unsigned v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
  pc_wait_ld();
  return v;
}
template <int N> __device__ __forceinline__ void pc_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void pc_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Shared memory: Q [tile][piece][head_dim / 64][128 rows][128 bytes], the ring of K and V tiles [head_dim / 64][128 keys][128 bytes], the
// codes on their way (8 and 4 bits), then this.
struct PcMeta {
  float kk[2][PC_N], fv[2][PC_N];           // of a key tile (two of them in turn): the keys' scales times q's, the value rows' scales over 2^e
  float beta[2], kmax[2];                   // 2^e, the largest kk
  unsigned flags[2];                        // 1: some key of the tile is not there, 2: value scales too far apart
  unsigned valid[2][4];                     // which keys are there
  unsigned long long bar[21];
  unsigned vote[2][2];
  unsigned tmem, qmax;
  unsigned char qexp[2 * PC_M], lift[2 * PC_M];      // of a row: exponent field of its largest |q|, and what it is lifted by
  int abort;
  int seq, tile;
};
template <int BITS, int DP> struct PcShape {
  static constexpr int STAGES = BITS == 16 ? 3 : 2, STAGE = DP / 64 * PC_N * 128, QPIECE = DP / 64 * PC_M * 128;
  static constexpr int PIECES = BITS == 16 ? DP / 8 : DP / 16;                    // of a row: 16 bytes, or 16 codes
  static constexpr int PER = PIECES / 2;                                          // of 16 rows, a lane
  static constexpr int RAW = BITS == 16 ? 0 : PIECES * PC_N * (BITS == 8 ? 16 : 8) + (BITS == 4 ? 1024 : 0);      // 4 bits: codes, then sub-scales
  static constexpr size_t SMEM = (size_t)4 * QPIECE + STAGES * STAGE + 2 * RAW + sizeof(PcMeta);
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <int BITS> __device__ __forceinline__ int pc_dim(int p) {      // the value that stands at place p of a row
  if constexpr (BITS == 4) return (p & ~7) | ((p & 7) >> 1) | (p & 1) << 2;
  return p;
}

template <int BITS, int DP>
__global__ void __launch_bounds__(PC_THREADS, 1) attn_chunk_kernel(const __grid_constant__ PaCall c) {
  using S = PcShape<BITS, DP>;
  constexpr int STAGES = S::STAGES, STAGE = S::STAGE, QPIECE = S::QPIECE;
  constexpr unsigned IDESC_S = (1u << 4) | (PC_N / 8 << 17) | (PC_M / 16 << 24);                   // f32 sums, f16 operands, both K-major
  constexpr unsigned IDESC_O = (1u << 4) | (1u << 16) | (DP / 8 << 17) | (PC_M / 16 << 24);        // B with its columns innermost
  extern __shared__ __align__(1024) unsigned char pc_smem[];
  unsigned char* s_q = pc_smem;
  unsigned char* s_kv = pc_smem + 4 * QPIECE;
  unsigned char* s_raw = s_kv + STAGES * STAGE;
  PcMeta& M = *reinterpret_cast<PcMeta*>(s_raw + 2 * S::RAW);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  auto full = [&](int s) { return smem_u32(&M.bar[s]); };
  auto empty = [&](int s) { return smem_u32(&M.bar[3 + s]); };
  auto s_full = [&](int t) { return smem_u32(&M.bar[6 + t]); };
  auto p_full = [&](int t) { return smem_u32(&M.bar[8 + t]); };
  auto o_full = [&](int t) { return smem_u32(&M.bar[10 + t]); };
  auto m_full = [&](int s) { return smem_u32(&M.bar[12 + s]); };
  auto m_empty = [&](int s) { return smem_u32(&M.bar[14 + s]); };
  const unsigned done = smem_u32(&M.bar[16]);
  auto v_bar = [&](int t) { return smem_u32(&M.bar[17 + t]); };
  auto x_bar = [&](int t) { return smem_u32(&M.bar[19 + t]); };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (smem_u32(pc_smem) & 1023u) { if (tid == 0) atomicCAS_system(c.err - 1, 0, 799); return; }    // the swizzle counts from 1024-byte boundaries

  // ---------------------------------------------------------------- which rows: tiles of 256 of the sequences that have more than rows_most
  const int kvh = blockIdx.x % c.g.kvh, flat = blockIdx.x / c.g.kvh, sp = blockIdx.y;
  if (warp == 0) {
    int seq, tile;
    pa_find(c, flat, 256, c.rows_most, blockIdx.x == 0 && sp == 0 ? c.err : nullptr, seq, tile);
    if (lane == 0) { M.seq = seq; M.tile = tile; M.qmax = 0; M.abort = 0; }
  }
  __syncthreads();
  const int seq = M.seq;
  if (seq < 0) return;
  const WvSeq sq = wv_seq(c.b, c.g.page, seq, sp == 0 && kvh == 0 ? c.err : nullptr);
  const int nrows = (sq.q1 - sq.q0) * c.group, r0 = M.tile * 256, rn = min(256, nrows - r0);
  int lo, hi;
  pa_range(sq, r0 / c.group, (r0 + rn - 1) / c.group, c.window, lo, hi);
  const unsigned first = (unsigned)lo + (unsigned)(sp * c.per);
  const int k0 = (int)min(first, (unsigned)hi), k1 = min(hi, k0 + c.per);
  const int hd = c.g.hd, pos0 = sq.p0;
  const size_t rec0 = ((size_t)flat * c.g.kvh + kvh) * 256;               // this block's rows in the split results
  if (k0 >= k1) {
    if (c.nsplit > 1) { if (tid < rn) c.ml[(rec0 + tid) * c.nsplit + sp] = make_float2(-INFINITY, 0.f); }
    else for (int i = tid; i < rn * hd; i += PC_THREADS) {
      const int r = r0 + i / hd;
      c.out[(size_t)(sq.q0 + r / c.group) * c.ldo + (size_t)(kvh * c.group + r % c.group) * hd + i % hd] = 0.f;
    }
    return;
  }
  const int n = (k1 - k0 + PC_N - 1) / PC_N;
  const bool two = rn > PC_M;

  if (tid == 0) {
    for (int s = 0; s < STAGES; s++) { mbar_init(full(s), PC_PRODUCERS); mbar_init(empty(s), 1); }
    for (int t = 0; t < 2; t++) {
      mbar_init(s_full(t), 1); mbar_init(p_full(t), 8); mbar_init(o_full(t), 1);
      mbar_init(m_full(t), 1); mbar_init(m_empty(t), two ? 16 : 8);
      mbar_init(v_bar(t), 8); mbar_init(x_bar(t), 8);
      M.vote[t][0] = M.vote[t][1] = 0;
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == PC_MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&M.tmem)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // ---------------------------------------------------------------- Q: a power of two, two pieces, the operand's layout
  // The power of two is that of the block's largest row, so that the keys' scales carry it for all rows. A row that lies further below
  // than its pieces reach (by more than 2^15: the second piece then ends above 2^-24 of the row's largest) is lifted by its own, and its
  // sums are put down again, by warps that have such a row. Rows before position 0 see nothing and are zeros, whatever they hold.
  auto qrow = [&](int r) { return c.q + (size_t)(sq.q0 + (r0 + r) / c.group) * c.ldq + (size_t)(kvh * c.group + (r0 + r) % c.group) * hd; };
  {
    unsigned top = 0;
    for (int r = warp; r < rn; r += PC_THREADS / 32) {
      const float* src = qrow(r);
      unsigned m = 0;
      for (int d = 4 * lane; d < hd; d += 128) {
        const float4 v = *reinterpret_cast<const float4*>(src + d);
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; e++) { const unsigned u = __float_as_uint(x[e]) & 0x7fffffffu; if (u < 0x7f800000u) m = max(m, u); }
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (pos0 + (r0 + r) / c.group >= 0) top = max(top, m);
      if (lane == 0) M.qexp[r] = (unsigned char)(m >> 23);
    }
    if (lane == 0) atomicMax(&M.qmax, top);
  }
  pc_fence_before();
  __syncthreads();
  pc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, *(volatile unsigned*)&M.tmem, 0);
  const int qe = min(max((int)(M.qmax >> 23) - 127 - 13, -100), 114);
  const float qinv = copysignf(__uint_as_float((unsigned)(127 - qe) << 23), c.scale);              // a negative scale turns q, so that kk is positive
  const float qf = fabsf(c.scale) * __uint_as_float((unsigned)(127 + qe) << 23);
  auto lift = [&](int r) {
    const int own = M.qexp[r], up = qe - max(own - 127 - 13, -100);
    return own && up > 15 ? min(up, 100) : 0;
  };
  if (tid < 2 * PC_M) M.lift[tid] = (unsigned char)(tid < rn ? lift(tid) : 0);
  for (int i = tid; i < 256 * (DP / 8); i += PC_THREADS) {               // 8 places of a row at a time
    const int r = i / (DP / 8), j = i % (DP / 8);
    if (r >= PC_M && !two) break;
    unsigned h[4] = {0u, 0u, 0u, 0u}, l[4] = {0u, 0u, 0u, 0u};
    if (r < rn && 8 * j < hd && pos0 + (r0 + r) / c.group >= 0) {
      const float* src = qrow(r) + 8 * j;
      const float f = qinv * __uint_as_float((unsigned)(127 + lift(r)) << 23);
      const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
      float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = x[e] - x[e] == 0.f ? x[e] * f : NAN;
#pragma unroll
      for (int p = 0; p < 4; p++) {
        const float u = x[pc_dim<BITS>(2 * p)], v = x[pc_dim<BITS>(2 * p + 1)];
        h[p] = pa_pack(u, v);
        const float2 back = pa_unpack(h[p]);
        l[p] = pa_pack(u - back.x, v - back.y);
      }
    }
    const int rr = r & (PC_M - 1);
    unsigned char* dst = s_q + (r / PC_M) * 2 * QPIECE + (j >> 3) * PC_M * 128 + rr * 128 + (((j & 7) ^ (rr & 7)) << 4);
    *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(dst + QPIECE) = make_uint4(l[0], l[1], l[2], l[3]);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");           // these stores before the MMAs' reads
  __syncthreads();

  auto fail = [&](int code) { atomicCAS_system(c.err - 1, 0, code); *(volatile int*)&M.abort = 1; };      // the word before is the waits'
  auto dead = [&]() { return *(volatile int*)&M.abort != 0; };

  if (warp < 16) {
    // ============================================================== half a tile: weights of 64 keys, sums of half of the values
    pc_regs_up<104>();
    constexpr int HD = DP / 2, HK = PC_N / 2;
    const int t = warp >> 3, hf = (warp >> 2) & 1, row = tid & (PC_M - 1), r = t * PC_M + row;
    if (t == 0 || two) {
      const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
      const unsigned ts = tmem + lanes + t * PC_N + hf * HK, to = tmem + lanes + 256 + t * 128 + hf * HD, tx = to + HD - 2 * hf * HD;
      const int prow = pos0 + (r0 + min(r, rn - 1)) / c.group;
      const int pmin = pos0 + (r0 + t * PC_M) / c.group, pmax = pos0 + (r0 + min(t * PC_M + PC_M, rn) - 1) / c.group;
      float o[HD], m = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int d = 0; d < HD; d++) o[d] = 0.f;
      bool ok = true;
      int nv = 0, nx = 0;                                                // votes and exchanges so far
      // a wait of the whole warp; false when it ran out or the block has given up
      auto wait = [&](unsigned bar, int use, int why) {
        if (ok && !mbar_wait(bar, use & 1, PC_SPIN)) { if (!dead()) fail(why); ok = false; }
        ok = !__any_sync(0xffffffffu, !ok);
        return ok;
      };
      // the tile's eight warps meet
      auto meet = [&](unsigned bar, int use, int why) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
        return wait(bar, use, why);
      };
      for (int j = 0; j < n; j++) {
        const int ms = j & 1, key0 = k0 + j * PC_N;
        // rows that are lifted or have a reference of 2^20 or more: the warp rounds its logits first
        const unsigned lifted = M.lift[r];
        auto apart = [&]() { return __any_sync(0xffffffffu, lifted || (__float_as_uint(m) & 0x7fffffffu) - __float_as_uint(1048576.f) < 0x7f800000u - __float_as_uint(1048576.f)); };
        bool slow = apart();
        if (!wait(m_full(ms), j >> 1, 700 + t) || !wait(s_full(t), j, 702 + t)) break;
        pc_fence_after();
        const unsigned kk = smem_u32(M.kk[ms]) + 4 * HK * hf, fv = smem_u32(M.fv[ms]) + 4 * HK * hf;
        float beta = M.beta[ms], alpha = 1.f;
        const float down = __uint_as_float((127u - lifted) << 23);
        const unsigned flags = M.flags[ms];
        const bool masked = (flags & 1u) || key0 + PC_N - 1 > pmin || key0 + PC_N > k1 || (c.window != 0 && key0 <= pmax - c.window);
        // bit k of `see`: the row sees key 32 q + k of the half
        auto sees = [&](int at, int word) {
          const int a = key0 + 32 * at, last = min(prow, k1 - 1) - a, first = c.window ? prow - c.window + 1 - a : 0;
          unsigned w = last < 0 ? 0u : last >= 31 ? ~0u : (2u << last) - 1u;
          if (first > 0) w &= first > 31 ? 0u : ~0u << first;
          return w & M.valid[ms][word];
        };
        unsigned see[2] = {~0u, ~0u};
        if (masked) { see[0] = sees(2 * hf, 2 * hf); see[1] = sees(2 * hf + 1, 2 * hf + 1); }
        // ---- the reference: may a logit lie too far above it?
        bool raise = masked;
        if (!masked) {
          float top = 0.f;
#pragma unroll
          for (int q = 0; q < 4; q++) {
            unsigned a[16];
            pc_ld16(ts + 16 * q, a);
            pc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i += 2) top = fmaxf(top, fmaxf(__uint_as_float(a[i]), __uint_as_float(a[i + 1])));
          }
          if (__any_sync(0xffffffffu, !(top * down * M.kmax[ms] <= m + PC_SLACK)) && lane == 0) atomicOr(&M.vote[t][nv & 1], 1u);
          if (!meet(v_bar(t), nv, 704 + t)) break;
          raise = *(volatile unsigned*)&M.vote[t][nv & 1] != 0;
          if ((warp & 7) == 0 && lane == 0) M.vote[t][(nv + 1) & 1] = 0; // nobody comes to the next vote before this warp's weights are there
          nv++;
        }
        if (raise) {
          float mx = m;
#pragma unroll 1
          for (int q = 0; q < 4; q++) {
            const unsigned bits = ((q < 2 ? see[0] : see[1]) >> (16 * (q & 1))) & 0xffffu;
            if (!__any_sync(0xffffffffu, bits)) continue;                // keys that none of the warp's rows sees
            unsigned a[16];
            pc_ld16(ts + 16 * q, a);
            pc_wait_ld();
            const bool all = __all_sync(0xffffffffu, bits == 0xffffu);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const uint4 k4 = lds128(kk + 64 * q + 4 * i);
              const float2 dd = make_float2(down, down);
              const float2 xa = __fmul2_rn(__fmul2_rn(make_float2(__uint_as_float(a[i]), __uint_as_float(a[i + 1])), dd), make_float2(__uint_as_float(k4.x), __uint_as_float(k4.y)));
              const float2 xb = __fmul2_rn(__fmul2_rn(make_float2(__uint_as_float(a[i + 2]), __uint_as_float(a[i + 3])), dd), make_float2(__uint_as_float(k4.z), __uint_as_float(k4.w)));
              float x[4] = {xa.x, xa.y, xb.x, xb.y};
              if (!all) {
#pragma unroll
                for (int u = 0; u < 4; u++) x[u] = (bits >> (i + u)) & 1u ? x[u] : -INFINITY;
              }
              mx = fmaxf(mx, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
            }
          }
          asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(to), "r"(__float_as_uint(mx)) : "memory");
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          pc_fence_before();
          if (!meet(x_bar(t), nx++, 706 + t)) break;
          pc_fence_after();
          mx = fmaxf(mx, __uint_as_float(pc_ld1(tx)));
          alpha = mx > m ? pa_ex2(m - mx) : 1.f;                         // 0 while there was nothing
          m = mx;
          slow = apart();
          l2 = __fmul2_rn(l2, make_float2(alpha, alpha));
        }
        const float2 off = m == -INFINITY ? make_float2(0.f, 0.f) : make_float2(PC_LIFT - m, PC_LIFT - m);
        if (flags & 2u) {
          // ---- value by value in float32: both threads of a row go through all 128 keys; then P is zero
          const int e = 2 * j + 1;
          if (!wait(full(e % STAGES), e / STAGES, 708)) break;
          const unsigned char* v = s_kv + (e % STAGES) * STAGE;
          const unsigned tt = tmem + lanes + t * PC_N;
#pragma unroll
          for (int d = 0; d < HD; d++) o[d] *= alpha;
          alpha = 1.f;
#pragma unroll 1
          for (int k = 0; k < PC_N; k++) {
            const float x = __fadd_rn(__fmul_rn(__uint_as_float(pc_ld1(tt + k)) * down, M.kk[ms][k]), off.x);
            const bool on = !masked || ((sees(k >> 5, k >> 5) >> (k & 31)) & 1u);
            const float p = on ? pa_ex2(x) : 0.f, w = on ? p * M.fv[ms][k] * beta : 0.f;
            if (k / HK == hf) l2.x += p;
#pragma unroll
            for (int g = 0; g < HD / 8; g++) {
              const int at = hf * (HD / 8) + g;                          // 16 bytes of the row
              const uint4 q = *reinterpret_cast<const uint4*>(v + (at >> 3) * PC_N * 128 + k * 128 + (((at & 7) ^ (k & 7)) << 4));
              const float2 a = pa_unpack(q.x), b = pa_unpack(q.y), d = pa_unpack(q.z), f = pa_unpack(q.w);
              o[8 * g] += w * a.x; o[8 * g + 1] += w * a.y; o[8 * g + 2] += w * b.x; o[8 * g + 3] += w * b.y;
              o[8 * g + 4] += w * d.x; o[8 * g + 5] += w * d.y; o[8 * g + 6] += w * f.x; o[8 * g + 7] += w * f.y;
            }
          }
          beta = 0.f;
          pc_fence_before();
          if (!meet(x_bar(t), nx++, 706 + t)) break;                     // the row's other thread has read S
          pc_fence_after();
          unsigned z[16];
#pragma unroll
          for (int i = 0; i < 16; i++) z[i] = 0u;
#pragma unroll
          for (int q = 0; q < 4; q++) pc_st16(ts + 16 * q, z);
        } else {
          // ---- weights: 16 keys of S become 8 columns of their hi pieces and 8 of their lo pieces
          auto weights = [&](auto some, int q, unsigned bits) {
            unsigned s[16], w[16];
            pc_ld16(ts + 16 * q, s);
            pc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const uint4 k4 = lds128(kk + 64 * q + 4 * i), f4 = lds128(fv + 64 * q + 4 * i);
#pragma unroll
              for (int u = 0; u < 4; u += 2) {
                float2 sv = make_float2(__uint_as_float(s[i + u]), __uint_as_float(s[i + u + 1]));
                if constexpr (decltype(some)::value) sv = __fmul2_rn(sv, make_float2(down, down));
                const float2 kv = u ? make_float2(__uint_as_float(k4.z), __uint_as_float(k4.w)) : make_float2(__uint_as_float(k4.x), __uint_as_float(k4.y));
                float2 x;                                                // (a packed product and sum may still be fused)
                if constexpr (decltype(some)::value) x = make_float2(__fadd_rn(__fmul_rn(sv.x, kv.x), off.x), __fadd_rn(__fmul_rn(sv.y, kv.y), off.x));
                else x = __ffma2_rn(sv, kv, off);
                float2 p = make_float2(pa_ex2(x.x), pa_ex2(x.y));
                float2 pf = __fmul2_rn(p, u ? make_float2(__uint_as_float(f4.z), __uint_as_float(f4.w)) : make_float2(__uint_as_float(f4.x), __uint_as_float(f4.y)));
                if constexpr (decltype(some)::value) {
                  const bool a = (bits >> (i + u)) & 1u, b = (bits >> (i + u + 1)) & 1u;
                  p = make_float2(a ? p.x : 0.f, b ? p.y : 0.f);
                  pf = make_float2(a ? pf.x : 0.f, b ? pf.y : 0.f);
                }
                l2 = __fadd2_rn(l2, p);
                const unsigned h = pa_pack(pf.x, pf.y);
                const float2 lo_ = __ffma2_rn(pa_unpack(h), make_float2(-1.f, -1.f), pf);
                w[(i + u) / 2] = h;
                w[8 + (i + u) / 2] = pa_pack(lo_.x, lo_.y);
              }
            }
            pc_st16(ts + 16 * q, w);
          };
          if (!masked && !slow) {
#pragma unroll
            for (int q = 0; q < 4; q++) weights(std::false_type(), q, 0u);
          } else {
#pragma unroll 1
            for (int q = 0; q < 4; q++) {
              const unsigned bits = ((q < 2 ? see[0] : see[1]) >> (16 * (q & 1))) & 0xffffu;
              if (!__any_sync(0xffffffffu, bits)) {
                unsigned z[16];
#pragma unroll
                for (int i = 0; i < 16; i++) z[i] = 0u;
                pc_st16(ts + 16 * q, z);
              } else {
                weights(std::true_type(), q, bits);
              }
            }
          }
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        pc_fence_before();
        __syncwarp();
        if (lane == 0) { mbar_arrive(p_full(t)); mbar_arrive(m_empty(ms)); }
        // ---- this tile's part of the sum
        if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
          for (int d = 0; d < HD; d += 2) { const float2 v = __fmul2_rn(make_float2(o[d], o[d + 1]), make_float2(alpha, alpha)); o[d] = v.x; o[d + 1] = v.y; }
        }
        if (!wait(o_full(t), j, 710 + t)) break;
        pc_fence_after();
#pragma unroll
        for (int q = 0; q < HD / 16; q++) {
          unsigned a[16];
          pc_ld16(to + 16 * q, a);
          pc_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 v = __ffma2_rn(make_float2(__uint_as_float(a[i]), __uint_as_float(a[i + 1])), make_float2(beta, beta), make_float2(o[16 * q + i], o[16 * q + i + 1]));
            o[16 * q + i] = v.x; o[16 * q + i + 1] = v.y;
          }
        }
      }
      // the row's divisor: the two halves' sums
      float l = l2.x + l2.y;
      if (ok) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(to), "r"(__float_as_uint(l)) : "memory");
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        pc_fence_before();
        if (meet(x_bar(t), nx++, 706 + t)) {
          pc_fence_after();
          l += __uint_as_float(pc_ld1(tx));
        }
      }
      if (r < rn) {
        float f = 1.f;
        float* dst;
        if (c.nsplit > 1) {
          dst = c.acc + ((rec0 + r) * c.nsplit + sp) * hd;
          if (hf == 0) c.ml[(rec0 + r) * c.nsplit + sp] = make_float2(m, l);
        } else {
          dst = c.out + (size_t)(sq.q0 + (r0 + r) / c.group) * c.ldo + (size_t)(kvh * c.group + (r0 + r) % c.group) * hd;
          f = l == 0.f ? 0.f : 1.f / l;
        }
#pragma unroll
        for (int g = 0; g < HD / 8; g++) {
          const int d = hf * HD + 8 * g;
          if (d < hd) {
            float x[8];
#pragma unroll
            for (int p = 0; p < 8; p++) x[pc_dim<BITS>(p)] = ok ? o[8 * g + p] * f : NAN;
            *reinterpret_cast<float4*>(dst + d) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(dst + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
          }
        }
      }
    }
  } else {
    pc_regs_down<64>();
    if (warp == PC_MMA_WARP) {
      // ============================================================ MMAs
      const bool leader = pc_elect();
      const unsigned qa = smem_u32(s_q), kv = smem_u32(s_kv);
      const int nt = two ? 2 : 1;
      bool ok = true;
      auto wait = [&](unsigned bar, int use, int code) {
        if (ok && !mbar_wait(bar, use & 1, PC_SPIN)) { if (!dead() && leader) fail(code); ok = false; }
        ok = !__any_sync(0xffffffffu, !ok || dead());
        return ok;
      };
      auto scores = [&](int t, int e) {                                  // S of tile t with the K tile that is element e of the ring
        if (leader) {
          const unsigned kb = kv + (e % STAGES) * STAGE;
#pragma unroll
          for (int p = 1; p >= 0; p--) {                                 // the small pieces first
            const unsigned qb = qa + (2 * t + p) * QPIECE;
#pragma unroll
            for (int k = 0; k < DP / 16; k++)
              pc_mma_ss(tmem + t * PC_N, pc_desc(qb + (k >> 2) * PC_M * 128 + (k & 3) * 32, 16), pc_desc(kb + (k >> 2) * PC_N * 128 + (k & 3) * 32, 16), IDESC_S, !(p == 1 && k == 0));
          }
          pc_commit(s_full(t));
        }
        __syncwarp();
      };
      auto values = [&](int t, int e) {
        if (leader) {
          const unsigned vb = kv + (e % STAGES) * STAGE;
#pragma unroll
          for (int p = 1; p >= 0; p--)
#pragma unroll
            for (int k = 0; k < PC_N / 16; k++)
              pc_mma_ts(tmem + 256 + t * 128, tmem + t * PC_N + 16 * k + 8 * p, pc_desc(vb + k * 2048, PC_N * 128), IDESC_O, !(p == 1 && k == 0));
          pc_commit(o_full(t));
        }
        __syncwarp();
      };
      auto release = [&](int e) { if (leader) pc_commit(empty(e % STAGES)); __syncwarp(); };
      if (wait(full(0), 0, 712)) {
        pc_fence_after();
        for (int t = 0; t < nt; t++) scores(t, 0);
        release(0);
      }
      // From then on whatever is ready first: a tile's values of step pv[t] when its weights and V are there, its scores of the next
      // step, which overwrite those weights, after that when K is. In a fixed order the pipe waited for K with another tile's
      // weights at hand.
      int pv[2] = {0, 0}, qk[2] = {1, 1};
      auto ready = [&](unsigned bar, int use) {
        unsigned yes;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes) : "r"(bar), "r"(use & 1) : "memory");
        return __any_sync(0xffffffffu, yes) != 0;
      };
      unsigned idle = 0;
      while (ok && (pv[0] < n || (nt == 2 && pv[1] < n))) {
        bool did = false;
        for (int t = 0; t < nt; t++) {
          if (pv[t] < n && pv[t] < qk[t] && ready(full((2 * pv[t] + 1) % STAGES), (2 * pv[t] + 1) / STAGES) && ready(p_full(t), pv[t])) {
            pc_fence_after();
            const int e = 2 * pv[t] + 1;
            values(t, e);
            pv[t]++;
            if (nt == 1 || pv[t ^ 1] >= pv[t]) release(e);               // the other tile has used it, too
            did = true;
          }
          if (qk[t] < n && pv[t] >= qk[t] && ready(full(2 * qk[t] % STAGES), 2 * qk[t] / STAGES)) {
            pc_fence_after();
            const int e = 2 * qk[t];
            scores(t, e);
            qk[t]++;
            if (nt == 1 || qk[t ^ 1] >= qk[t]) release(e);
            did = true;
          }
        }
        idle = did ? 0 : idle + 1;
        if (idle > PC_SPIN) { if (leader) fail(713); ok = false; }
        if ((idle & 255) == 255 && __any_sync(0xffffffffu, dead())) ok = false;
      }
      if (!ok) {                                                         // what was issued has to end before tensor memory is given back
        if (leader) pc_commit(done);
        __syncwarp();
        mbar_wait(done, 0, PC_SPIN);
      }
    } else {
    // ============================================================== K and V tiles
    const int pw = warp - 16, code = c.g.code, page = c.g.page;
    // A warp takes the groups pw, pw + 3, .. of a tile's eight groups of 16 rows; a lane's piece (16 bytes of 16-bit rows, else 16 codes) is
    // number x of rows lr, lr + STEP, ..
    constexpr int STEP = 32 / S::PIECES, PER = S::PER;
    const int x = lane % S::PIECES, lr = lane / S::PIECES, n16 = hd / 16;
    const bool mine = BITS == 16 ? 8 * x < hd : 16 * x < hd;
    // page numbers of 32 groups of 16 keys (four tiles) at a time, a lane each, as offsets in the pool (-1: not there)
    long long blk = 0;
    int slots = 0;
    auto places = [&](int j) {
      if ((j & 3) == 0) {
        const int key = k0 + j * PC_N + 16 * lane, at = key / page;
        int id = key < k1 ? c.b.pages[(size_t)seq * c.b.table_stride + at] : 0;
        if (id < 0 || id >= c.g.num_pages) { if (pw == 0) wv_paged_report(c.err, WV_PAGED_PAGE); id = -1; }
        blk = id < 0 || key >= k1 ? -1LL : ((long long)id * c.g.kvh + kvh) * c.g.block;
        slots = key - at * page;
      }
    };
    float4 ks = make_float4(0.f, 0.f, 0.f, 0.f), vs = ks;                // the first of the warps: four keys a lane of the next tile
    bool there = true;
    auto scales = [&](int j) {
      const int g = 8 * (j & 3) + (lane >> 2);
      const long long at = __shfl_sync(0xffffffffu, blk, g);
      const int slot = __shfl_sync(0xffffffffu, slots, g) + 4 * (lane & 3);
      there = at >= 0 || k0 + j * PC_N + 16 * (lane >> 2) >= k1;         // what lies beyond the keys is not missing
      ks = vs = make_float4(0.f, 0.f, 0.f, 0.f);
      if (at >= 0) {
        ks = *reinterpret_cast<const float4*>(c.g.pool + at + c.g.kscale + 4 * slot);
        vs = *reinterpret_cast<const float4*>(c.g.pool + at + c.g.vscale + 4 * slot);
      }
    };
    // the copies of element e: into its stage (16 bits), or as they are
    auto copy = [&](int e) {
      const int j = e >> 1;
      const bool is_v = e & 1;
      const unsigned stage = smem_u32(s_kv) + (e % STAGES) * STAGE, raw = smem_u32(s_raw) + (e & 1) * S::RAW;
      for (int g = pw; g < 8; g += PC_PRODUCERS) {
        const long long at = __shfl_sync(0xffffffffu, blk, 8 * (j & 3) + g);
        const int slot = __shfl_sync(0xffffffffu, slots, 8 * (j & 3) + g) + lr;
        const int left = at < 0 ? 0 : k1 - (k0 + j * PC_N + 16 * g) - lr;          // the lane's rows 0, STEP, .. below this exist
        const unsigned char* block = c.g.pool + (at < 0 ? 0 : at);
        const unsigned char* src = block + (is_v ? page * code : 0) + slot * code + (BITS == 4 ? 8 : 16) * x;
#pragma unroll
        for (int i = 0; i < PER; i++) {
          const bool on = mine && STEP * i < left;
          const unsigned char* s = on ? src + STEP * i * code : block;
          if constexpr (BITS == 16) {
            const int r = 16 * g + lr + STEP * i;
            const unsigned to = stage + (x >> 3) * PC_N * 128 + r * 128 + (((x & 7) ^ (r & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(s), "r"(on ? 16 : 0) : "memory");
          } else if constexpr (BITS == 8) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(raw + ((g * PER + i) * 32 + lane) * 16), "l"(s), "r"(on ? 16 : 0) : "memory");
          } else {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(raw + ((g * PER + i) * 32 + lane) * 8), "l"(s), "r"(on ? 8 : 0) : "memory");
          }
        }
        // the group's sub-scales, 16 n16 bytes; the warp shares them
        if (BITS == 4 && lane < n16)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(raw + 8 * PER * 256 + g * 128 + 16 * lane),
                       "l"(block + (at < 0 ? 0 : (is_v ? c.g.vsub : c.g.ksub) + (slot - lr) * n16 + 16 * lane)), "r"(at < 0 ? 0 : 16) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Element e out of its copies into its stage. A lane stores two neighbouring 16-byte pieces; those of the upper half of a row start
    // with the second, so that eight lanes reach all banks.
    auto convert = [&](int e) {
      const unsigned stage = smem_u32(s_kv) + (e % STAGES) * STAGE, raw = smem_u32(s_raw) + (e & 1) * S::RAW;
      const bool turned = (x >> 2) & 1;
      for (int g = pw; g < 8; g += PC_PRODUCERS) {
        // all of a group's loads before the first store: the compiler may not move them past it
        unsigned c4[PER][BITS == 8 ? 4 : 2], sc[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) {
          if constexpr (BITS == 8) {
            const uint4 q = lds128(raw + ((g * PER + i) * 32 + lane) * 16);
            c4[i][0] = turned ? q.z : q.x; c4[i][1] = turned ? q.w : q.y; c4[i][BITS == 8 ? 2 : 0] = turned ? q.x : q.z; c4[i][BITS == 8 ? 3 : 1] = turned ? q.y : q.w;
          } else {
            const uint2 q = lds64(raw + ((g * PER + i) * 32 + lane) * 8);
            c4[i][0] = turned ? q.y : q.x; c4[i][1] = turned ? q.x : q.y;
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(sc[i]) : "r"(raw + 8 * PER * 256 + g * 128 + (lr + STEP * i) * n16 + x));
          }
        }
#pragma unroll
        for (int i = 0; i < PER; i++) {
          const int r = 16 * g + lr + STEP * i;
          unsigned v[8];
          if constexpr (BITS == 8) {
#pragma unroll
            for (int k = 0; k < 4; k++) { const unsigned w = c4[i][k] ^ 0x80808080u; v[2 * k] = pa_bytes<0x4140>(w); v[2 * k + 1] = pa_bytes<0x4342>(w); }
          } else {
            const PaSub t2 = pa_pair(sc[i], sc[i]);
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = pa_nibbles(c4[i][k >> 2], k & 3, t2, c.one);
          }
          const unsigned to = stage + (x >> 2) * PC_N * 128 + r * 128 + ((((2 * x + turned) & 7) ^ (r & 7)) << 4);
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to ^ 16u), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
        }
      }
    };
    // what the weights need of tile j
    auto meta = [&](int j) {
      const int ms = j & 1, key0 = k0 + j * PC_N;
      const float kx[4] = {ks.x * qf, ks.y * qf, ks.z * qf, ks.w * qf}, vx[4] = {vs.x, vs.y, vs.z, vs.w};
      int emax = -90, emin = 1000;
      float kmax = 0.f;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int ex = min((int)((__float_as_uint(vx[i]) >> 23) & 255u) - 127, 100);
        if (key0 + 4 * lane + i < k1) {
          if (vx[i] == vx[i] && ex > -90) { emax = max(emax, ex); emin = min(emin, ex); }
          kmax = fmaxf(kmax, kx[i]);
        }
      }
      emax = __reduce_max_sync(0xffffffffu, emax);
      emin = __reduce_min_sync(0xffffffffu, emin);
      kmax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(kmax)));
      const float down = __uint_as_float((unsigned)(127 - emax) << 23);
      *reinterpret_cast<float4*>(&M.kk[ms][4 * lane]) = make_float4(kx[0], kx[1], kx[2], kx[3]);
      *reinterpret_cast<float4*>(&M.fv[ms][4 * lane]) = make_float4(vx[0] * down, vx[1] * down, vx[2] * down, vx[3] * down);
      const unsigned have = __ballot_sync(0xffffffffu, there);           // a bit for 4 keys
      if (lane < 4) {
        unsigned w = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) if ((have >> (8 * lane + i)) & 1u) w |= 15u << (4 * i);
        M.valid[ms][lane] = w;
      }
      if (lane == 0) {
        M.beta[ms] = __uint_as_float((unsigned)(127 + emax) << 23);
        M.kmax[ms] = kmax;
        M.flags[ms] = (have != ~0u ? 1u : 0u) | (emin < emax - 8 ? 2u : 0u);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(m_full(ms));
    };
    auto arrive = [&](int e) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(full(e % STAGES));
    };
    bool ok = true;
    auto wait = [&](unsigned bar, int use, int why) {
      if (!mbar_wait(bar, use & 1, PC_SPIN)) { if (!dead()) fail(why); ok = false; }
      ok = !__any_sync(0xffffffffu, !ok || dead());
      return ok;
    };
    auto room = [&](int e) { return e < STAGES || wait(empty(e % STAGES), e / STAGES - 1, 720); };
    // the tile's page numbers and scales, then its copies, are asked for two elements (one tile) ahead
    auto ahead = [&](int e) {
      if (e >= 2 * n) { asm volatile("cp.async.commit_group;" ::: "memory"); return; }
      if (!(e & 1)) { places(e >> 1); if (pw == 0) scales(e >> 1); }
      copy(e);
    };
    if constexpr (BITS == 16) {
      ahead(0);
      if (pw == 0) meta(0);
      ahead(1);
      for (int e = 0; e < 2 * n && ok; e++) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        arrive(e);
        if ((e & 1) && e + 1 < 2 * n && pw == 0) { const int j = (e + 1) >> 1; if (j >= 2 && !wait(m_empty(j & 1), (j >> 1) - 1, 721)) break; meta(j); }
        if (e + 2 < 2 * n && !room(e + 2)) break;
        ahead(e + 2);
      }
    } else {
      ahead(0);
      if (pw == 0) meta(0);
      ahead(1);
      for (int e = 0; e < 2 * n && ok; e++) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        if (!room(e)) break;
        convert(e);
        arrive(e);
        if ((e & 1) && e + 1 < 2 * n && pw == 0) { const int j = (e + 1) >> 1; if (j >= 2 && !wait(m_empty(j & 1), (j >> 1) - 1, 721)) break; meta(j); }
        ahead(e + 2);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    }
  }
  pc_fence_before();
  __syncthreads();
  if (warp == PC_MMA_WARP) {
    pc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

// The splits' results of a tile's rows joined: a warp per row.
__global__ void __launch_bounds__(256) chunk_join_kernel(const __grid_constant__ PaCall c) {
  __shared__ int s_at[2];
  __shared__ float s_w[8][16];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int kvh = blockIdx.x % c.g.kvh, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) {
    int seq, tile;
    pa_find(c, blockIdx.x / c.g.kvh, 256, c.rows_most, nullptr, seq, tile);
    if (lane == 0) { s_at[0] = seq; s_at[1] = tile; }
  }
  __syncthreads();
  if (s_at[0] < 0) return;
  const WvSeq sq = wv_seq(c.b, c.g.page, s_at[0], nullptr);
  const int nrows = (sq.q1 - sq.q0) * c.group;
  for (int i = blockIdx.y * 8 + warp; i < 256; i += 8 * gridDim.y) {
    const int r = s_at[1] * 256 + i;
    if (r >= nrows) break;
    const size_t rec = (size_t)blockIdx.x * 256 + i;
    const float inv = pa_join_weights(c, rec, s_w[warp]);
    __syncwarp();
    pa_join_sums(c, rec, sq.q0 + r / c.group, kvh * c.group + r % c.group, s_w[warp], inv, lane, 32);
    __syncwarp();
  }
}

template <int BITS, int DP>
static cudaError_t chunk_go(const PaCall& c, long long flat, cudaStream_t st) {
  constexpr size_t smem = PcShape<BITS, DP>::SMEM;
  auto kern = attn_chunk_kernel<BITS, DP>;
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
  cfg.gridDim = dim3((unsigned)(flat * c.g.kvh), (unsigned)c.nsplit); cfg.blockDim = dim3(PC_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, c);
  if (e != cudaSuccess || c.nsplit == 1) return e;
  cfg.gridDim = dim3((unsigned)(flat * c.g.kvh), 16); cfg.blockDim = dim3(256); cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, chunk_join_kernel, c);
}

// keys: what a sequence's new tokens see at most; alike: every sequence can have max_q new tokens.
int wv_launch_attn_chunk(PaCall c, int bits, long long keys, bool alike, cudaStream_t st) {
  const long long each = ((long long)c.b.max_q * c.group + 255) / 256, upto = (long long)c.b.total_q * c.group / 256 + c.b.num_seqs;
  const long long flat = alike || c.b.num_seqs * each < upto ? c.b.num_seqs * each : upto, blocks = flat * c.g.kvh;
  if (blocks * 256 > INT_MAX) { wv_set_error("wv_attn_paged_dev: %lld tiles of rows are too many", blocks); return WV_ESHAPE; }
  // Splits of the keys where the blocks do not fill the chip: the number that costs least in waves of blocks, each worth its key
  // tiles and some four more of start and end.
  const long long tiles = (keys + PC_N - 1) / PC_N, sms = wv_sm_count();
  long long best = 1, cost = -1;
  for (long long ns = 1; ns <= 16 && ns <= tiles; ns++) {      // 16: chunk_join_kernel's room for weights
    if (ns > 1 && blocks * 256 * ns * (c.g.hd + 2) * 4 > PA_SCRATCH) break;
    const long long t = (tiles + ns - 1) / ns, w = (blocks * ns + sms - 1) / sms * (t + 4 + (ns > 1 ? 2 : 0));
    if (cost < 0 || w < cost) { cost = w; best = ns; }
  }
  long long t = tiles > 0 ? (tiles + best - 1) / best : 1;
  c.per = (int)(t * PC_N > INT_MAX / 2 ? INT_MAX / 2 / PC_N * PC_N : t * PC_N);
  c.nsplit = tiles > 0 ? (int)((tiles + t - 1) / t) : 1;
  WvLease lease;
  if (c.nsplit > 1) {
    const size_t n = (size_t)blocks * 256 * c.nsplit;
    if (const int rc = wv_lease(lease, n * (2 + c.g.hd), st, "wv_attn_paged_dev: the splits' results")) return rc;
    c.ml = reinterpret_cast<float2*>(lease.p);
    c.acc = lease.p + 2 * n;
  }
  const bool small = c.g.hd <= 64;
  const cudaError_t e = bits == 16 ? (small ? chunk_go<16, 64>(c, flat, st) : chunk_go<16, 128>(c, flat, st))
                      : bits == 8 ? (small ? chunk_go<8, 64>(c, flat, st) : chunk_go<8, 128>(c, flat, st))
                                  : (small ? chunk_go<4, 64>(c, flat, st) : chunk_go<4, 128>(c, flat, st));
  if (e != cudaSuccess) { wv_set_error("wv_attn_paged_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA; }
  return WV_OK;
}
