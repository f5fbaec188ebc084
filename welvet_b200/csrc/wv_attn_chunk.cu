// Attention of many new tokens of a sequence over the paged cache (prompts and pieces of them) on tcgen05.
//
// A block takes 256 rows (tokens x query heads of one kv head, so that a cached row is read once for the group) as two tiles of 128
// and walks the keys, 128 at a time, with a running maximum:
//   S = Q K^T    Q (two float16 pieces, hi and lo) and K in shared memory, S in tensor memory       2 x 128 x 128 x head_dim products
//   P            weights in two float16 pieces, written over S, 32 keys a piece pair                 one row a thread
//   O_j = P V    P out of tensor memory, V in shared memory, keys being V's rows                     2 x 128 x head_dim x 128
// O is summed up over the key tiles in registers (128 float32 a row): the tensor core cuts instead of rounding as it adds, which over
// thousands of keys would show, a tile's 128 do not; and the maximum's correction is a factor in that sum instead of a pass over
// tensor memory. Codes are exact in float16, so with hi and lo the products carry 22 bits: float32's accuracy costs two products
// where 16-bit activations would take one, which is what bounds the kernel (the tensor pipe runs 4096 cycles for 256 x 128 x
// head_dim 128, the weights take some 1300 a tile on the other pipes, and the two tiles take turns).
//
// Roles: two warpgroups own a tile each (a thread a row: maximum, weights, sums), one warp issues the MMAs, three fill the ring of
// three stages, K and V tiles in turn, turning 8- and 4-bit codes into float16 on the way (16-bit ones are copied asynchronously).
// Codes of 4 bits lie in the order in which they unpack two at a time (0 4 1 5 2 6 3 7); Q follows, and the outputs are put back.
//
// A key's scale multiplies its column of S; a value row's, relative to the largest of its tile, its weight, and the tile's own power
// of two goes into the sum over tiles. Where the scales in a tile lie further apart than the pieces' range holds (2^16), the tile's
// weighted sum is taken value by value in float32 instead.
//
// Every wait is bounded: when one runs out the block records a code, all roles leave their loops, and tensor memory is released
// after the MMAs in flight (waited for, bounded again).
#include "wv_attn_paged.cuh"
#include "wv_tma_common.cuh"
#include "wv_lease.h"
#include <type_traits>

#define PC_THREADS 384
#define PC_M 128                    // rows of a tile
#define PC_N 128                    // keys of a tile
#define PC_STAGES 3
#define PC_PRODUCERS 96
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
__device__ __forceinline__ void pc_st32(unsigned taddr, const unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), PC_W8(r, 0), PC_W8(r, 8), PC_W8(r, 16), PC_W8(r, 24) : "memory");
}
__device__ __forceinline__ unsigned pc_ld1(unsigned taddr) {
  unsigned v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
  pc_wait_ld();
  return v;
}
template <int N> __device__ __forceinline__ void pc_regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void pc_regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Shared memory: Q [tile][piece][head_dim / 64][128 rows][128 bytes], the ring of K and V tiles [head_dim / 64][128 keys][128 bytes],
// then this.
struct PcMeta {
  float kk[2][PC_N], fv[2][PC_N];           // of a key tile (two of them in turn): the keys' scales times q's, the value rows' scales over 2^e
  float beta[2];                            // 2^e
  unsigned flags[2];                        // 1: some key of the tile is not there, 2: value scales too far apart
  unsigned valid[2][4];                     // which keys are there
  unsigned long long bar[2 * PC_STAGES + 11];
  unsigned tmem, qmax;
  int abort;
  int seq, tile;
};

// The flat-th tile of 256 rows of the sequences that have more than rows_most rows, found by a whole warp: its sequence (-1: none)
// and its place in it, the later tokens, which see most, first.
__device__ __forceinline__ void pc_find(const PaCall& c, int flat, int* err, int& seq, int& tile) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  seq = -1; tile = 0;
  for (int s0 = 0; s0 < c.b.num_seqs && seq < 0; s0 += 32) {
    int n = 0;
    if (s0 + lane < c.b.num_seqs) {
      const WvSeq q = wv_seq(c.b, c.g.page, s0 + lane, err);
      const long long rows = (long long)(q.q1 - q.q0) * c.group;
      n = rows > c.rows_most && q.q1 - q.q0 <= c.b.max_q ? (int)((rows + 255) / 256) : 0;
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > flat);
    if (hit) {
      const int at = __ffs(hit) - 1;
      seq = s0 + at;
      tile = before + __shfl_sync(0xffffffffu, upto, at) - 1 - flat;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

template <int BITS> __device__ __forceinline__ int pc_dim(int p) {      // the value that stands at place p of a row
  if constexpr (BITS == 4) return (p & ~7) | ((p & 7) >> 1) | (p & 1) << 2;
  return p;
}

template <int BITS, int DP>
__global__ void __launch_bounds__(PC_THREADS, 1) attn_chunk_kernel(const __grid_constant__ PaCall c) {
  constexpr int HALVES = DP / 64, STAGE = HALVES * PC_N * 128, QPIECE = HALVES * PC_M * 128;
  constexpr unsigned IDESC_S = (1u << 4) | (PC_N / 8 << 17) | (PC_M / 16 << 24);                   // f32 sums, f16 operands, both K-major
  constexpr unsigned IDESC_O = (1u << 4) | (1u << 16) | (DP / 8 << 17) | (PC_M / 16 << 24);        // B with its columns innermost
  extern __shared__ __align__(1024) unsigned char pc_smem[];
  unsigned char* s_q = pc_smem;
  unsigned char* s_kv = pc_smem + 4 * QPIECE;
  PcMeta& M = *reinterpret_cast<PcMeta*>(s_kv + PC_STAGES * STAGE);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  auto full = [&](int s) { return smem_u32(&M.bar[s]); };
  auto empty = [&](int s) { return smem_u32(&M.bar[PC_STAGES + s]); };
  auto s_full = [&](int t) { return smem_u32(&M.bar[2 * PC_STAGES + t]); };
  auto p_full = [&](int t) { return smem_u32(&M.bar[2 * PC_STAGES + 2 + t]); };
  auto o_full = [&](int t) { return smem_u32(&M.bar[2 * PC_STAGES + 4 + t]); };
  auto m_full = [&](int s) { return smem_u32(&M.bar[2 * PC_STAGES + 6 + s]); };
  auto m_empty = [&](int s) { return smem_u32(&M.bar[2 * PC_STAGES + 8 + s]); };
  const unsigned done = smem_u32(&M.bar[2 * PC_STAGES + 10]);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (smem_u32(pc_smem) & 1023u) { if (tid == 0) atomicCAS_system(c.err - 1, 0, 799); return; }    // the swizzle counts from 1024-byte boundaries

  // ---------------------------------------------------------------- which rows: tiles of 256 of the sequences that have more than rows_most
  const int kvh = blockIdx.x % c.g.kvh, flat = blockIdx.x / c.g.kvh, sp = blockIdx.y;
  if (warp == 0) {
    int seq, tile;
    pc_find(c, flat, blockIdx.x == 0 && sp == 0 ? c.err : nullptr, seq, tile);
    if (lane == 0) { M.seq = seq; M.tile = tile; M.qmax = 0; M.abort = 0; }
  }
  __syncthreads();
  const int seq = M.seq;
  if (seq < 0) return;
  const WvSeq sq = wv_seq(c.b, c.g.page, seq, sp == 0 && kvh == 0 ? c.err : nullptr);
  const int nrows = (sq.q1 - sq.q0) * c.group, r0 = M.tile * 256, rn = min(256, nrows - r0);
  int lo, hi;
  pa_range(sq, r0 / c.group, (r0 + rn - 1) / c.group, c.window, lo, hi);
  const int k0 = lo + sp * c.per, k1 = min(hi, k0 + c.per);
  const int hd = c.g.hd, pos0 = sq.kv - (sq.q1 - sq.q0);
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
    for (int s = 0; s < PC_STAGES; s++) { mbar_init(full(s), PC_PRODUCERS / 32); mbar_init(empty(s), 1); }
    for (int t = 0; t < 2; t++) {
      mbar_init(s_full(t), 1); mbar_init(p_full(t), 4); mbar_init(o_full(t), 1);
      mbar_init(m_full(t), 1); mbar_init(m_empty(t), two ? 8 : 4);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 11) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&M.tmem)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // ---------------------------------------------------------------- Q: a common power of two, two pieces, the operand's layout
  auto qrow = [&](int r) { return c.q + (size_t)(sq.q0 + (r0 + r) / c.group) * c.ldq + (size_t)(kvh * c.group + (r0 + r) % c.group) * hd; };
  {
    unsigned m = 0;
    for (int r = warp; r < rn; r += PC_THREADS / 32) {
      const float* src = qrow(r);
      for (int d = 4 * lane; d < hd; d += 128) {
        const float4 v = *reinterpret_cast<const float4*>(src + d);
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; e++) { const unsigned u = __float_as_uint(x[e]) & 0x7fffffffu; if (u < 0x7f800000u) m = max(m, u); }
      }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) atomicMax(&M.qmax, m);
  }
  pc_fence_before();
  __syncthreads();
  pc_fence_after();
  const unsigned tmem = __shfl_sync(0xffffffffu, *(volatile unsigned*)&M.tmem, 0);
  const int qe = min(max((int)(M.qmax >> 23) - 127 - 13, -100), 114);
  const float qinv = __uint_as_float((unsigned)(127 - qe) << 23);
  const float qf = c.scale * __uint_as_float((unsigned)(127 + qe) << 23);
  for (int i = tid; i < 256 * (DP / 8); i += PC_THREADS) {               // 8 places of a row at a time
    const int r = i / (DP / 8), j = i % (DP / 8);
    if (r >= PC_M && !two) break;
    unsigned h[4] = {0u, 0u, 0u, 0u}, l[4] = {0u, 0u, 0u, 0u};
    if (r < rn && 8 * j < hd) {
      const float* src = qrow(r) + 8 * j;
      const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
      float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = x[e] - x[e] == 0.f ? x[e] * qinv : NAN;
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

  if (warp < 8) {
    // ============================================================== a tile's rows: weights and sums, a thread a row
    pc_regs_up<216>();
    const int t = warp >> 2, row = tid & (PC_M - 1), r = t * PC_M + row;
    if (t == 0 || two) {
      const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
      const unsigned ts = tmem + lanes + t * PC_N, to = tmem + lanes + 256 + t * 128;
      const int prow = pos0 + (r0 + min(r, rn - 1)) / c.group;
      const int pmin = pos0 + (r0 + t * PC_M) / c.group, pmax = pos0 + (r0 + min(t * PC_M + PC_M, rn) - 1) / c.group;
      float o[DP], m = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int d = 0; d < DP; d++) o[d] = 0.f;
      bool ok = true;
      for (int j = 0; j < n; j++) {
        const int ms = j & 1, key0 = k0 + j * PC_N;
        if (!mbar_wait(m_full(ms), (j >> 1) & 1, PC_SPIN) || !mbar_wait(s_full(t), j & 1, PC_SPIN)) { if (!dead()) fail(700 + t); ok = false; }
        if (__any_sync(0xffffffffu, !ok)) { ok = false; break; }
        pc_fence_after();
        const float* kk = M.kk[ms];
        const float* fv = M.fv[ms];
        float beta = M.beta[ms], alpha;
        const unsigned flags = M.flags[ms];
        const bool masked = (flags & 1u) || key0 + PC_N - 1 > pmin || key0 + PC_N > k1 || (c.window != 0 && key0 <= pmax - c.window);
        // bit k of `see`: the row sees key 32 q + k of the tile
        unsigned see[4];
        if (masked) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            const int a = key0 + 32 * q, last = min(prow, k1 - 1) - a, first = c.window ? prow - c.window + 1 - a : 0;
            unsigned w = last < 0 ? 0u : last >= 31 ? ~0u : (2u << last) - 1u;
            if (first > 0) w &= first > 31 ? 0u : ~0u << first;
            see[q] = w & M.valid[ms][q];
          }
        }
        // ---- the maximum over the tile
        float mx = m;
        if (!masked) {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            unsigned s[32];
            pc_ld32(ts + 32 * q, s);
            pc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 k4 = *reinterpret_cast<const float4*>(kk + 32 * q + i);
              const float2 a = __fmul2_rn(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), make_float2(k4.x, k4.y));
              const float2 b = __fmul2_rn(make_float2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), make_float2(k4.z, k4.w));
              mx = fmaxf(mx, fmaxf(fmaxf(a.x, a.y), fmaxf(b.x, b.y)));
            }
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; q++) {
            unsigned s[32];
            pc_ld32(ts + 32 * q, s);
            pc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i++) if ((see[q] >> i) & 1u) mx = fmaxf(mx, __uint_as_float(s[i]) * kk[32 * q + i]);
          }
        }
        const float ref = mx == -INFINITY ? 0.f : mx;
        alpha = pa_ex2(m - ref);                                         // 0 while there was nothing
        m = mx;
        l2 = __fmul2_rn(l2, make_float2(alpha, alpha));
        const float2 off = make_float2(PA_LIFT - ref, PA_LIFT - ref);
        if (flags & 2u) {
          // ---- value by value in float32; P is zero
          const int e = 2 * j + 1;
          if (!mbar_wait(full(e % PC_STAGES), (e / PC_STAGES) & 1, PC_SPIN)) { if (!dead()) fail(702); ok = false; }
          if (__any_sync(0xffffffffu, !ok)) { ok = false; break; }
          const unsigned char* v = s_kv + (e % PC_STAGES) * STAGE;
#pragma unroll
          for (int d = 0; d < DP; d++) o[d] *= alpha;
          alpha = 1.f;
#pragma unroll 1
          for (int k = 0; k < PC_N; k++) {
            const float x = __uint_as_float(pc_ld1(ts + k)) * kk[k];
            const unsigned word = k < 32 ? see[0] : k < 64 ? see[1] : k < 96 ? see[2] : see[3];
            const bool on = !masked || ((word >> (k & 31)) & 1u);
            const float p = on ? pa_ex2(x + off.x) : 0.f, w = on ? p * fv[k] * beta : 0.f;
            l2.x += p;
#pragma unroll
            for (int g = 0; g < DP / 8; g++) {
              const uint4 q = *reinterpret_cast<const uint4*>(v + (g >> 3) * PC_N * 128 + k * 128 + (((g & 7) ^ (k & 7)) << 4));
              const float2 a = pa_unpack(q.x), b = pa_unpack(q.y), d = pa_unpack(q.z), f = pa_unpack(q.w);
              o[8 * g] += w * a.x; o[8 * g + 1] += w * a.y; o[8 * g + 2] += w * b.x; o[8 * g + 3] += w * b.y;
              o[8 * g + 4] += w * d.x; o[8 * g + 5] += w * d.y; o[8 * g + 6] += w * f.x; o[8 * g + 7] += w * f.y;
            }
          }
          beta = 0.f;
          unsigned z[32];
#pragma unroll
          for (int i = 0; i < 32; i++) z[i] = 0u;
#pragma unroll
          for (int q = 0; q < 4; q++) pc_st32(ts + 32 * q, z);
        } else {
          // ---- weights: 32 keys of S become 16 columns of their hi pieces and 16 of their lo pieces
          auto weights = [&](auto some) {
#pragma unroll
            for (int q = 0; q < 4; q++) {
              unsigned s[32], w[32];
              pc_ld32(ts + 32 * q, s);
              pc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(kk + 32 * q + i), f4 = *reinterpret_cast<const float4*>(fv + 32 * q + i);
#pragma unroll
                for (int u = 0; u < 4; u += 2) {
                  const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[i + u]), __uint_as_float(s[i + u + 1])), u ? make_float2(k4.z, k4.w) : make_float2(k4.x, k4.y), off);
                  float2 p = make_float2(pa_ex2(x.x), pa_ex2(x.y));
                  float2 pf = __fmul2_rn(p, u ? make_float2(f4.z, f4.w) : make_float2(f4.x, f4.y));
                  if constexpr (decltype(some)::value) {
                    const bool a = (see[q] >> (i + u)) & 1u, b = (see[q] >> (i + u + 1)) & 1u;
                    p = make_float2(a ? p.x : 0.f, b ? p.y : 0.f);
                    pf = make_float2(a ? pf.x : 0.f, b ? pf.y : 0.f);
                  }
                  l2 = __fadd2_rn(l2, p);
                  const unsigned h = pa_pack(pf.x, pf.y);
                  const float2 back = pa_unpack(h);
                  w[(i + u) / 2] = h;
                  w[16 + (i + u) / 2] = pa_pack(pf.x - back.x, pf.y - back.y);
                }
              }
              pc_st32(ts + 32 * q, w);
            }
          };
          if (masked) weights(std::true_type()); else weights(std::false_type());
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        pc_fence_before();
        __syncwarp();
        if (lane == 0) { mbar_arrive(p_full(t)); mbar_arrive(m_empty(ms)); }
        // ---- this tile's part of the sum
        if (!mbar_wait(o_full(t), j & 1, PC_SPIN)) { if (!dead()) fail(704 + t); ok = false; }
        if (__any_sync(0xffffffffu, !ok)) { ok = false; break; }
        pc_fence_after();
#pragma unroll
        for (int q = 0; q < DP / 32; q++) {
          unsigned s[32];
          pc_ld32(to + 32 * q, s);
          pc_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 a = __fmul2_rn(make_float2(o[32 * q + i], o[32 * q + i + 1]), make_float2(alpha, alpha));
            const float2 v = __ffma2_rn(make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), make_float2(beta, beta), a);
            o[32 * q + i] = v.x; o[32 * q + i + 1] = v.y;
          }
        }
      }
      const float l = l2.x + l2.y;
      if (r < rn) {
        float f = 1.f;
        float* dst;
        if (c.nsplit > 1) {
          dst = c.acc + ((rec0 + r) * c.nsplit + sp) * hd;
          c.ml[(rec0 + r) * c.nsplit + sp] = make_float2(m, l);
        } else {
          dst = c.out + (size_t)(sq.q0 + (r0 + r) / c.group) * c.ldo + (size_t)(kvh * c.group + (r0 + r) % c.group) * hd;
          f = l == 0.f ? 0.f : 1.f / l;
        }
#pragma unroll
        for (int g = 0; g < DP / 8; g++) {
          if (8 * g < hd) {
            float x[8];
#pragma unroll
            for (int p = 0; p < 8; p++) x[pc_dim<BITS>(p)] = ok ? (c.nsplit > 1 ? o[8 * g + p] : o[8 * g + p] * f) : NAN;
            *reinterpret_cast<float4*>(dst + 8 * g) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(dst + 8 * g + 4) = make_float4(x[4], x[5], x[6], x[7]);
          }
        }
      }
    }
  } else {
    pc_regs_down<72>();
    if (warp == 11) {
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
          const unsigned kb = kv + (e % PC_STAGES) * STAGE;
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
          const unsigned vb = kv + (e % PC_STAGES) * STAGE;
#pragma unroll
          for (int p = 1; p >= 0; p--)
#pragma unroll
            for (int k = 0; k < PC_N / 16; k++)
              pc_mma_ts(tmem + 256 + t * 128, tmem + t * PC_N + (k >> 1) * 32 + p * 16 + (k & 1) * 8, pc_desc(vb + k * 2048, PC_N * 128), IDESC_O, !(p == 1 && k == 0));
          pc_commit(o_full(t));
        }
        __syncwarp();
      };
      auto release = [&](int e) { if (leader) pc_commit(empty(e % PC_STAGES)); __syncwarp(); };
      if (wait(full(0), 0, 710)) {
        pc_fence_after();
        for (int t = 0; t < nt; t++) scores(t, 0);
        release(0);
      }
      for (int j = 0; j < n && ok; j++) {
        const int ev = 2 * j + 1, ek = 2 * j + 2;
        if (!wait(full(ev % PC_STAGES), ev / PC_STAGES, 711)) break;
        for (int t = 0; t < nt && ok; t++) {
          if (!wait(p_full(t), j, 712 + t)) break;
          pc_fence_after();
          values(t, ev);
          if (t == nt - 1) release(ev);
          if (j + 1 < n) {
            if (t == 0 && !wait(full(ek % PC_STAGES), ek / PC_STAGES, 714)) break;
            pc_fence_after();
            scores(t, ek);
            if (t == nt - 1) release(ek);
          }
        }
      }
      if (!ok) {                                                         // what was issued has to end before tensor memory is given back
        if (leader) pc_commit(done);
        __syncwarp();
        mbar_wait(done, 0, PC_SPIN);
      }
    } else {
      // ============================================================ K and V tiles
      const int pw = warp - 8, pt = tid - 256;                           // 0 .. 2, 0 .. 95
      const int code = c.g.code, page = c.g.page;
      constexpr int PER = BITS == 16 ? DP / 8 : DP / 16;                 // pieces of a row: 16 bytes of codes (8 in 4 bits)
      const int pieces = BITS == 16 ? hd / 8 : hd / 16;
      bool ok = true;
      for (int e = 0; e < 2 * n && ok; e++) {
        const int j = e >> 1, key0 = k0 + j * PC_N, s = e % PC_STAGES;
        const bool is_v = e & 1;
        // page numbers of the tile's 8 groups of 16 keys, a lane each
        int id = -1;
        if (lane < 8 && key0 + 16 * lane < k1) {
          id = c.b.pages[(size_t)seq * c.b.table_stride + (key0 + 16 * lane) / page];
          if (id < 0 || id >= c.g.num_pages) { if (pw == 0) wv_paged_report(c.err, WV_PAGED_PAGE); id = -1; }
        }
        const int slot = (key0 + 16 * min(lane, 7)) % page;
        if (e >= PC_STAGES && !mbar_wait(empty(s), (e / PC_STAGES - 1) & 1, PC_SPIN)) { if (!dead()) fail(720); ok = false; }
        if (!is_v && pw == 0 && j >= 2 && ok && !mbar_wait(m_empty(j & 1), ((j >> 1) - 1) & 1, PC_SPIN)) { if (!dead()) fail(721); ok = false; }
        if (__any_sync(0xffffffffu, !ok || dead())) { ok = false; break; }
        if (!is_v && pw == 0) {
          // what the weights need: four keys a lane
          const int ms = j & 1, gi = lane >> 2, gid = __shfl_sync(0xffffffffu, id, gi), gs = __shfl_sync(0xffffffffu, slot, gi) + 4 * (lane & 3);
          float4 ks = make_float4(0.f, 0.f, 0.f, 0.f), vs = ks;
          if (gid >= 0) {
            const unsigned char* block = c.g.pool + ((size_t)gid * c.g.kvh + kvh) * c.g.block;
            ks = *reinterpret_cast<const float4*>(block + c.g.kscale + 4 * gs);
            vs = *reinterpret_cast<const float4*>(block + c.g.vscale + 4 * gs);
          }
          const float kx[4] = {ks.x, ks.y, ks.z, ks.w}, vx[4] = {vs.x, vs.y, vs.z, vs.w};
          int emax = -90, emin = 1000;
          bool there = gid >= 0;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int ex = min((int)((__float_as_uint(vx[i]) >> 23) & 255u) - 127, 100);
            if (there && key0 + 4 * lane + i < k1 && vx[i] == vx[i] && ex > -90) { emax = max(emax, ex); emin = min(emin, ex); }
          }
          emax = __reduce_max_sync(0xffffffffu, emax);
          emin = __reduce_min_sync(0xffffffffu, emin);
          const float down = __uint_as_float((unsigned)(127 - emax) << 23);
          *reinterpret_cast<float4*>(&M.kk[ms][4 * lane]) = make_float4(kx[0] * qf, kx[1] * qf, kx[2] * qf, kx[3] * qf);
          *reinterpret_cast<float4*>(&M.fv[ms][4 * lane]) = make_float4(vx[0] * down, vx[1] * down, vx[2] * down, vx[3] * down);
          const unsigned have = __ballot_sync(0xffffffffu, there);       // a bit for 4 keys; 4 lanes of a group alike
          if (lane < 4) {
            unsigned w = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) if ((have >> (8 * lane + i)) & 1u) w |= 15u << (4 * i);
            M.valid[ms][lane] = w;
          }
          if (lane == 0) {
            M.beta[ms] = __uint_as_float((unsigned)(127 + emax) << 23);
            M.flags[ms] = (have != ~0u ? 1u : 0u) | (emin < emax - 16 ? 2u : 0u);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(m_full(ms));
        }
        unsigned char* dst = s_kv + s * STAGE;
        const int part = is_v ? page * code : 0;
        if constexpr (BITS == 16) {
          for (int i = pt; i < PC_N * PER; i += PC_PRODUCERS) {
            const int r = i / PER, x = i % PER;
            const int gid = __shfl_sync(0xffffffffu, id, r >> 4), gs = __shfl_sync(0xffffffffu, slot, r >> 4);
            const bool on = gid >= 0 && key0 + r < k1 && x < pieces;
            const unsigned char* src = c.g.pool + ((size_t)max(gid, 0) * c.g.kvh + kvh) * c.g.block + part + (on ? (gs + (r & 15)) * code + 16 * x : 0);
            const unsigned to = smem_u32(dst) + (x >> 3) * PC_N * 128 + r * 128 + (((x & 7) ^ (r & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(on ? 16 : 0) : "memory");
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
          constexpr int B = 4;                                           // pieces in flight a thread
          const int sub = is_v ? c.g.vsub : c.g.ksub, n16 = hd / 16;
          for (int i0 = pt; i0 < PC_N * PER; i0 += B * PC_PRODUCERS) {
            uint4 w[B];
            unsigned t[B];
            bool on[B];
#pragma unroll
            for (int u = 0; u < B; u++) {
              const int i = i0 + u * PC_PRODUCERS, r = min(i / PER, PC_N - 1), x = i % PER;
              const int gid = __shfl_sync(0xffffffffu, id, r >> 4), gs = __shfl_sync(0xffffffffu, slot, r >> 4) + (r & 15);
              on[u] = i < PC_N * PER && gid >= 0 && key0 + r < k1 && x < pieces;
              const unsigned char* block = c.g.pool + ((size_t)max(gid, 0) * c.g.kvh + kvh) * c.g.block;
              if constexpr (BITS == 8) {
                if (on[u]) w[u] = *reinterpret_cast<const uint4*>(block + part + gs * code + 16 * x);
              } else {
                if (on[u]) {
                  const uint2 v = *reinterpret_cast<const uint2*>(block + part + gs * code + 8 * x);
                  w[u].x = v.x; w[u].y = v.y;
                  t[u] = block[sub + gs * n16 + x];
                }
              }
            }
#pragma unroll
            for (int u = 0; u < B; u++) {
              const int i = i0 + u * PC_PRODUCERS, r = i / PER, x = i % PER;
              if (i >= PC_N * PER) break;
              unsigned v[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
              if (on[u]) {
                if constexpr (BITS == 8) {
                  const unsigned q[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
                  for (int k = 0; k < 4; k++) { const unsigned b = q[k] ^ 0x80808080u; v[2 * k] = pa_bytes<0x4140>(b); v[2 * k + 1] = pa_bytes<0x4342>(b); }
                } else {
                  const unsigned q[2] = {w[u].x, w[u].y};
                  const PaSub t2 = pa_pair(t[u], t[u]);
#pragma unroll
                  for (int k = 0; k < 8; k++) v[k] = pa_nibbles(q[k >> 2], k & 3, t2);
                }
              }
              unsigned char* at = dst + (x >> 2) * PC_N * 128 + r * 128;
              *reinterpret_cast<uint4*>(at + ((((2 * x) & 7) ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
              *reinterpret_cast<uint4*>(at + ((((2 * x + 1) & 7) ^ (r & 7)) << 4)) = make_uint4(v[4], v[5], v[6], v[7]);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(full(s));
      }
    }
  }
  pc_fence_before();
  __syncthreads();
  if (warp == 11) {
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
    pc_find(c, blockIdx.x / c.g.kvh, nullptr, seq, tile);
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
  constexpr size_t smem = (size_t)(DP / 64) * 128 * (4 * PC_M + PC_STAGES * PC_N) + sizeof(PcMeta);
  static_assert(smem <= 227 * 1024, "shared memory");
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

// keys: what a sequence's new tokens see at most; alike: every sequence has max_q new tokens.
int wv_launch_attn_chunk(PaCall c, int bits, long long keys, bool alike, cudaStream_t st) {
  const long long each = ((long long)c.b.max_q * c.group + 255) / 256, upto = (long long)c.b.total_q * c.group / 256 + c.b.num_seqs;
  const long long flat = alike || c.b.num_seqs * each < upto ? c.b.num_seqs * each : upto, blocks = flat * c.g.kvh;
  if (blocks * 256 > INT_MAX) { wv_set_error("wv_attn_paged_dev: %lld tiles of rows are too many", blocks); return WV_ESHAPE; }
  // Splits of the keys where the blocks do not fill the chip: the number that costs least in waves of blocks, each worth its key
  // tiles and some four more of start and end.
  const long long tiles = (keys + PC_N - 1) / PC_N, sms = wv_sm_count();
  long long best = 1, cost = -1;
  for (long long ns = 1; ns <= 16 && ns <= tiles; ns++) {      // 16: chunk_join_kernel's room for weights
    if (ns > 1 && blocks * 256 * ns * (c.g.hd + 2) * 4 > (256LL << 20)) break;
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
