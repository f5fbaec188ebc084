// What the kernels of the paged attention share: the weights' units, the split results and their merge.
//
// A key's logit is x = scale log2(e) q.k, its weight 2^x, its value row v = f 2^E c with c the codes and 2^E the largest value scale's power
// of two among the keys at hand. What goes through the tensor cores is 2^(x - m) f in two float16 pieces (22 bits), the divisor is
// sum 2^(x - m) in float32. m follows the running maximum of x and may lie 2^7 (few rows) or 2^10 (chunks) below it; both sums carry a
// factor, 2^6 and 2^4, that uses the float16 range and cancels. With f below 2 a weight is at most 2^14 and 2^15, and what rounds away of
// one is below 2^-30 and 2^-28 of the largest.
#pragma once
#include "wv_paged.cuh"
#include <math.h>

#define PA_SCRATCH (256LL << 20)        // bytes that a call may keep for its splits' results

struct PaCall {
  WvKvGeom g;
  WvKvBatch b;
  const float* q; int ldq;
  float* out; int ldo;
  int group;                       // query heads of one kv head
  float scale;                     // times log2(e)
  int window;                      // 0: none
  unsigned one;                    // 0x3c003c00, for pa_nibbles
  int rows_most;                   // sequences with more rows (tokens x group) than this go to the chunk kernel (0: all that have any)
  int nsplit, per;                 // splits of a sequence's keys, keys of a split (a multiple of 16; of 128 for chunks)
  unsigned tiles, first, kept;     // few rows: tiles of a sequence (0: see pa_find), the launch's first block of rows, rows of a block with split results
  float2* ml;                      // split results [row][nsplit]: {M, divisor}; {-inf, 0} and no sums for a split without keys
  float* acc;                      // [row][nsplit][head_dim]
  int* err;
  // wv_attn_shared_dev alone: groups of sequences whose first keys are the same pages. A launch takes those of all groups (part 1) or every
  // sequence's own behind them (part 2); a row, token * heads + head, has nslots results, the launch's from slot0 on. Where the same kernel takes
  // both they are one launch: its first `split` blocks are part 1, the others part 2 with what own_ says.
  WvKvGroups share;
  int part, slot0, nslots;
  unsigned split, own_tiles;
  int own_per, own_nsplit, own_slot0;
};

__device__ __forceinline__ float pa_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ unsigned pa_pack(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ float2 pa_unpack(unsigned v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }

__device__ __forceinline__ unsigned pa_sub2(unsigned v, unsigned m) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&m));
  return *reinterpret_cast<const unsigned*>(&r);
}
__device__ __forceinline__ unsigned pa_mul2(unsigned v, unsigned m) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&m));
  return *reinterpret_cast<const unsigned*>(&r);
}
// Integer bytes or nibbles become float16 without a conversion: a byte in the mantissa of 1024, then 1024 + offset is subtracted.
// The low two (SEL 0x4140) or high two (0x4342) bytes of w, biased by 128, as signed values.
template <unsigned SEL> __device__ __forceinline__ unsigned pa_bytes(unsigned w) { return pa_sub2(__byte_perm(w, 0x64646464u, SEL), 0x64806480u); }
// Nibbles j and j + 4 of w, biased by 8, times the sub-scales t (a pair of float16): the nibble n in the upper mantissa of 1 is
// 1 + n / 16, and (1 + n / 16) 16 t - 24 t = (n - 8) t is exact in one instruction. `one` is that 1 twice, PaCall::one: a constant that
// the compiler cannot see, so that it masks and merges in one instruction with it in a register.
struct PaSub { unsigned a, b; };
__device__ __forceinline__ unsigned pa_nibbles(unsigned w, int j, const PaSub& t, unsigned one) {
  const unsigned s = j == 0 ? w << 6 : j == 1 ? w << 2 : j == 2 ? w >> 2 : w >> 6, x = (s & 0x03c003c0u) | one;
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&t.a), *reinterpret_cast<const __half2*>(&t.b));
  return *reinterpret_cast<const unsigned*>(&r);
}
// Two sub-scales (bytes) as the factors of pa_nibbles.
__device__ __forceinline__ PaSub pa_pair(unsigned a, unsigned b) {
  const unsigned t = pa_sub2(0x64006400u | a | (b << 16), 0x64006400u);
  return PaSub{pa_mul2(t, 0x4c004c00u), pa_mul2(t, 0xce00ce00u)};        // 16 t and -24 t
}


// The positions that a block of consecutive rows of a sequence sees: [lo, hi), lo cut down to a multiple of 16. The first row may stand
// before position 0, where p0 - window has no room in 32 bits for the widest windows. A split's first key lo + split * per may lie past
// hi; with at most 2^30 cached tokens it stays below 2^32, and k0 + per of a split with keys below 2^31.
__device__ __forceinline__ void pa_range(const WvSeq& s, int tok0, int tok1, int window, int& lo, int& hi) {
  const int p0 = s.p0 + tok0;
  hi = max(0, s.p0 + tok1 + 1);
  lo = window > 0 ? max(0, max(p0, 0) - window + 1) & ~15 : 0;
}

// The flat-th tile of `size` rows (tokens x group) of the sequences that have more than `above` rows, found by a whole warp: its sequence
// (-1: none) and its place in it, the later tokens, which see most, first. With err it reads on through all sequences and reports.
__device__ __forceinline__ void pa_find(const PaCall& c, int flat, int size, int above, int* err, int& seq, int& tile) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  seq = -1; tile = 0;
  for (int s0 = 0; s0 < c.b.num_seqs && (seq < 0 || err); s0 += 32) {
    int n = 0;
    if (s0 + lane < c.b.num_seqs) {
      const WvSeq q = wv_seq(c.b, c.g.page, s0 + lane, err);
      const long long rows = (long long)(q.q1 - q.q0) * c.group;
      n = rows > above ? (int)((rows + size - 1) / size) : 0;
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > flat);
    if (hit && seq < 0) {
      const int at = __ffs(hit) - 1;
      seq = s0 + at;
      tile = before + __shfl_sync(0xffffffffu, upto, at) - 1 - flat;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

// ------------------------------------------------------------------ shared prefixes
// The sequences [s0, s1) of group g, cut to the batch, and how many tokens they are said to share.
struct PaGroup { int s0, s1, n; };
__device__ __forceinline__ PaGroup pa_group(const PaCall& c, int g, int* err) {
  PaGroup r;
  const int a = c.share.start[g], e = c.share.start[g + 1], n = c.share.shared[g];
  r.s0 = min(max(a, 0), c.b.num_seqs);
  r.s1 = min(max(e, r.s0), c.b.num_seqs);
  r.n = min(max(n, 0), c.share.max_shared);
  if (r.s0 != a || r.s1 != e || r.n != n) wv_paged_report(err, WV_PAGED_LENGTH);
  return r;
}
// By a whole warp: the keys that the group's rows all see and that lie in whole pages, which is what they share, and the first of its sequences
// with new tokens, whose row of the table says where they are. 128 sequences are loaded at once.
__device__ __forceinline__ int pa_shared_keys(const PaCall& c, const PaGroup& r, int& table) {
  const int lane = threadIdx.x & 31;
  int n = r.n, first = INT_MAX;
  for (int s0 = r.s0; s0 < r.s1; s0 += 128) {
    WvSeq q[4];
#pragma unroll
    for (int u = 0; u < 4; u++) q[u] = wv_seq(c.b, c.g.page, min(s0 + 32 * u + lane, r.s1 - 1), nullptr);
#pragma unroll
    for (int u = 0; u < 4; u++)
      if (q[u].q1 > q[u].q0) { n = min(n, max(q[u].p0 + 1, 0)); first = min(first, min(s0 + 32 * u + lane, r.s1 - 1)); }
  }
  n = __reduce_min_sync(0xffffffffu, n);
  first = __reduce_min_sync(0xffffffffu, first);
  table = first == INT_MAX ? 0 : first;
  return first == INT_MAX ? 0 : n / c.g.page * c.g.page;
}
// What sequence seq shares with its group (0: it has none), by a whole warp.
__device__ __forceinline__ int pa_shared_of(const PaCall& c, int seq) {
  const int lane = threadIdx.x & 31;
  for (int g0 = 0; g0 < c.share.num_groups; g0 += 32) {
    PaGroup r{0, 0, 0};
    if (g0 + lane < c.share.num_groups) r = pa_group(c, g0 + lane, nullptr);
    const unsigned m = __ballot_sync(0xffffffffu, r.s0 <= seq && seq < r.s1);
    if (!m) continue;
    const int at = __ffs(m) - 1;
    r = PaGroup{__shfl_sync(0xffffffffu, r.s0, at), __shfl_sync(0xffffffffu, r.s1, at), __shfl_sync(0xffffffffu, r.n, at)};
    int table;
    return pa_shared_keys(c, r, table);
  }
  return 0;
}
// The flat-th tile of `size` rows (tokens x group) of the groups, as pa_find: false if there is none, else its place in its group, the group, the
// rows [q0, q1) of its sequences' new tokens.
__device__ __forceinline__ bool pa_find_group(const PaCall& c, int flat, int size, int* err, PaGroup& group, int& q0, int& q1, int& tile) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  bool found = false;
  for (int g0 = 0; g0 < c.share.num_groups && (!found || err); g0 += 32) {
    PaGroup r{0, 0, 0};
    int a = 0, e = 0;
    if (g0 + lane < c.share.num_groups) {
      r = pa_group(c, g0 + lane, err);
      a = min(max(c.b.q_start[r.s0], 0), c.b.total_q);
      e = min(max(c.b.q_start[r.s1], a), c.b.total_q);
    }
    const int n = (int)(((long long)(e - a) * c.group + size - 1) / size);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > flat);
    if (hit && !found) {
      const int at = __ffs(hit) - 1;
      found = true;
      group = PaGroup{__shfl_sync(0xffffffffu, r.s0, at), __shfl_sync(0xffffffffu, r.s1, at), __shfl_sync(0xffffffffu, r.n, at)};
      q0 = __shfl_sync(0xffffffffu, a, at); q1 = __shfl_sync(0xffffffffu, e, at);
      tile = flat - before - __shfl_sync(0xffffffffu, upto - n, at);
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return found;
}

// A row out of its splits' results, in two steps. By a whole warp (each of a block's may do it): the splits' weights into w[nsplit];
// returns the divisor's reciprocal. All maxima and divisors are loaded at once: one after the other they were a chain of
// round trips to L2 (33 splits took 12 us).
__device__ __forceinline__ float pa_join_weights(const PaCall& c, size_t rec, int nsplit, float* w) {
  const int lane = threadIdx.x & 31;
  const float2* ml = c.ml + rec * nsplit;
  float M = -INFINITY, L = 0.f;
  for (int s0 = 0; s0 < nsplit; s0 += 128) {
#pragma unroll
    for (int u = 0; u < 4; u++) { const int s = s0 + 32 * u + lane; if (s < nsplit) M = fmaxf(M, ml[s].x); }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float ref = M == -INFINITY ? 0.f : M;
  for (int s = lane; s < nsplit; s += 32) {
    const float2 x = ml[s];
    const float f = x.y == 0.f ? 0.f : x.x == -INFINITY ? 1.f : pa_ex2(x.x - ref);      // -inf with a divisor: NaN, which counts
    if (f != 0.f) L += x.y * f;
    w[s] = f;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  return L == 0.f ? 0.f : 1.f / L;
}
// Values first, first + step, ... of the row: the sums of the splits with weight, in their order, eight loads at a time.
__device__ __forceinline__ void pa_join_sums(const PaCall& c, size_t rec, int nsplit, int token, int head, const float* w, float inv, int first, int step) {
  const float* acc = c.acc + rec * nsplit * c.g.hd;
  float* out = c.out + (size_t)token * c.ldo + (size_t)head * c.g.hd;
  for (int d = first; d < c.g.hd; d += step) {
    float a = 0.f;
    for (int s0 = 0; s0 < nsplit; s0 += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; u++) v[u] = s0 + u < nsplit && w[s0 + u] != 0.f ? acc[(size_t)(s0 + u) * c.g.hd + d] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; u++) if (s0 + u < nsplit) a += v[u] * w[s0 + u];
    }
    out[d] = a * inv;
  }
}

int wv_launch_attn_chunk(PaCall c, int bits, long long keys, bool alike, cudaStream_t st);      // wv_attn_chunk.cu
cudaError_t wv_launch_chunk_part(const PaCall& c, int bits, long long flat, cudaStream_t st);                                // a part of wv_attn_shared_dev
