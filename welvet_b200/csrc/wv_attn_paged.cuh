// What the kernels of the paged attention share: the weights' units, the split results and their merge.
//
// A key's logit is x = scale log2(e) q.k, its weight 2^x, its value row v = f 2^e c with c the codes, f in [1, 2) and 2^e the rest of the
// row's scale. What goes through the tensor cores is 2^(x + e - M) f in two float16 pieces (22 bits), M the running maximum of
// x + e over the keys seen so far, so that the largest contribution keeps its bits whatever the scales are; the divisor is
// sum 2^(x - M). e is held to [-90, 100], the rest of a scale beyond that stays in f, so that the divisor's terms stay in range.
// Both sums carry a factor of 2^13 that uses the float16 range and cancels.
#pragma once
#include "wv_paged.cuh"
#include <math.h>

#define PA_LIFT 13.f

struct PaCall {
  WvKvGeom g;
  WvKvBatch b;
  const float* q; int ldq;
  float* out; int ldo;
  int heads, group;                // query heads, and those of one kv head
  float scale;                     // times log2(e)
  int window;                      // 0: none
  int rows_most;                   // sequences with more rows (tokens x group) than this go to the chunk kernel
  int nsplit, per;                 // splits of a sequence's keys, keys of a split (a multiple of 16; of 128 for chunks)
  float2* ml;                      // split results [row][nsplit]: {M, divisor}; {-inf, 0} and no sums for a split without keys
  float* acc;                      // [row][nsplit][head_dim]
  int* err;
};

__device__ __forceinline__ float pa_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// A value row's scale as 2^e f; returns e, sets f and 2^-e.
__device__ __forceinline__ float pa_split_scale(float s, float& f, float& inv) {
  const int e = min(max((int)((__float_as_uint(s) >> 23) & 255u) - 127, -90), 100);
  inv = __uint_as_float((unsigned)(127 - e) << 23);
  f = s * inv;
  return (float)e;
}
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
// Nibbles j and j + 4 of w, biased by 8, times the sub-scale in both halves of t.
__device__ __forceinline__ unsigned pa_nibbles(unsigned w, int j, unsigned t) {
  return pa_mul2(pa_sub2(((w >> (4 * j)) & 0x000f000fu) | 0x64006400u, 0x64086408u), t);
}
// Two bytes as a pair of float16.
__device__ __forceinline__ unsigned pa_pair(unsigned a, unsigned b) { return pa_sub2(0x64006400u | a | (b << 16), 0x64006400u); }


// The positions that a block of consecutive rows of a sequence sees: [lo, hi), lo cut down to a multiple of 16.
__device__ __forceinline__ void pa_range(const WvSeq& s, int tok0, int tok1, int window, int& lo, int& hi) {
  const int p0 = s.kv - (s.q1 - s.q0) + tok0;
  hi = max(0, s.kv - (s.q1 - s.q0) + tok1 + 1);
  lo = window > 0 ? max(0, p0 - window + 1) & ~15 : 0;
}

// One value of a row out of its splits' results, in their order.
__device__ __forceinline__ void pa_join(const PaCall& c, size_t rec, int token, int head, int d) {
  const float2* ml = c.ml + rec * c.nsplit;
  const float* acc = c.acc + rec * c.nsplit * c.g.hd + d;
  float M = -INFINITY, L = 0.f, a = 0.f;
  for (int s = 0; s < c.nsplit; s++) M = fmaxf(M, ml[s].x);
  const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll 4
  for (int s = 0; s < c.nsplit; s++) {
    const float2 x = ml[s];
    if (x.y == 0.f) continue;
    const float w = x.x == -INFINITY ? 1.f : pa_ex2(x.x - ref);          // -inf with a divisor: NaN, which counts
    L += x.y * w;
    a += acc[(size_t)s * c.g.hd] * w;
  }
  c.out[(size_t)token * c.ldo + (size_t)head * c.g.hd + d] = L == 0.f ? 0.f : a / L;
}

int wv_launch_attn_chunk(PaCall c, int bits, long long keys, bool alike, cudaStream_t st);      // wv_attn_chunk.cu
