// The paged key/value cache: rows rounded to 16, 8 or 4 bits as they are written, with the rotary embedding of Q and K in the same
// pass, and read back. include/welvet_cuda.h (WvKvPages) defines layout and arithmetic.
//
// Bound: HBM for prompts, latency for single tokens. A CTA takes one token or two (their angles are the same for all heads), a warp
// a kv head's K and V and four query heads at a time, all of them under way at once; a lane holds four consecutive values of each row
// (and four more beyond 128): float4 in, 8 / 4 / 2 bytes of codes out, and a row's maximum is one reduction away. With heads of 128 the
// value that a value is turned with comes from the lane 16 away; loading it a second time took 135 us for the prompts below. Two tokens
// share the chain of loads that finds a token's place (its sequence, length, page) and fill the CTA with their angles.
//
// Prompts of 9900 tokens together, 32 query heads and 8 kv heads of 128, 8 bits, written and read back: 118 us, 4.4 TB/s; neither DRAM
// (52 %) nor issue (56 %) is full, a CTA asks for a token's rows and then waits for them.
// One token: 5.7 us; 200 tokens in 4 bits: 9.0 us (two launches each, captured in a graph; called one by one, the host's part of the
// two calls makes it 13 us for either).
#include "wv_paged.cuh"
#include <float.h>
#include <math.h>
#include <string.h>

#define KVC_WARPS 8
// The prompts' times in us with other settings: 3 blocks 129, 5 blocks 134 (of 122 with 4); 2 heads 128 (122); 3, 4 and 6 tokens 119, 122, 124
// (119); 2 rows 118 (117).
#define KVC_BLOCKS 4            // an SM: 64 registers
#define KVC_HEADS 4             // query heads of a warp at a time, heads of 128; else 2
#define KVR_ROWS 4              // rows that a warp reads back at a time
#define KVC_TOKENS 2            // of a CTA, where there are enough of them

// theta^(2 d / head_dim) for every pair, computed on the host once per (theta, head_dim) and passed by value.
struct WvRopeFreq { double p[128]; };

// A token's place: its sequence's page table says which page and slot; no page (block < 0) before position 0 or on a page number
// outside the pool.
struct KvPlace { int pos; long long page; int slot; };
__device__ __forceinline__ KvPlace kv_place(const WvKvGeom& g, const WvKvBatch& b, int row, int* err) {
  KvPlace p{0, -1, 0};
  const int s = wv_seq_of_row(b, row);
  if (s >= b.num_seqs) { p.pos = INT_MIN; return p; }
  const WvSeq q = wv_seq(b, g.page, s, err);
  if (row < q.q0 || row >= q.q1) { p.pos = INT_MIN; return p; }
  p.pos = q.p0 + (row - q.q0);
  if (p.pos < 0) return p;
  const int i = p.pos / g.page, id = b.pages[(size_t)s * b.table_stride + i];
  p.slot = p.pos - i * g.page;
  if (id < 0 || id >= g.num_pages) wv_paged_report(err, WV_PAGED_PAGE);
  else p.page = id;
  return p;
}

// a * c - b * s with c and s in two float32 pieces each: the products' errors by fma, the sum's by Knuth's two-sum, so that the
// result is the float64 expression's, rounded, but for one in some 10^7. (float64 itself issues at half the float32 rate here and its
// conversions at a sixteenth.) Two values at a time; ns is -s. Where an operand is not finite, neither is the result, and rot64 has
// to say which one it is.
__device__ __forceinline__ float2 rot2(float2 a, float2 b, float2 ch, float2 cl, float2 nsh, float2 nsl) {
  const float2 m1 = make_float2(-1.f, -1.f);
  const float2 p = __fmul2_rn(a, ch), q = __fmul2_rn(b, nsh);
  const float2 pe = __ffma2_rn(a, ch, __fmul2_rn(p, m1)), qe = __ffma2_rn(b, nsh, __fmul2_rn(q, m1));
  const float2 t = __fadd2_rn(__ffma2_rn(a, cl, pe), __ffma2_rn(b, nsl, qe));
  const float2 s = __fadd2_rn(p, q), z = __ffma2_rn(p, m1, s);
  const float2 e = __fadd2_rn(__ffma2_rn(__ffma2_rn(z, m1, s), m1, p), __ffma2_rn(z, m1, q));
  return __fadd2_rn(s, __fadd2_rn(e, t));
}
__device__ __noinline__ float rot64(float a, float b, float ch, float cl, float nsh, float nsl) {
  return (float)((double)a * ((double)ch + (double)cl) + (double)b * ((double)nsh + (double)nsl));
}
// rint(x / s) of the float32 quotient for |x / s| < 2^22, as the low bits of the result: the product with the reciprocal is off by
// two units in the last place at most, so the division is only needed near the middle between two whole numbers.
__device__ __forceinline__ unsigned kv_round(float x, float s, float inv) {
  const float magic = 12582912.f;                                  // 1.5 2^23: the sum's last bit is 1
  const float q = x * inv;
  float m = __fadd_rn(q, magic);
  if (fabsf(fabsf(q - __fsub_rn(m, magic)) - 0.5f) < 1.f / 4096.f) m = __fadd_rn(__fdiv_rn(x, s), magic);
  return __float_as_uint(m);
}

// One row of V4 x 4 x 32 values at most: lane l holds 4 l .. 4 l + 3 (and 128 + those), lanes past head_dim hold zeros.
template <int BITS, int V4, bool FULL>
__device__ __forceinline__ void kv_store_row(const WvKvGeom& g, unsigned char* block, bool is_v, int slot, const float (&x)[V4][4], int lane) {
  unsigned m = 0;                  // the largest magnitude's bits; infinities and NaN are above all others
#pragma unroll
  for (int i = 0; i < V4; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) m = max(m, __float_as_uint(x[i][e]) & 0x7fffffffu);
  unsigned mg[V4];                 // 4 bits: of the four lanes that share a group of 16
#pragma unroll
  for (int i = 0; i < V4; i++) {
    mg[i] = 0;
    if (BITS == 4) {
#pragma unroll
      for (int e = 0; e < 4; e++) mg[i] = max(mg[i], __float_as_uint(x[i][e]) & 0x7fffffffu);
      mg[i] = max(mg[i], __shfl_xor_sync(0xffffffffu, mg[i], 1));
      mg[i] = max(mg[i], __shfl_xor_sync(0xffffffffu, mg[i], 2));
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  const bool fine = m < 0x7f800000u;
  const float a = __uint_as_float(m);
  float s;
  if (BITS == 16) s = __uint_as_float((unsigned)max((int)(m >> 23) - 14, 1) << 23);   // a subnormal has exponent 0: the smallest scale
  else s = fmaxf(__fmul_rn(a, BITS == 8 ? 1.f / 127.f : 1.f / 1785.f), FLT_MIN);
  const float inv = __fdiv_rn(1.f, s);                             // 16 bits: a power of two (s <= 2^113), exact
  unsigned char* codes = block + (is_v ? g.page * g.code : 0) + slot * g.code;
#pragma unroll
  for (int i = 0; i < V4; i++) {
    const int d = 4 * (lane + 32 * i);
    if (!FULL && d >= g.hd) break;
    if (BITS == 16) {
      __half2 h[2] = {__floats2half2_rn(fine ? x[i][0] * inv : 0.f, fine ? x[i][1] * inv : 0.f),
                      __floats2half2_rn(fine ? x[i][2] * inv : 0.f, fine ? x[i][3] * inv : 0.f)};
      *reinterpret_cast<uint2*>(codes + 2 * d) = make_uint2(*reinterpret_cast<unsigned*>(&h[0]), *reinterpret_cast<unsigned*>(&h[1]));
    } else if (BITS == 8) {
      unsigned c[4];
#pragma unroll
      for (int e = 0; e < 4; e++) c[e] = fine ? kv_round(x[i][e], s, inv) : 0u;
      *reinterpret_cast<unsigned*>(codes + d) = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    } else {
      const float t = fine ? fminf(fmaxf(ceilf(__fdiv_rn(__fmul_rn(__uint_as_float(mg[i]), 1.f / 7.f), s)), 1.f), 255.f) : 1.f;
      const float st = __fmul_rn(s, t), ist = __fdiv_rn(1.f, st);
      unsigned w = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int c = fine ? (int)(kv_round(x[i][e], st, ist) - 0x4b400000u) : 0;
        w |= (unsigned)(min(max(c, -7), 7) + 8) << (4 * e);
      }
      *reinterpret_cast<unsigned short*>(codes + d / 2) = (unsigned short)w;
      if ((lane & 3) == 0) block[(is_v ? g.vsub : g.ksub) + slot * (g.hd / 16) + d / 16] = (unsigned char)t;
    }
  }
  if (lane == 0) *reinterpret_cast<float*>(block + (is_v ? g.vscale : g.kscale) + 4 * slot) = fine ? s : __uint_as_float(0x7fc00000u);
}

// grid (tokens / TOK, pieces of a token's rows). FULL: head_dim is 128.
template <int BITS, int V4, int TOK, bool FULL>
__global__ void __launch_bounds__(32 * KVC_WARPS, V4 == 1 ? KVC_BLOCKS : 2) kv_write_kernel(const WvKvGeom g, const WvKvBatch b, const float* __restrict__ k, int ldk,
                                                                  const float* __restrict__ v, int ldv, const float* q, int ldq, float* q_out,
                                                                  int ldqo, int heads, int rotate, const __grid_constant__ WvRopeFreq freq,
                                                                  int* __restrict__ err) {
  __shared__ __align__(16) float s_cs[TOK][4][128];      // cos and sin of a pair, in two pieces each
  __shared__ KvPlace s_at[TOK];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int row0 = blockIdx.x * TOK, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hd = FULL ? 128 : g.hd, half = hd >> 1;
  if (warp < TOK) {
    KvPlace p{INT_MIN, -1, 0};      // a row that no sequence owns
    if (row0 + warp < b.total_q) p = kv_place(g, b, row0 + warp, err);
    if (lane == 0) s_at[warp] = p;
  }
  __syncthreads();
  if (rotate) {
    for (int i = threadIdx.x; i < TOK * half; i += 32 * KVC_WARPS) {
      const int t = TOK == 1 ? 0 : i / half, d = i - t * half;
      if (s_at[t].pos == INT_MIN) continue;
      double c, s;
      sincos((double)s_at[t].pos / freq.p[d], &s, &c);
      s_cs[t][0][d] = (float)c; s_cs[t][1][d] = (float)(c - (double)(float)c);
      s_cs[t][2][d] = (float)s; s_cs[t][3][d] = (float)(s - (double)(float)s);
    }
    __syncthreads();
  }
  constexpr int U = FULL ? KVC_HEADS : 2;
  const int gw = blockIdx.y * KVC_WARPS + warp, nw = gridDim.y * KVC_WARPS;
  for (int tok = 0; tok < TOK; tok++) {
    const KvPlace at = s_at[tok];
    if (at.pos == INT_MIN) continue;
    const size_t row = row0 + tok;
    // the lane's angles, for all rows of the token: cos, and the sine's negative in the first half of a row (a c - b s), itself in
    // the second (with b the first one's value, a c + b s)
    float2 cs[V4][4][2];
    if (rotate) {
#pragma unroll
      for (int i = 0; i < V4; i++) {
        const int d = 4 * (lane + 32 * i);
#pragma unroll
        for (int p = 0; p < 4; p++) {
          const float4 c = (FULL || d < hd) ? *reinterpret_cast<const float4*>(&s_cs[tok][p][d < half ? d : d - half]) : make_float4(0.f, 0.f, 0.f, 0.f);
          const float f = p < 2 || d >= half ? 1.f : -1.f;
          cs[i][p][0] = make_float2(f * c.x, f * c.y); cs[i][p][1] = make_float2(f * c.z, f * c.w);
        }
      }
    }
    auto load = [&](const float* src, float (&x)[V4][4], bool on) {
#pragma unroll
      for (int i = 0; i < V4; i++) {
        const int d = 4 * (lane + 32 * i);
        const float4 o = on && (FULL || d < hd) ? *reinterpret_cast<const float4*>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
        x[i][0] = o.x; x[i][1] = o.y; x[i][2] = o.z; x[i][3] = o.w;
      }
    };
    // what x is turned with: the value half a head away, which another lane holds
    auto partners = [&](const float* src, const float (&x)[V4][4], float (&w)[V4][4], bool on) {
#pragma unroll
      for (int i = 0; i < V4; i++) {
        if (FULL) {
#pragma unroll
          for (int e = 0; e < 4; e++) w[i][e] = __shfl_xor_sync(0xffffffffu, x[i][e], 16);
        } else {
          const int d = 4 * (lane + 32 * i);
          const float4 o = on && d < hd ? *reinterpret_cast<const float4*>(src + (d < half ? d + half : d - half)) : make_float4(0.f, 0.f, 0.f, 0.f);
          w[i][0] = o.x; w[i][1] = o.y; w[i][2] = o.z; w[i][3] = o.w;
        }
      }
    };
    auto turn = [&](float (&x)[V4][4], const float (&w)[V4][4]) {
#pragma unroll
      for (int i = 0; i < V4; i++) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float2 v = rot2(make_float2(x[i][e], x[i][e + 1]), make_float2(w[i][e], w[i][e + 1]), cs[i][0][e / 2], cs[i][1][e / 2], cs[i][2][e / 2], cs[i][3][e / 2]);
          y[e] = v.x; y[e + 1] = v.y;
        }
        if (!(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))) <= FLT_MAX) || y[0] + y[1] + y[2] + y[3] != y[0] + y[1] + y[2] + y[3]) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float2 *c = &cs[i][0][e / 2];
            if (!(fabsf(y[e]) <= FLT_MAX)) y[e] = e & 1 ? rot64(x[i][e], w[i][e], c[0].y, c[2].y, c[4].y, c[6].y) : rot64(x[i][e], w[i][e], c[0].x, c[2].x, c[4].x, c[6].x);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; e++) x[i][e] = y[e];
      }
    };
    // a kv head's K and V, the last warps first: with few tokens they have no query heads. They are under way while Q is turned.
    const int hk = nw - 1 - gw;
    const bool kv = at.page >= 0 && hk < g.kvh;
    float x[V4][4], y[V4][4];
    load(k + row * ldk + (size_t)hk * hd, x, kv);
    load(v + row * ldv + (size_t)hk * hd, y, kv);
    // U query heads at a time
    for (int h = U * gw; h < heads; h += U * nw) {
      float z[U][V4][4], w[FULL ? 1 : U][V4][4];
      const float* src = q + row * ldq + (size_t)h * hd;
#pragma unroll
      for (int u = 0; u < U; u++) {
        load(src + u * hd, z[u], h + u < heads);
        if (!FULL && rotate) partners(src + u * hd, z[u], w[FULL ? 0 : u], h + u < heads);
      }
      __syncwarp();                 // in place: every lane has its partner's value
      float* dst = q_out + row * ldqo + (size_t)h * hd;
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (h + u >= heads) break;
        if (FULL && rotate) partners(src, z[u], w[0], true);
        if (rotate) turn(z[u], w[FULL ? 0 : u]);
#pragma unroll
        for (int i = 0; i < V4; i++) {
          const int d = 4 * (lane + 32 * i);
          if ((FULL || d < hd)) *reinterpret_cast<float4*>(dst + u * hd + d) = make_float4(z[u][i][0], z[u][i][1], z[u][i][2], z[u][i][3]);
        }
      }
    }
    if (!kv) continue;
    for (int h = hk; h < g.kvh; h += nw) {
      const float* src = k + row * ldk + (size_t)h * hd;
      if (h != hk) {
        load(src, x, true);
        load(v + row * ldv + (size_t)h * hd, y, true);
      }
      if (rotate) {
        float w[V4][4];
        partners(src, x, w, true);
        turn(x, w);
      }
      unsigned char* block = g.pool + ((size_t)at.page * g.kvh + h) * g.block;
      kv_store_row<BITS, V4, FULL>(g, block, false, at.slot, x, lane);
      kv_store_row<BITS, V4, FULL>(g, block, true, at.slot, y, lane);
    }
  }
}

template <int BITS, int V4, int TOK>
__global__ void __launch_bounds__(32 * KVC_WARPS) kv_read_kernel(const WvKvGeom g, const WvKvBatch b, float* __restrict__ k, int ldk,
                                                                 float* __restrict__ v, int ldv, int* __restrict__ err) {
  __shared__ KvPlace s_at[TOK];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int row0 = blockIdx.x * TOK, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp < TOK) {
    KvPlace p{INT_MIN, -1, 0};
    if (row0 + warp < b.total_q) p = kv_place(g, b, row0 + warp, err);
    if (lane == 0) s_at[warp] = p;
  }
  __syncthreads();
  const int nr = 2 * g.kvh;
  // KVR_ROWS rows of a warp at a time: their loads are all under way before the first is stored
  const int step = gridDim.y * KVC_WARPS;
  for (int r0 = blockIdx.y * KVC_WARPS + warp; r0 < TOK * nr; r0 += KVR_ROWS * step) {
    float* dst[KVR_ROWS];
    float s[KVR_ROWS];
    uint2 w[KVR_ROWS][V4];
    int t[KVR_ROWS][V4];
#pragma unroll
    for (int u = 0; u < KVR_ROWS; u++) {
      const int i0 = r0 + u * step, tok = TOK == 1 ? 0 : i0 / nr, r = i0 - tok * nr;
      dst[u] = nullptr;
      if (i0 >= TOK * nr || s_at[tok].pos == INT_MIN) continue;
      const KvPlace at = s_at[tok];
      const size_t row = row0 + tok;
      const bool is_v = r >= g.kvh;
      const int h = is_v ? r - g.kvh : r;
      dst[u] = (is_v ? v + row * ldv : k + row * ldk) + (size_t)h * g.hd;
      const unsigned char* block = g.pool + ((size_t)max(at.page, 0LL) * g.kvh + h) * g.block;
      const unsigned char* codes = block + (is_v ? g.page * g.code : 0) + at.slot * g.code;
      s[u] = at.page < 0 ? 0.f : *reinterpret_cast<const float*>(block + (is_v ? g.vscale : g.kscale) + 4 * at.slot);
#pragma unroll
      for (int i = 0; i < V4; i++) {
        const int d = 4 * (lane + 32 * i);
        w[u][i] = make_uint2(BITS == 4 ? 0x8888u : 0u, 0u);              // no page: zeros
        t[u][i] = 0;
        if (d >= g.hd || at.page < 0) continue;
        if (BITS == 16) w[u][i] = *reinterpret_cast<const uint2*>(codes + 2 * d);
        if (BITS == 8) w[u][i].x = *reinterpret_cast<const unsigned*>(codes + d);
        if (BITS == 4) {
          w[u][i].x = *reinterpret_cast<const unsigned short*>(codes + d / 2);
          t[u][i] = block[(is_v ? g.vsub : g.ksub) + at.slot * (g.hd / 16) + d / 16];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < KVR_ROWS; u++) {
      if (!dst[u]) continue;
#pragma unroll
      for (int i = 0; i < V4; i++) {
        const int d = 4 * (lane + 32 * i);
        if (d >= g.hd) break;
        float c[4];
        if (BITS == 16) {
          const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&w[u][i].x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&w[u][i].y));
          c[0] = lo.x; c[1] = lo.y; c[2] = hi.x; c[3] = hi.y;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (BITS == 8) c[e] = (float)(int)(signed char)(w[u][i].x >> (8 * e));
          if (BITS == 4) c[e] = (float)(((int)((w[u][i].x >> (4 * e)) & 15u) - 8) * t[u][i]);
        }
        *reinterpret_cast<float4*>(dst[u] + d) = make_float4(s[u] * c[0], s[u] * c[1], s[u] * c[2], s[u] * c[3]);
      }
    }
  }
}

int wv_sm_count();
// Enough CTAs for the chip where there are few tokens; with many, a CTA for KVC_TOKENS of them.
static int kvc_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* at, int tokens, int rows, cudaStream_t st) {
  const int ctas = KVC_BLOCKS * wv_sm_count();
  const int tok = tokens / KVC_TOKENS >= ctas ? KVC_TOKENS : 1;
  const int most = (rows + KVC_WARPS - 1) / KVC_WARPS, want = ctas / tokens;
  cfg.gridDim = dim3((tokens + tok - 1) / tok, want < 1 ? 1 : (want > most ? most : want));
  cfg.blockDim = dim3(32 * KVC_WARPS); cfg.stream = st;
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at; cfg.numAttrs = 1;
  return tok;
}

int wv_launch_kv_write(const WvKvPages& kv, const WvKvBatch& b, const float* dk, int ldk, const float* dv, int ldv, const float* dq, int ldq,
                       float* dq_out, int ldqo, int heads, double theta, cudaStream_t st) {
  const WvKvGeom g = wv_kv_geom(kv);
  static thread_local WvRopeFreq freq;
  static thread_local double freq_theta = 0.0;
  static thread_local int freq_hd = 0;
  if (theta > 0.0 && (freq_theta != theta || freq_hd != g.hd)) {
    for (int d = 0; d < g.hd / 2; d++) freq.p[d] = pow(theta, (double)(2 * d) / (double)g.hd);
    freq_theta = theta; freq_hd = g.hd;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  const bool many = kvc_config(cfg, at, b.total_q, (2 * g.kvh + heads + 1) / 2, st) > 1;      // two rows a warp
  auto go = [&](auto kern) { return cudaLaunchKernelEx(&cfg, kern, g, b, dk, ldk, dv, ldv, dq, ldq, dq_out, ldqo, heads, theta > 0.0 ? 1 : 0, freq, wv_paged_err_ptr()); };
  cudaError_t e;
#define KVC_GO(V4_, TOK_, FULL_) (kv.bits == 16 ? go(kv_write_kernel<16, V4_, TOK_, FULL_>) : kv.bits == 8 ? go(kv_write_kernel<8, V4_, TOK_, FULL_>) : go(kv_write_kernel<4, V4_, TOK_, FULL_>))
  if (g.hd > 128) e = many ? KVC_GO(2, KVC_TOKENS, false) : KVC_GO(2, 1, false);
  else if (g.hd == 128) e = many ? KVC_GO(1, KVC_TOKENS, true) : KVC_GO(1, 1, true);
  else e = many ? KVC_GO(1, KVC_TOKENS, false) : KVC_GO(1, 1, false);
#undef KVC_GO
  if (e != cudaSuccess) { wv_set_error("wv_kv_write_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA; }
  return WV_OK;
}

int wv_launch_kv_read(const WvKvPages& kv, const WvKvBatch& b, float* dk, int ldk, float* dv, int ldv, cudaStream_t st) {
  const WvKvGeom g = wv_kv_geom(kv);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  const bool many = kvc_config(cfg, at, b.total_q, 2 * g.kvh, st) > 1;
  auto go = [&](auto kern) { return cudaLaunchKernelEx(&cfg, kern, g, b, dk, ldk, dv, ldv, wv_paged_err_ptr()); };
  cudaError_t e;
#define KVC_GO(V4_, TOK_) (kv.bits == 16 ? go(kv_read_kernel<16, V4_, TOK_>) : kv.bits == 8 ? go(kv_read_kernel<8, V4_, TOK_>) : go(kv_read_kernel<4, V4_, TOK_>))
  if (g.hd > 128) e = many ? KVC_GO(2, KVC_TOKENS) : KVC_GO(2, 1);
  else e = many ? KVC_GO(1, KVC_TOKENS) : KVC_GO(1, 1);
#undef KVC_GO
  if (e != cudaSuccess) { wv_set_error("wv_kv_read_dev: launch: %s", cudaGetErrorString(cudaGetLastError())); return WV_ECUDA; }
  return WV_OK;
}

// ------------------------------------------------------------------ C ABI: the calls' checks
int wv_api_bind_device();
int wv_launch_attn_paged(const WvKvPages& kv, const WvKvBatch& b, const float* dq, int ldq, float* dout, int ldo, int heads, float scale,
                         int window, cudaStream_t st);
int wv_launch_attn_shared(const WvKvPages& kv, const WvKvBatch& b, const WvKvGroups& share, const float* dq, int ldq, float* dout, int ldo, int heads, float scale,
                          cudaStream_t st);

extern "C" int wv_kv_block_bytes(int bits, int page_size, int head_dim, uint64_t* bytes) {
  if (!bytes) { wv_set_error("wv_kv_block_bytes: null pointer"); return WV_EARG; }
  if (bits != 16 && bits != 8 && bits != 4) { wv_set_error("wv_kv_block_bytes: %d bits (16, 8 or 4)", bits); return WV_EFORMAT; }
  if (!wv_kv_shape_ok(bits, page_size, head_dim)) { wv_set_error("wv_kv_block_bytes: page_size %d, head_dim %d (multiples of 16, head_dim at most 256)", page_size, head_dim); return WV_ESHAPE; }
  WvKvPages p = {nullptr, bits, 1, page_size, 1, head_dim};
  *bytes = (uint64_t)wv_kv_geom(p).block;
  return WV_OK;
}

// What the three calls check alike. 1: nothing to do (no rows).
static int kv_check(const char* who, const WvKvPages* kv, const WvKvBatch* b) {
  if (!kv || !b || !kv->pool || !b->q_start || !b->kv_len || !b->pages) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  if (kv->bits != 16 && kv->bits != 8 && kv->bits != 4) { wv_set_error("%s: %d bits (16, 8 or 4)", who, kv->bits); return WV_EFORMAT; }
  if (!wv_kv_shape_ok(kv->bits, kv->page_size, kv->head_dim) || kv->num_pages < 1 || kv->num_kv_heads < 1) {
    wv_set_error("%s: %d pages of %d, %d kv heads of %d (page_size and head_dim are multiples of 16, head_dim at most 256)", who, kv->num_pages, kv->page_size,
                 kv->num_kv_heads, kv->head_dim);
    return WV_ESHAPE;
  }
  if (reinterpret_cast<uintptr_t>(kv->pool) & 15) { wv_set_error("%s: the pool is not 16-byte aligned", who); return WV_EARG; }
  if (b->num_seqs < 1 || b->table_stride < 0 || b->total_q < 0 || b->max_q < 0 || b->max_kv < 0) { wv_set_error("%s: a negative or zero count in the batch", who); return WV_EARG; }
  if ((long long)b->max_kv > (long long)b->table_stride * kv->page_size) {
    wv_set_error("%s: max_kv %d does not fit %d pages of %d", who, b->max_kv, b->table_stride, kv->page_size); return WV_ESHAPE;
  }
  return b->total_q == 0 || b->max_q == 0 ? 1 : WV_OK;
}
static int kv_rows(const char* who, const char* name, const void* p, int* ld, long long width) {
  if (!p) { wv_set_error("%s: %s is null", who, name); return WV_EARG; }
  if (width > INT_MAX) { wv_set_error("%s: rows of %lld values", who, width); return WV_ESHAPE; }
  if (*ld == 0) *ld = (int)width;
  if (*ld < width || (*ld & 3)) { wv_set_error("%s: the row stride of %s is %d for %lld values (a multiple of 4)", who, name, *ld, width); return WV_ESHAPE; }
  if (reinterpret_cast<uintptr_t>(p) & 15) { wv_set_error("%s: %s is not 16-byte aligned", who, name); return WV_EARG; }
  return WV_OK;
}

extern "C" int wv_kv_write_dev(const WvKvPages* kv, const WvKvBatch* batch, const float* dk, int ldk, const float* dv, int ldv,
                               const float* dq, int ldq, float* dq_out, int ldqo, int num_heads, double theta, void* stream) {
  const char* who = "wv_kv_write_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = kv_check(who, kv, batch)) < 0) return rc;
  const bool none = rc == 1;
  const long long kw = (long long)kv->num_kv_heads * kv->head_dim, qw = (long long)num_heads * kv->head_dim;
  if ((rc = kv_rows(who, "k", dk, &ldk, kw)) || (rc = kv_rows(who, "v", dv, &ldv, kw))) return rc;
  if (dq || dq_out) {
    if (num_heads < 1) { wv_set_error("%s: %d heads", who, num_heads); return WV_ESHAPE; }
    if ((rc = kv_rows(who, "q", dq, &ldq, qw)) || (rc = kv_rows(who, "q_out", dq_out, &ldqo, qw))) return rc;
    if (dq == dq_out && ldq != ldqo) { wv_set_error("%s: q in place with two strides", who); return WV_EARG; }
  } else {
    num_heads = 0;
  }
  if (!(theta == theta)) { wv_set_error("%s: theta is NaN", who); return WV_EARG; }
  if (none) return WV_OK;
  return wv_launch_kv_write(*kv, *batch, dk, ldk, dv, ldv, dq, ldq, dq_out, ldqo, num_heads, theta, static_cast<cudaStream_t>(stream));
}

extern "C" int wv_kv_read_dev(const WvKvPages* kv, const WvKvBatch* batch, float* dk, int ldk, float* dv, int ldv, void* stream) {
  const char* who = "wv_kv_read_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = kv_check(who, kv, batch)) < 0) return rc;
  const bool none = rc == 1;
  const long long kw = (long long)kv->num_kv_heads * kv->head_dim;
  if ((rc = kv_rows(who, "k", dk, &ldk, kw)) || (rc = kv_rows(who, "v", dv, &ldv, kw))) return rc;
  if (none) return WV_OK;
  return wv_launch_kv_read(*kv, *batch, dk, ldk, dv, ldv, static_cast<cudaStream_t>(stream));
}

extern "C" int wv_attn_paged_dev(const WvKvPages* kv, const WvKvBatch* batch, const float* dq, int ldq, float* dout, int ldo, int num_heads,
                                 float scale, int window, void* stream) {
  const char* who = "wv_attn_paged_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = kv_check(who, kv, batch)) < 0) return rc;
  const bool none = rc == 1;
  if (num_heads < 1 || num_heads % kv->num_kv_heads) { wv_set_error("%s: %d heads over %d kv heads", who, num_heads, kv->num_kv_heads); return WV_ESHAPE; }
  if (!(scale == scale) || scale - scale != 0.f) { wv_set_error("%s: the scale is not finite", who); return WV_EARG; }
  if (batch->max_kv > 1 << 30) { wv_set_error("%s: max_kv %d (at most 2^30)", who, batch->max_kv); return WV_ESHAPE; }
  const long long qw = (long long)num_heads * kv->head_dim;
  if ((rc = kv_rows(who, "q", dq, &ldq, qw)) || (rc = kv_rows(who, "out", dout, &ldo, qw))) return rc;
  if (none) return WV_OK;
  if (window < 0 || window >= batch->max_kv) window = 0;              // wider than any sequence: none
  return wv_launch_attn_paged(*kv, *batch, dq, ldq, dout, ldo, num_heads, scale, window, static_cast<cudaStream_t>(stream));
}

extern "C" int wv_attn_shared_dev(const WvKvPages* kv, const WvKvBatch* batch, const WvKvGroups* groups, const float* dq, int ldq, float* dout, int ldo,
                                  int num_heads, float scale, void* stream) {
  const char* who = "wv_attn_shared_dev";
  int rc = wv_api_bind_device();
  if (rc < 0) return rc;
  if ((rc = kv_check(who, kv, batch)) < 0) return rc;
  const bool none = rc == 1;
  if (!groups) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  if (groups->num_groups < 0 || groups->num_groups > batch->num_seqs || groups->max_shared < 0) {
    wv_set_error("%s: %d groups of %d sequences, %d tokens shared", who, groups->num_groups, batch->num_seqs, groups->max_shared); return WV_EARG;
  }
  if (groups->num_groups > 0 && (!groups->start || !groups->shared)) { wv_set_error("%s: null pointer", who); return WV_EARG; }
  if (num_heads < 1 || num_heads % kv->num_kv_heads) { wv_set_error("%s: %d heads over %d kv heads", who, num_heads, kv->num_kv_heads); return WV_ESHAPE; }
  if (!(scale == scale) || scale - scale != 0.f) { wv_set_error("%s: the scale is not finite", who); return WV_EARG; }
  if (batch->max_kv > 1 << 30) { wv_set_error("%s: max_kv %d (at most 2^30)", who, batch->max_kv); return WV_ESHAPE; }
  const long long qw = (long long)num_heads * kv->head_dim;
  if ((rc = kv_rows(who, "q", dq, &ldq, qw)) || (rc = kv_rows(who, "out", dout, &ldo, qw))) return rc;
  if (none) return WV_OK;
  return wv_launch_attn_shared(*kv, *batch, *groups, dq, ldq, dout, ldo, num_heads, scale, static_cast<cudaStream_t>(stream));
}
