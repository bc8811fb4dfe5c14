// Tree attention with few rows: one token of decode, or a draft of a token or two
// (n_rep query heads of a KV head times T tokens). The same formula and records as
// attn_tree.cu, whose 128-row tiles would be almost empty here; what counts is how
// soon the last byte of the cache has been asked for.
//
// A warp takes 16 positions at a time and eight rows for its columns, so a tile of
// the two products is one m16n8 tensor-core tile: S^T = K Q^T and O^T = V^T P^T. The
// cache goes from global memory straight into the MMAs' registers. From a Q8_0 cache:
//   * a lane's eight bytes of a block of 32 dims are two k-steps of K's operand (the
//     queries are held in the same order of dims, as fp16 pairs hi + lo);
//   * four bytes of each of four positions, transposed by byte permutes, are two
//     k-steps of V^T's.
// int8 is exact in fp16, so S needs two MMAs (hi, lo) per step and block, the block's
// scale multiplies its sum in float, and P carries the values' scales: P d_v 2^(13 -
// E), again as hi + lo, turned from S's layout into the operand's by an 8 x 8
// transpose. E is the exponent of the row's largest P d_v in the step, so that hi + lo
// holds 22 bits of what counts for this row: a masked position has P = 0 and a scale
// that is NaN is left out, so neither moves E, and a large scale moves it only by
// what its weight leaves of it. (One E a warp, from all scales that it holds, cost
// values of 0.01 beside a masked NaN 2.7e-3.)
//
// From an F32 cache the same tiles as m16n8k8 of tf32, every operand as hi + lo (11
// bits each: 2^-21 of a value is left out) and three MMAs a product; tf32 has float's
// range, so nothing has to be scaled. The queries' planes lie in shared memory, the
// registers are full of cache. A position whose values hold an infinity or a NaN
// counts with zeros, and with a weight of NaN where it is attended to: a masked
// weight, 0, takes nothing from it.
//
// Four warps per CTA, each with its own running maxima, sums and O in registers. The
// CTA's warps meet in shared memory and the CTAs of a cluster in distributed shared
// memory, so up to 16 steps (2048 positions, D <= 64) are one launch; longer caches
// leave one record per cluster for the join.
//
// Bound by latency: a step's loads, its two products, the two reductions and, past
// 2048 positions, the join: one token of 14 / 2 heads of 64 takes 5.8 us at 2000
// positions and 11.5 us at 32000 (8.7 MB of cache, 0.8 TB/s).
#include <algorithm>

#include "attn_tree.cuh"

namespace mi {

namespace {

constexpr int kFewNT = 128;
constexpr int kFewWarps = kFewNT / 32;

// positions that a warp has in registers at a time, in tiles of 16
template <int D, bool Q8>
constexpr int kFewTiles = D <= (Q8 ? 64 : 32) ? 2 : 1;
template <int D, bool Q8>
constexpr int kFewStep = kFewWarps * 16 * kFewTiles<D, Q8>;  // positions of a CTA's step

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo as tf32: hi is cut (a rounded one could leave float's range), lo rounded
// (the MMA drops the bits behind its eleventh).
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi))) + 0x1000u;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Two bytes of b (chosen by `sel` against 0x64), each already offset by 128, as fp16:
// 1024 + (byte + 128) - 1152.
__device__ __forceinline__ uint32_t bytes_to_h2(uint32_t b, uint32_t sel) {
  const uint32_t t = __byte_perm(b, 0x64646464u, sel);
  return h2_bits(__hsub2_rn(*reinterpret_cast<const __half2*>(&t), __floats2half2_rn(1152.0f, 1152.0f)));
}
__device__ __forceinline__ float dsmem_ld(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(dsmem_addr(p, rank)) : "memory");
  return v;
}

template <int D, int NR, bool Q8>
struct FewSmem {
  static constexpr int R = 8 * NR;
  float part[kFewWarps][R][D];  // the warps' O, then (in [0]) the CTA's
  float m[kFewWarps][R], l[kFewWarps][R], scale[kFewWarps][R];
  float cm[R], cl[R];           // the CTA's
  uint4 q[Q8 ? 1 : NR][Q8 ? 1 : D / 32][4][Q8 ? 1 : 32];  // F32: [hi, hi, lo, lo] of a lane's eight dims of each block
};

// What a warp holds of the cache: PT tiles of 16 positions.
template <int D, bool Q8>
struct FewCache;

template <int D>
struct FewCache<D, true> {
  static constexpr int NC = D / 32, ND = (NC + 1) / 2, PT = kFewTiles<D, true>;
  uint2 K[PT][2][NC];                  // positions g, g + 8; eight bytes of each block
  uint32_t V[PT][4][NC];               // positions 2t, 2t + 1, 2t + 8, 2t + 9; four bytes of each block
  uint32_t dk[PT][2][ND], dv[PT][2][ND];  // scales of positions g, g + 8, two a word
  const uint8_t *kq, *vq;
  const uint16_t *ks, *vs;

  __device__ __forceinline__ FewCache(const TreeAttnParams& p, int kvh) {
    const int64_t head = (int64_t)kvh * p.n_ctx, plane = (int64_t)p.HKV * p.n_ctx * D;
    kq = (const uint8_t*)p.cache_k + head * D;
    vq = (const uint8_t*)p.cache_v + head * D;
    ks = (const uint16_t*)((const uint8_t*)p.cache_k + plane) + head * NC;
    vs = (const uint16_t*)((const uint8_t*)p.cache_v + plane) + head * NC;
  }
  static __device__ __forceinline__ void scales(const uint16_t* s, int64_t pos, bool in, uint32_t (&o)[ND]) {
    s += pos * NC;
#pragma unroll
    for (int i = 0; i < ND; i++)
      o[i] = !in ? 0u : NC % 2 == 0 ? *(const uint32_t*)(s + 2 * i) : s[2 * i] | (2 * i + 1 < NC ? (uint32_t)s[2 * i + 1] << 16 : 0u);
  }
  __device__ __forceinline__ void load(int64_t at, int64_t end, int g, int t) {
#pragma unroll
    for (int q = 0; q < PT; q++) {
      const int64_t tp = at + q * 16;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int64_t pos = tp + g + 8 * h;
        const bool in = pos < end;
        scales(ks, pos, in, dk[q][h]);
        scales(vs, pos, in, dv[q][h]);
#pragma unroll
        for (int c = 0; c < NC; c++) K[q][h][c] = in ? *(const uint2*)(kq + pos * D + 32 * c + 8 * t) : make_uint2(0u, 0u);
      }
#pragma unroll
      for (int h = 0; h < 4; h++) {
        const int64_t pos = tp + 2 * t + (h & 1) + 4 * (h & 2);
#pragma unroll
        for (int c = 0; c < NC; c++) V[q][h][c] = pos < end ? *(const uint32_t*)(vq + pos * D + 32 * c + 4 * g) : 0u;
      }
    }
  }
};

template <int D>
struct FewCache<D, false> {
  static constexpr int NC = D / 32, PT = kFewTiles<D, false>;
  float K[PT][2][NC][8];  // positions g, g + 8; eight dims of each block
  float V[PT][4][NC][4];  // positions 2t, 2t + 1, 2t + 8, 2t + 9; four dims of each block
  const float *k, *v;
  int64_t row;

  __device__ __forceinline__ FewCache(const TreeAttnParams& p, int kvh) {
    k = (const float*)p.cache_k + (int64_t)kvh * D;
    v = (const float*)p.cache_v + (int64_t)kvh * D;
    row = (int64_t)p.HKV * D;
  }
  static __device__ __forceinline__ void load4(float* to, const float* from, bool in) {
    const float4 x = in ? *(const float4*)from : make_float4(0.f, 0.f, 0.f, 0.f);
    to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
  }
  __device__ __forceinline__ void load(int64_t at, int64_t end, int g, int t) {
#pragma unroll
    for (int q = 0; q < PT; q++) {
      const int64_t tp = at + q * 16;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int64_t pos = tp + g + 8 * h;
#pragma unroll
        for (int c = 0; c < NC; c++) {
          load4(&K[q][h][c][0], k + pos * row + 32 * c + 8 * t, pos < end);
          load4(&K[q][h][c][4], k + pos * row + 32 * c + 8 * t + 4, pos < end);
        }
      }
#pragma unroll
      for (int h = 0; h < 4; h++) {
        const int64_t pos = tp + 2 * t + (h & 1) + 4 * (h & 2);
#pragma unroll
        for (int c = 0; c < NC; c++) load4(V[q][h][c], v + pos * row + 32 * c + 4 * g, pos < end);
      }
    }
  }
};

// NR: groups of eight rows. Grid (splits, KV heads, groups of 8 NR rows), clusters
// along the splits.
//
// Registers: one group over a Q8_0 cache for 4 CTAs of an SM (3 of 96 and 128 dims; 2
// took 36 us for a token over 32000 positions of 28 / 4 heads of 128, 3 take 24.6); over
// an F32 cache for 3 of 32 dims (16 heads over 2000 positions: 11.5 us with 2, 7.2 with 3).
// Over an F32 cache of 128 dims they do not hold the planes: 192 bytes are spilled with one
// row group and 640 with two (376 of 96 dims with two).
template <int D, int NR, bool Q8>
__global__ void __launch_bounds__(kFewNT, NR > 1 ? 1 : Q8 ? (D <= 64 ? 4 : 3) : D <= 32 ? 3 : 1) attn_few_kernel(const __grid_constant__ TreeAttnParams p, const TreeSplit sp,
                                                          const int cluster) {
  constexpr int NC = D / 32, PT = kFewTiles<D, Q8>, step = kFewStep<D, Q8>;
  extern __shared__ __align__(16) uint8_t few_raw[];
  FewSmem<D, NR, Q8>& sm = *reinterpret_cast<FewSmem<D, NR, Q8>*>(few_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, r0 = blockIdx.z * 8 * NR, rep = p.H / p.HKV;
  const int64_t n_kv = (int64_t)p.n_past + p.T;
  const int64_t begin = (int64_t)blockIdx.x * sp.per * step, end = min(n_kv, begin + (int64_t)sp.per * step);
  FewCache<D, Q8> kv(p, kvh);
  if (begin < end) kv.load(begin + warp * PT * 16, end, g, t);

  // the queries: row 8n + g, the dims that this lane's key bytes stand for
  uint32_t qh[Q8 ? NR : 1][NC][4], ql[Q8 ? NR : 1][NC][4];  // (F32: in shared memory)
  float rf[NR][2];  // |scale| * log2(e) * the factor of rows 8n + 2t, 8n + 2t + 1 (F32: 2^-16 of it)
  int tok[NR][2];
#pragma unroll
  for (int n = 0; n < NR; n++) {
    const int r = min(r0 + 8 * n + g, sp.R - 1), i = r / rep;
    const float* src = p.q + i * p.q_stride + (int64_t)(kvh * rep + r - i * rep) * D + 8 * t;
    float x[NC][8], m = 0.0f;
    bool fine = true;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x[c][e] = src[32 * c + e];
        m = fmaxf(m, fabsf(x[c][e]));
        fine &= fabsf(x[c][e]) <= 3.402823466e38f;
      }
    if (!fine) m = INFINITY;
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    fine = m <= 3.402823466e38f;
    // The row's largest value becomes 2^14..2^15; with an F32 cache 2^-9..2^-8, so that
    // no score leaves a float's range before its factor. (Both in two steps there, for
    // their powers of two pass a float's range.) A row with an infinity or a NaN: NaN.
    constexpr int up = Q8 ? 14 : 23;
    const int ex = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 127);
    const float f = p.scale < 0.0f ? -pow2f(up - ex) : pow2f(up - ex);
#pragma unroll
    for (int c = 0; c < NC; c++) {
      if constexpr (Q8) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float a = __fmul_rn(x[c][2 * e], f), b = __fmul_rn(x[c][2 * e + 1], f);
          const __half2 hh = __floats2half2_rn(a, b);
          const float2 back = __half22float2(hh);
          qh[n][c][e] = fine ? h2_bits(hh) : 0x7e007e00u;
          ql[n][c][e] = fine ? h2_bits(__floats2half2_rn(__fsub_rn(a, back.x), __fsub_rn(b, back.y))) : 0u;
        }
      } else if (c % kFewWarps == warp) {
        uint32_t h[8], l[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          split_tf32(__fmul_rn(__fmul_rn(x[c][e], f), pow2f(-32)), h[e], l[e]);
          if (!fine) h[e] = 0x7fc00000u;
        }
        sm.q[n][c][0][lane] = make_uint4(h[0], h[1], h[2], h[3]);
        sm.q[n][c][1][lane] = make_uint4(h[4], h[5], h[6], h[7]);
        sm.q[n][c][2][lane] = make_uint4(l[0], l[1], l[2], l[3]);
        sm.q[n][c][3][lane] = make_uint4(l[4], l[5], l[6], l[7]);
      }
    }
    const float own = __fmul_rn(__fmul_rn(fabsf(p.scale), 1.4426950408889634f), pow2f(Q8 ? ex - up : ex - up + 16));
#pragma unroll
    for (int u = 0; u < 2; u++) {
      rf[n][u] = __shfl_sync(0xffffffffu, own, 4 * (2 * t + u));
      tok[n][u] = min(r0 + 8 * n + 2 * t + u, sp.R - 1) / rep;
    }
  }

  if (!Q8) __syncthreads();

  float M[NR][2], l[NR][2], acc[NR][NC][2][4];
  int E[NR][2];  // O is in units of 2^(E - 13) (F32: of 1)
#pragma unroll
  for (int n = 0; n < NR; n++) {
    E[n][0] = E[n][1] = 13;
    M[n][0] = M[n][1] = -INFINITY;
    l[n][0] = l[n][1] = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) acc[n][c][i][k] = 0.0f;
  }
  for (int64_t b = begin; b < end; b += step) {
    if (b != begin) kv.load(b + warp * PT * 16, end, g, t);
    // ---- scores, in units of log2: x[tile][row group][position g + 8 (k / 2), row 2t + k % 2]
    float x[PT][NR][4];
#pragma unroll
    for (int q = 0; q < PT; q++) {
      if constexpr (Q8) {
#pragma unroll
        for (int n = 0; n < NR; n++) x[q][n][0] = x[q][n][1] = x[q][n][2] = x[q][n][3] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++) {
          uint32_t a[2][4];  // [row g / g + 8][byte pair]
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t w0 = kv.K[q][h][c].x ^ 0x80808080u, w1 = kv.K[q][h][c].y ^ 0x80808080u;
            a[h][0] = bytes_to_h2(w0, 0x5140);
            a[h][1] = bytes_to_h2(w0, 0x7362);
            a[h][2] = bytes_to_h2(w1, 0x5140);
            a[h][3] = bytes_to_h2(w1, 0x7362);
          }
          const float s0 = __half2float(__ushort_as_half((uint16_t)(c & 1 ? kv.dk[q][0][c / 2] >> 16 : kv.dk[q][0][c / 2])));
          const float s1 = __half2float(__ushort_as_half((uint16_t)(c & 1 ? kv.dk[q][1][c / 2] >> 16 : kv.dk[q][1][c / 2])));
#pragma unroll
          for (int n = 0; n < NR; n++) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816(s, a[0][0], a[1][0], a[0][1], a[1][1], ql[n][c][0], ql[n][c][1]);
            mma16816(s, a[0][2], a[1][2], a[0][3], a[1][3], ql[n][c][2], ql[n][c][3]);
            mma16816(s, a[0][0], a[1][0], a[0][1], a[1][1], qh[n][c][0], qh[n][c][1]);
            mma16816(s, a[0][2], a[1][2], a[0][3], a[1][3], qh[n][c][2], qh[n][c][3]);
            x[q][n][0] = __fmaf_rn(s[0], s0, x[q][n][0]);
            x[q][n][1] = __fmaf_rn(s[1], s0, x[q][n][1]);
            x[q][n][2] = __fmaf_rn(s[2], s1, x[q][n][2]);
            x[q][n][3] = __fmaf_rn(s[3], s1, x[q][n][3]);
          }
        }
      } else {
        float s[NR][3][4];  // lo hi, hi lo, hi hi
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
          for (int i = 0; i < 12; i++) s[n][i / 4][i % 4] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
          for (int e = 0; e < 4; e++) {  // dims 8t + 2e, 8t + 2e + 1 of the block
            uint32_t h[4], l[4];
#pragma unroll
            for (int i = 0; i < 4; i++) split_tf32(kv.K[q][i & 1][c][2 * e + (i >> 1)], h[i], l[i]);
#pragma unroll
            for (int n = 0; n < NR; n++) {
              const uint2 bh = ((const uint2*)&sm.q[n][c][e >> 1][lane])[e & 1], bl = ((const uint2*)&sm.q[n][c][2 + (e >> 1)][lane])[e & 1];
              mma1688(s[n][0], l, bh.x, bh.y);
              mma1688(s[n][1], h, bl.x, bl.y);
              mma1688(s[n][2], h, bh.x, bh.y);
            }
          }
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
          for (int k = 0; k < 4; k++) {
            // (a finite key's score is finite: one that is not comes from an infinity or a NaN in
            // the key or the query, whatever the halves made of it, and becomes NaN)
            const float y = __fadd_rn(s[n][2][k], __fadd_rn(s[n][0][k], s[n][1][k]));
            x[q][n][k] = __fmaf_rn(y, 0.0f, y);
          }
      }
    }
    // ---- masks, maxima
    uint32_t seen[PT][NR];  // bit k: x[..][k] is attended to
    float fac[NR][2];
    float dmax[Q8 ? PT : 1][2];  // the values' largest scale of positions g, g + 8 that is no NaN
    if constexpr (Q8) {
#pragma unroll
      for (int q = 0; q < PT; q++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          dmax[q][h] = 0.0f;
#pragma unroll
          for (int i = 0; i < FewCache<D, Q8>::ND; i++) {
            const float2 d = __half22float2(__habs2(*reinterpret_cast<const __half2*>(&kv.dv[q][h][i])));
            dmax[q][h] = fmaxf(dmax[q][h], fmaxf(d.x, d.y));
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NR; n++) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int q = 0; q < PT; q++) {
        const int64_t tp = b + (warp * PT + q) * 16;
        seen[q][n] = 15u;
        if (tp + 16 > p.n_past) {
          const uint32_t m0 = attended32(p, tok[n][0], tp, end) >> g, m1 = attended32(p, tok[n][1], tp, end) >> g;
          seen[q][n] = (m0 & 1u) | (m1 & 1u) << 1 | (m0 >> 8 & 1u) << 2 | (m1 >> 8 & 1u) << 3;
        } else if (tp + 16 > end) {
          seen[q][n] = (tp + g < end ? 3u : 0u) | (tp + g + 8 < end ? 12u : 0u);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
          x[q][n][k] = (seen[q][n] >> k) & 1u ? __fmul_rn(x[q][n][k], rf[n][k & 1]) : -INFINITY;
          if (!Q8) x[q][n][k] = __fmul_rn(x[q][n][k], 65536.0f);
          mx[k & 1] = fmaxf(mx[k & 1], x[q][n][k]);
        }
      }
#pragma unroll
      for (int u = 0; u < 2; u++) {
#pragma unroll
        for (int s = 4; s < 32; s *= 2) mx[u] = fmaxf(mx[u], __shfl_xor_sync(0xffffffffu, mx[u], s));
        const float Mn = fmaxf(M[n][u], mx[u]), Mr = Mn == -INFINITY ? 0.0f : Mn;
        const float f = exp2_approx(__fsub_rn(M[n][u], Mr));
        fac[n][u] = f;
        l[n][u] = __fmul_rn(l[n][u], f);
        M[n][u] = Mn;
        // weights
#pragma unroll
        for (int q = 0; q < PT; q++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float& y = x[q][n][2 * h + u];
            y = exp2_approx(__fsub_rn(y, Mr));
            l[n][u] = __fadd_rn(l[n][u], y);
          }
      }
      if constexpr (Q8) {
        // both rows' E in one word (not below -40, so that O, which moves to the new unit,
        // stays in a float's range)
        float top[2] = {0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < PT; q++)
#pragma unroll
          for (int k = 0; k < 4; k++) top[k & 1] = fmaxf(top[k & 1], __fmul_rn(x[q][n][k], dmax[q][k >> 1]));
        uint32_t both = __float_as_uint(top[0]) >> 23 | __float_as_uint(top[1]) >> 23 << 16;
#pragma unroll
        for (int s = 4; s < 32; s *= 2) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, s));
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const int En = min(max((int)(both >> (16 * u) & 0xffffu) - 127, -40), 16);
          fac[n][u] = __fmul_rn(fac[n][u], pow2f(E[n][u] - En));
          E[n][u] = En;
        }
      }
    }
    // ---- O = O fac + P V
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < NR; n++)
#pragma unroll
        for (int q = 0; q < PT; q++)
#pragma unroll
          for (int k = 0; k < 4; k++) x[q][n][k] = __fmul_rn(x[q][n][k], pow2f(13 - E[n][k & 1]));
#pragma unroll
      for (int q = 0; q < PT; q++)
#pragma unroll
        for (int c = 0; c < NC; c++) {
          // V^T: dims 32c + 4g + e of positions 2t, 2t + 1 (v[0][e]) and 2t + 8, 2t + 9 (v[1][e])
          uint32_t v[2][4];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const uint32_t w0 = kv.V[q][2 * h][c] ^ 0x80808080u, w1 = kv.V[q][2 * h + 1][c] ^ 0x80808080u;
            const uint32_t lo = __byte_perm(w0, w1, 0x5140), hi = __byte_perm(w0, w1, 0x7362);
            v[h][0] = bytes_to_h2(lo, 0x4140);
            v[h][1] = bytes_to_h2(lo, 0x4342);
            v[h][2] = bytes_to_h2(hi, 0x4140);
            v[h][3] = bytes_to_h2(hi, 0x4342);
          }
          const float s0 = __half2float(__ushort_as_half((uint16_t)(c & 1 ? kv.dv[q][0][c / 2] >> 16 : kv.dv[q][0][c / 2])));
          const float s1 = __half2float(__ushort_as_half((uint16_t)(c & 1 ? kv.dv[q][1][c / 2] >> 16 : kv.dv[q][1][c / 2])));
#pragma unroll
          for (int n = 0; n < NR; n++) {
            float w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = (seen[q][n] >> k) & 1u ? __fmul_rn(x[q][n][k], k < 2 ? s0 : s1) : 0.0f;
            const __half2 h0 = __floats2half2_rn(w[0], w[1]), h1 = __floats2half2_rn(w[2], w[3]);
            const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
            const uint32_t b0 = transpose8x8(h2_bits(h0)), b1 = transpose8x8(h2_bits(h1));
            const uint32_t c0 = transpose8x8(h2_bits(__floats2half2_rn(__fsub_rn(w[0], f0.x), __fsub_rn(w[1], f0.y))));
            const uint32_t c1 = transpose8x8(h2_bits(__floats2half2_rn(__fsub_rn(w[2], f1.x), __fsub_rn(w[3], f1.y))));
#pragma unroll
            for (int i = 0; i < 2; i++) {
              // (a sum of its own for every 16 positions: the MMA cuts what it accumulates, and
              // one-signed, 4e-6 of the result over 2000 positions a warp)
              float o[4] = {0.f, 0.f, 0.f, 0.f};
              mma16816(o, v[0][2 * i], v[0][2 * i + 1], v[1][2 * i], v[1][2 * i + 1], c0, c1);
              mma16816(o, v[0][2 * i], v[0][2 * i + 1], v[1][2 * i], v[1][2 * i + 1], b0, b1);
#pragma unroll
              for (int k = 0; k < 4; k++)
                acc[n][c][i][k] = q == 0 ? __fmaf_rn(acc[n][c][i][k], fac[n][k & 1], o[k]) : __fadd_rn(acc[n][c][i][k], o[k]);
            }
          }
        }
    } else {
#pragma unroll
      for (int q = 0; q < PT; q++) {
        // positions whose values are not all finite
        uint32_t bad = 0;
#pragma unroll
        for (int h = 0; h < 4; h++) {
          float z = 0.0f;
#pragma unroll
          for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) z = __fmaf_rn(kv.V[q][h][c][e], 0.0f, z);
          if (z != 0.0f) bad |= 1u << (2 * t + (h & 1) + 4 * (h & 2));
        }
        bad = __reduce_or_sync(0xffffffffu, bad);
        if (bad) {
#pragma unroll
          for (int h = 0; h < 4; h++)
            if (bad >> (2 * t + (h & 1) + 4 * (h & 2)) & 1u)
#pragma unroll
              for (int c = 0; c < NC; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) kv.V[q][h][c][e] = 0.0f;
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {  // positions 8h .. 8h + 7
          uint32_t wh[NR][2], wl[NR][2];  // weights of positions 8h + 2t, 8h + 2t + 1, row g
#pragma unroll
          for (int n = 0; n < NR; n++) {
            float w[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
              w[u] = (seen[q][n] >> (2 * h + u)) & 1u ? x[q][n][2 * h + u] : 0.0f;
              if (bad && (bad >> (8 * h + g) & 1u) && ((seen[q][n] >> (2 * h + u)) & 1u)) w[u] = __int_as_float(0x7fffffff);
            }
            const uint32_t a = __float_as_uint(w[0]), b = __float_as_uint(w[1]);
            const uint32_t top = transpose8x8(__byte_perm(a, b, 0x7632)), low = transpose8x8(__byte_perm(a, b, 0x5410));
            split_tf32(__uint_as_float(__byte_perm(low, top, 0x5410)), wh[n][0], wl[n][0]);
            split_tf32(__uint_as_float(__byte_perm(low, top, 0x7632)), wh[n][1], wl[n][1]);
          }
#pragma unroll
          for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
              uint32_t vh[4], vl[4];
#pragma unroll
              for (int k = 0; k < 4; k++) split_tf32(kv.V[q][2 * h + (k >> 1)][c][2 * i + (k & 1)], vh[k], vl[k]);
#pragma unroll
              for (int n = 0; n < NR; n++) {
                // (a sum of its own for every eight positions: the MMA cuts what it
                // accumulates, and one-signed; over 2000 positions that was 2e-5)
                float o[4] = {0.f, 0.f, 0.f, 0.f};
                mma1688(o, vl, wh[n][0], wh[n][1]);
                mma1688(o, vh, wl[n][0], wl[n][1]);
                mma1688(o, vh, wh[n][0], wh[n][1]);
#pragma unroll
                for (int k = 0; k < 4; k++)
                  acc[n][c][i][k] = q == 0 && h == 0 ? __fmaf_rn(acc[n][c][i][k], fac[n][k & 1], o[k]) : __fadd_rn(acc[n][c][i][k], o[k]);
              }
            }
        }
      }
    }
  }
  // ---- the CTA's warps
#pragma unroll
  for (int n = 0; n < NR; n++) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
#pragma unroll
      for (int s = 4; s < 32; s *= 2) l[n][u] = __fadd_rn(l[n][u], __shfl_xor_sync(0xffffffffu, l[n][u], s));
      if (g == 0) {
        sm.m[warp][8 * n + 2 * t + u] = M[n][u];
        sm.l[warp][8 * n + 2 * t + u] = l[n][u];
        sm.scale[warp][8 * n + 2 * t + u] = pow2f(E[n][u] - 13);
      }
    }
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          sm.part[warp][8 * n + 2 * t + (k & 1)][32 * c + 4 * g + 2 * i + (k >> 1)] = acc[n][c][i][k];
  }
  __syncthreads();
  for (int e = tid; e < 8 * NR * D; e += kFewNT) {
    const int r = e / D, d = e - r * D;
    float m = sm.m[0][r];
#pragma unroll
    for (int w = 1; w < kFewWarps; w++) m = fmaxf(m, sm.m[w][r]);
    const float mr = m == -INFINITY ? 0.0f : m;
    float o = 0.0f, s = 0.0f;
#pragma unroll
    for (int w = 0; w < kFewWarps; w++) {
      const float f = exp2_approx(__fsub_rn(sm.m[w][r], mr));
      o = __fmaf_rn(sm.part[w][r][d], __fmul_rn(f, sm.scale[w][r]), o);
      s = __fmaf_rn(sm.l[w][r], f, s);
    }
    sm.part[0][r][d] = o;  // (read by this thread alone)
    if (d == 0) {
      sm.cm[r] = m;
      sm.cl[r] = s;
    }
  }
  // ---- the cluster's CTAs: each takes a share of the (row, dim) pairs
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int rank = (int)cluster_ctarank(), c_id = blockIdx.x / cluster;
  for (int e = rank * kFewNT + tid; e < 8 * NR * D; e += cluster * kFewNT) {
    const int r = e / D, d = e - r * D, row = r0 + r;
    if (row >= sp.R) break;  // (rows go up)
    float m = -INFINITY;
    for (int c = 0; c < cluster; c++) m = fmaxf(m, dsmem_ld(&sm.cm[r], c));
    const float mr = m == -INFINITY ? 0.0f : m;
    float o = 0.0f, s = 0.0f;
    for (int c = 0; c < cluster; c++) {
      const float f = exp2_approx(__fsub_rn(dsmem_ld(&sm.cm[r], c), mr));
      o = __fmaf_rn(dsmem_ld(&sm.part[0][r][d], c), f, o);
      s = __fmaf_rn(dsmem_ld(&sm.cl[r], c), f, s);
    }
    if (sp.S == 1) {
      const int i = row / rep;
      p.out[((int64_t)i * p.H + kvh * rep + (row - i * rep)) * D + d] = s == 0.0f ? 0.0f : __fdiv_rn(o, s);
    } else {
      float* rec = (float*)p.scratch + (((int64_t)kvh * sp.S + c_id) * sp.R + row) * (D + 4);
      rec[4 + d] = o;
      if (d == 0) *(float4*)rec = make_float4(m, m, s, 0.0f);
    }
  }
  // (no CTA leaves while another reads its shared memory)
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int D, int NR, bool Q8>
cudaError_t launch_few(const TreeAttnParams& p, cudaStream_t s) {
  TreeSplit sp{};
  sp.R = p.T * (p.H / p.HKV);
  sp.RG = (sp.R + 8 * NR - 1) / (8 * NR);
  const int64_t n_kv = (int64_t)p.n_past + p.T, steps = (n_kv + kFewStep<D, Q8> - 1) / kFewStep<D, Q8>;
  // One cluster where it holds every step; else clusters of 8 (fewer where a KV head's
  // share of the GPU has no room for them), for 4 CTAs an SM up to 64 dims and 2 above.
  // (That is what runs at once of Q8_0 builds of 64 dims. Their registers let 3 run of 96
  // and 128 dims, 2 of F32 builds of 64 dims, 3 of 32, and 2 of all with two row groups.)
  int cluster = 1;
  const int64_t room = std::max<int64_t>(1, kTrSms * (D <= 64 ? 4 : 2) / ((int64_t)p.HKV * sp.RG));
  if (steps <= 16) {
    while (cluster < steps) cluster *= 2;
    sp.per = 1;
    sp.S = 1;
  } else {
    cluster = 8;
    while (cluster > room) cluster /= 2;
    const int64_t ctas = room / cluster * cluster;
    sp.per = (int32_t)((steps + ctas - 1) / ctas);
    sp.S = (int32_t)((steps + (int64_t)sp.per * cluster - 1) / ((int64_t)sp.per * cluster));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(sp.S * cluster), (unsigned)p.HKV, (unsigned)sp.RG);
  cfg.blockDim = dim3(kFewNT);
  cfg.dynamicSmemBytes = sizeof(FewSmem<D, NR, Q8>);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_few_kernel<D, NR, Q8>, p, sp, cluster);
  if (e != cudaSuccess || sp.S == 1) return e;
  return launch_tree_join<D>(p, sp, s);
}

template <int D, int NR, bool Q8>
cudaError_t prepare_few() {
  cudaError_t e = cudaFuncSetAttribute(attn_few_kernel<D, NR, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(FewSmem<D, NR, Q8>));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(attn_few_kernel<D, NR, Q8>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

template <int D>
cudaError_t prepare_few_of() {
  cudaError_t e = prepare_few<D, 1, true>();
  if (e == cudaSuccess) e = prepare_few<D, 2, true>();
  if (e == cudaSuccess) e = prepare_few<D, 1, false>();
  return e == cudaSuccess ? prepare_few<D, 2, false>() : e;
}
template <int D>
cudaError_t launch_few_of(const TreeAttnParams& p, cudaStream_t s) {
  const bool one = p.T * (p.H / p.HKV) <= 8;
  if (p.q8) return one ? launch_few<D, 1, true>(p, s) : launch_few<D, 2, true>(p, s);
  return one ? launch_few<D, 1, false>(p, s) : launch_few<D, 2, false>(p, s);
}

}  // namespace

cudaError_t prepare_attn_few_kernels() {
  cudaError_t e = prepare_few_of<32>();
  if (e == cudaSuccess) e = prepare_few_of<64>();
  if (e == cudaSuccess) e = prepare_few_of<96>();
  return e == cudaSuccess ? prepare_few_of<128>() : e;
}

cudaError_t launch_attn_few(const TreeAttnParams& p, cudaStream_t s) {
  switch (p.D) {
    case 32: return launch_few_of<32>(p, s);
    case 64: return launch_few_of<64>(p, s);
    case 96: return launch_few_of<96>(p, s);
    case 128: return launch_few_of<128>(p, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace mi
