// What the tree-attention kernels share: the mask, the records of their splits, and
// the kernel that joins them.
#pragma once

#include <cuda_fp16.h>

#include "mi_device.cuh"

namespace mi {

namespace {

constexpr int kTrSms = 148;

struct TreeSplit {
  int32_t R, RG, S, per;  // rows of a KV head, groups of them, splits, steps per split
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x 2^k for a whole k, where 2^k alone may lie outside of a float's normal range
// (ex2.approx.ftz gives 0 below 2^-126).
__device__ __forceinline__ float times_pow2(float x, float k) {
  const float h = truncf(__fmul_rn(0.5f, k));
  return __fmul_rn(__fmul_rn(x, exp2_approx(h)), exp2_approx(__fsub_rn(k, h)));
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126..127

// Bit c: whether token t attends to position pos0 + c (c < 32).
__device__ __forceinline__ uint32_t attended32(const TreeAttnParams& p, int t, int64_t pos0, int64_t n_kv) {
  uint32_t m = 0;
  const int64_t j0 = pos0 - p.n_past;  // drafted index of bit 0 (negative: cached text)
  if (p.mask) {
    const int words = (p.T + 31) >> 5;
    const uint32_t* row = p.mask + (int64_t)t * words;
    // the words that hold drafted tokens j0 .. j0 + 31
    const int64_t w = j0 >= 0 ? j0 >> 5 : 0, sh = w * 32 - j0;  // -31 .. 0, or above 0
    if (sh < 32 && w < words) m = sh >= 0 ? row[w] << sh : row[w] >> -sh;
    if (sh < 0 && w + 1 < words) m |= row[w + 1] << (32 + sh);
  } else {
    const int64_t n = (int64_t)t - j0 + 1;  // drafted tokens 0..t
    m = n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
  }
  if (j0 < 0) m |= j0 <= -32 ? ~0u : (1u << -j0) - 1;
  const int64_t left = n_kv - pos0;
  if (left < 32) m &= left <= 0 ? 0u : (1u << left) - 1;
  return m;
}

// Joins the splits of a row: with a_s = 2^(M_s - max M) and b_s = 2^(m_s - max m),
// out = sum a_s O_s / sum b_s l_s * 2^(max M - max m). W warps a row, over its splits;
// the lanes over the dims.
constexpr int kTrJoinNT = 256;
template <int D, int W>
__global__ void __launch_bounds__(kTrJoinNT) attn_tree_join_kernel(const TreeAttnParams p, const TreeSplit sp) {
  constexpr int V = D % 128 == 0 ? 4 : D % 64 == 0 ? 2 : 1, N = D / 32 / V;  // N vectors of V floats a lane
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = W > 1 ? blockIdx.x : blockIdx.x * (kTrJoinNT / 32) + warp, kvh = blockIdx.y;
  if (r >= sp.R) return;
  const float* rec = (const float*)p.scratch + ((int64_t)kvh * sp.S * sp.R + r) * (D + 4);
  const int64_t step = (int64_t)sp.R * (D + 4);
  float M = -INFINITY, m = -INFINITY;
  for (int s = lane; s < sp.S; s += 32) {
    const float2 h = *(const float2*)(rec + s * step);
    M = fmaxf(M, h.x);
    m = fmaxf(m, h.y);
  }
  M = warp_max(M);
  m = warp_max(m);
  const float Mr = M == -INFINITY ? 0.0f : M, mr = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, acc[D / 32];
#pragma unroll
  for (int k = 0; k < D / 32; k++) acc[k] = 0.0f;
#pragma unroll 8
  for (int s = W > 1 ? warp : 0; s < sp.S; s += W) {
    const float* x = rec + s * step;
    const float4 h = *(const float4*)x;
    float v[D / 32];
#pragma unroll
    for (int k = 0; k < N; k++) {
      const float* src = x + 4 + (lane + 32 * k) * V;
      if constexpr (V == 4) *(float4*)(v + 4 * k) = *(const float4*)src;
      else if constexpr (V == 2) *(float2*)(v + 2 * k) = *(const float2*)src;
      else v[k] = *src;
    }
    const float a = exp2_approx(__fsub_rn(h.x, Mr));
    l = __fmaf_rn(h.z, exp2_approx(__fsub_rn(h.y, mr)), l);
#pragma unroll
    for (int k = 0; k < D / 32; k++) acc[k] = __fmaf_rn(v[k], a, acc[k]);
  }
  const int rep = p.H / p.HKV, i = r / rep;
  float* out = p.out + ((int64_t)i * p.H + kvh * rep + (r - i * rep)) * D;
  if constexpr (W == 1) {
#pragma unroll
    for (int k = 0; k < D / 32; k++)
      out[(lane + 32 * (k / V)) * V + k % V] = l == 0.0f ? 0.0f : times_pow2(__fdiv_rn(acc[k], l), __fsub_rn(Mr, mr));
  } else {
    __shared__ float red[W][D + 1];
#pragma unroll
    for (int k = 0; k < D / 32; k++) red[warp][(lane + 32 * (k / V)) * V + k % V] = acc[k];
    if (lane == 0) red[warp][D] = l;
    __syncthreads();
    if (tid < D) {
      float o = red[0][tid];
      l = red[0][D];
#pragma unroll
      for (int w = 1; w < W; w++) {
        o = __fadd_rn(o, red[w][tid]);
        l = __fadd_rn(l, red[w][D]);
      }
      out[tid] = l == 0.0f ? 0.0f : times_pow2(__fdiv_rn(o, l), __fsub_rn(Mr, mr));
    }
  }
}

// (Launched as a programmatic dependent: no kernel has an early trigger, so it starts when
// the records are complete. With one, 64 tokens over 32764 positions took 41.5 us, not 40.1.)
template <int D>
cudaError_t launch_tree_join(const TreeAttnParams& p, const TreeSplit& sp, cudaStream_t s) {
  constexpr int W = kTrJoinNT / 32;
  // A warp a row where CTAs of a row each would not all run at once (2048 rows of 9
  // splits: 2.0 us less), otherwise a CTA (896 rows of 18: 0.8 us less than with a
  // warp; 14 rows of 32: 3.6 us less).
  const bool one = sp.S <= 32 && (int64_t)sp.R * p.HKV > 8 * kTrSms;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(one ? (sp.R + W - 1) / W : sp.R), (unsigned)p.HKV);
  cfg.blockDim = dim3(kTrJoinNT);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return one ? cudaLaunchKernelEx(&cfg, attn_tree_join_kernel<D, 1>, p, sp)
             : cudaLaunchKernelEx(&cfg, attn_tree_join_kernel<D, W>, p, sp);
}

}  // namespace

}  // namespace mi
