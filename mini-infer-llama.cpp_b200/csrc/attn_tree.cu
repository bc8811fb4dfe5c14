// Attention of a tree of drafted tokens over a cache. No counterpart in the
// reference, whose attention knows only a causal run of tokens
// (ref src/ops_cpu.cpp:304-410).
//
// Token i of T attends to cache rows [0, n_past) and to row n_past + j (drafted
// token j's) where bit j of its mask is set; without a mask to j <= i.
//   s = scale q.k,  p = exp(s - max s),  out = sum p v / sum p
// over the attended rows, and zeros where there is none. The cache is F32
// ([n_ctx][n_head_kv][D]) or Q8_0 (kv_q8.cu).
#include <algorithm>

#include "mi_device.cuh"

namespace mi {

namespace {

constexpr int kTrNT = 128;

__device__ __forceinline__ bool attends(const TreeAttnParams& p, int t, int64_t pos) {
  if (pos < p.n_past) return true;
  const int j = (int)(pos - p.n_past);
  if (!p.mask) return j <= t;
  return (p.mask[(int64_t)t * ((p.T + 31) / 32) + (j >> 5)] >> (j & 31)) & 1u;
}

template <bool Q8>
__device__ __forceinline__ float cached(const TreeAttnParams& p, const void* c, int kvh, int64_t pos, int e) {
  if (!Q8) return ((const float*)c)[(pos * p.HKV + kvh) * p.D + e];
  const int64_t at = (int64_t)kvh * p.n_ctx + pos, plane = (int64_t)p.HKV * p.n_ctx * p.D;
  return __fmul_rn((float)((const int8_t*)c)[at * p.D + e],
                   __half2float(((const __half*)((const uint8_t*)c + plane))[at * (p.D / 32) + (e >> 5)]));
}

// One CTA per (head, token), 128 positions at a time.
template <bool Q8>
__global__ void __launch_bounds__(kTrNT) attn_tree_kernel(const TreeAttnParams p) {
  __shared__ float q[128], e_s[kTrNT], red[kTrNT / 32];
  const int h = blockIdx.x, t = blockIdx.y, tid = threadIdx.x, kvh = h / (p.H / p.HKV);
  const int64_t n_kv = p.n_past + p.T;
  if (tid < p.D) q[tid] = p.q[t * p.q_stride + (int64_t)h * p.D + tid];
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  for (int64_t t0 = 0; t0 < n_kv; t0 += kTrNT) {
    __syncthreads();
    const int64_t pos = t0 + tid;
    float s = -INFINITY;
    if (pos < n_kv && attends(p, t, pos)) {
      s = 0.0f;
      for (int e = 0; e < p.D; e++) s = __fmaf_rn(q[e], cached<Q8>(p, p.cache_k, kvh, pos, e), s);
      s = __fmul_rn(s, p.scale);
      if (s != s) s = INFINITY;  // (the maximum passes a NaN over; e^(inf - inf) brings it back)
    }
    const float wm = warp_max(s);
    if ((tid & 31) == 0) red[tid >> 5] = wm;
    __syncthreads();
    float mn = m;
    for (int w = 0; w < kTrNT / 32; w++) mn = fmaxf(mn, red[w]);
    if (mn == -INFINITY) continue;
    e_s[tid] = expf(s - mn);
    __syncthreads();
    const float f = expf(m - mn);
    l = __fmul_rn(l, f);
    acc = __fmul_rn(acc, f);
    m = mn;
    const int n = (int)min((int64_t)kTrNT, n_kv - t0);
    for (int i = 0; i < n; i++) {
      l = __fadd_rn(l, e_s[i]);
      if (tid < p.D && e_s[i] != 0.0f) acc = __fmaf_rn(e_s[i], cached<Q8>(p, p.cache_v, kvh, t0 + i, tid), acc);
    }
  }
  if (tid < p.D) p.out[((int64_t)t * p.H + h) * p.D + tid] = l == 0.0f ? 0.0f : __fdiv_rn(acc, l);
}

}  // namespace

bool attn_tree_fits(int64_t D, int64_t H, int64_t HKV, int64_t T) {
  return (D == 32 || D == 64 || D == 96 || D == 128) && H > 0 && HKV > 0 && H % HKV == 0 && H <= 65535 && T >= 0 &&
         T <= kTreeMaxTokens;
}

size_t attn_tree_scratch_bytes(int64_t H, int64_t HKV, int64_t n_kv, int64_t T, int64_t D) { return 16; }

cudaError_t launch_attn_tree(const TreeAttnParams& p, cudaStream_t s) {
  if (p.T == 0) return cudaSuccess;
  const dim3 grid((unsigned)p.H, (unsigned)p.T);
  if (p.q8) attn_tree_kernel<true><<<grid, kTrNT, 0, s>>>(p);
  else attn_tree_kernel<false><<<grid, kTrNT, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace mi
