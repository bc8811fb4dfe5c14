// Norms of queries and keys per head with the position rotation in the same
// pass. No counterpart in the reference as one operator: its rms_norm and its
// NEOX rope (ref src/ops_cpu.cpp:143-165, 270-302) are separate nodes, and its
// rope knows only consecutive positions.
//
//   y = x / sqrt(mean(x^2) + eps) * w           (w absent: y = x)
//   a_p = pos * base^(-2p / n),  p < n / 2
//   out[p]         = y[p] cos a_p - y[p + n/2] sin a_p
//   out[p + n / 2] = y[p] sin a_p + y[p + n/2] cos a_p,   out[i] = y[i] for i >= n
//
// The angle of position 100000 is 1e5 radians in its first pair: a float holds
// it to 0.004, so the angles are formed in turns, and their whole turns taken off,
// in 64 bits; only the remainder (half a turn at most) is rounded to a float.
//
// One pass over the data, 8 bytes per element: bound by HBM for many tokens, by
// launch and latency for few. A CTA takes one token, so that its angles (64-bit
// arithmetic and a sincospif per pair) are formed once for all heads, under the
// first rows' loads. A head's pairs (p, p + n/2) lie in one lane, so a head is read
// once, before any of it is written (in place is safe).
#include <cmath>
#include <mutex>

#include "mi_device.cuh"

namespace mi {

namespace {

constexpr int kRopeNT = 256;

// cos and sin of every pair of token t, in shared memory.
__device__ __forceinline__ void token_angles(const QkRopeParams& p, int64_t t, float2* cs) {
  for (int i = threadIdx.x; i < p.n_dims / 2; i += kRopeNT) {
    const double pos = p.pos ? (double)p.pos[t] : (double)p.n_past + (double)t;
    const double turns = pos * p.turns[i];
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[i] = make_float2(c, s);
  }
}

__device__ __forceinline__ float inv_rms(float ss, int D, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)D), eps)));
}

__device__ __forceinline__ float4 scaled(float4 x, float r, const float* w, int e) {
  const float4 v = *(const float4*)(w + e);
  return make_float4(__fmul_rn(__fmul_rn(x.x, r), v.x), __fmul_rn(__fmul_rn(x.y, r), v.y), __fmul_rn(__fmul_rn(x.z, r), v.z),
                     __fmul_rn(__fmul_rn(x.w, r), v.w));
}
__device__ __forceinline__ float square_sum(float4 x, float s) {
  return __fmaf_rn(x.x, x.x, __fmaf_rn(x.y, x.y, __fmaf_rn(x.z, x.z, __fmaf_rn(x.w, x.w, s))));
}

// Rows of whole 16-byte pieces (head_dim and n_dims / 2 multiples of 4, aligned
// rows): `group` lanes (a power of two, at least head_dim / 8) hold a head, each
// four pairs and up to eight of the elements that are not rotated; a warp takes
// 32 / group heads.
__global__ void __launch_bounds__(kRopeNT) qk_norm_rope_vec_kernel(const __grid_constant__ QkRopeParams p, const int group) {
  __shared__ __align__(16) float2 cs[kRopeMaxDim / 2];
  const int64_t t = blockIdx.x;
  const int l = threadIdx.x & (group - 1), heads = p.H + p.HKV, half = p.n_dims / 2;
  const int e = 4 * l, r0 = p.n_dims + 4 * l, r1 = r0 + 4 * group;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  bool first = true;
  // (whole warps stay in the loop for the shuffles)
  for (int h0 = 0; h0 < heads; h0 += kRopeNT / group) {
    const int h = h0 + threadIdx.x / group;
    const bool in = h < heads, is_q = h < p.H;
    const float* x = is_q ? p.q + t * p.q_stride + (int64_t)h * p.D : p.k + t * p.k_stride + (int64_t)(h - p.H) * p.D;
    const float* w = is_q ? p.wq : p.wk;
    float4 lo = zero, hi = zero, a = zero, b = zero;
    if (in && e < half) {
      lo = *(const float4*)(x + e);
      hi = *(const float4*)(x + half + e);
    }
    if (in && r0 < p.D) a = *(const float4*)(x + r0);
    if (in && r1 < p.D) b = *(const float4*)(x + r1);
    if (first) {
      token_angles(p, t, cs);
      __syncthreads();
      first = false;
    }
    if (p.wq || p.wk) {
      float ss = square_sum(lo, square_sum(hi, square_sum(a, square_sum(b, 0.0f))));
      for (int s = group / 2; s > 0; s >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, s));
      if (in && w) {
        const float r = inv_rms(ss, p.D, p.eps);
        if (e < half) {
          lo = scaled(lo, r, w, e);
          hi = scaled(hi, r, w, half + e);
        }
        if (r0 < p.D) a = scaled(a, r, w, r0);
        if (r1 < p.D) b = scaled(b, r, w, r1);
      }
    }
    if (!in) continue;
    float* o = is_q ? p.q_out + (t * p.H + h) * p.D : p.k_out + (t * p.HKV + h - p.H) * p.D;
    if (e < half) {
      const float4 c0 = *(const float4*)(cs + e), c1 = *(const float4*)(cs + e + 2);  // cos, sin, cos, sin
      *(float4*)(o + e) = make_float4(__fmaf_rn(lo.x, c0.x, -__fmul_rn(hi.x, c0.y)), __fmaf_rn(lo.y, c0.z, -__fmul_rn(hi.y, c0.w)),
                                      __fmaf_rn(lo.z, c1.x, -__fmul_rn(hi.z, c1.y)), __fmaf_rn(lo.w, c1.z, -__fmul_rn(hi.w, c1.w)));
      *(float4*)(o + half + e) =
          make_float4(__fmaf_rn(lo.x, c0.y, __fmul_rn(hi.x, c0.x)), __fmaf_rn(lo.y, c0.w, __fmul_rn(hi.y, c0.z)),
                      __fmaf_rn(lo.z, c1.y, __fmul_rn(hi.z, c1.x)), __fmaf_rn(lo.w, c1.w, __fmul_rn(hi.w, c1.z)));
    }
    if (r0 < p.D) *(float4*)(o + r0) = a;
    if (r1 < p.D) *(float4*)(o + r1) = b;
  }
}

// Any rows: a warp per head, element by element.
__global__ void __launch_bounds__(kRopeNT) qk_norm_rope_kernel(const __grid_constant__ QkRopeParams p) {
  constexpr int NP = kRopeMaxDim / 64, NR = kRopeMaxDim / 32;
  __shared__ __align__(16) float2 cs[kRopeMaxDim / 2];
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  token_angles(p, t, cs);
  __syncthreads();
  const int half = p.n_dims / 2;
  for (int h = warp; h < p.H + p.HKV; h += kRopeNT / 32) {
    const bool is_q = h < p.H;
    const float* x = is_q ? p.q + t * p.q_stride + (int64_t)h * p.D : p.k + t * p.k_stride + (int64_t)(h - p.H) * p.D;
    float* o = is_q ? p.q_out + (t * p.H + h) * p.D : p.k_out + (t * p.HKV + h - p.H) * p.D;
    const float* w = is_q ? p.wq : p.wk;
    float lo[NP], hi[NP], rest[NR];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int e = lane + 32 * i;
      lo[i] = e < half ? x[e] : 0.0f;
      hi[i] = e < half ? x[e + half] : 0.0f;
      ss = __fmaf_rn(lo[i], lo[i], ss);
      ss = __fmaf_rn(hi[i], hi[i], ss);
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
      const int e = p.n_dims + lane + 32 * i;
      rest[i] = e < p.D ? x[e] : 0.0f;
      ss = __fmaf_rn(rest[i], rest[i], ss);
    }
    float r = 1.0f;
    if (w) {
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, s));
      r = inv_rms(ss, p.D, p.eps);
    }
    __syncwarp();  // every lane has read the head before any of it is written
#pragma unroll
    for (int i = 0; i < NP; i++) {
      const int e = lane + 32 * i;
      if (e < half) {
        const float a = w ? __fmul_rn(__fmul_rn(lo[i], r), w[e]) : lo[i];
        const float b = w ? __fmul_rn(__fmul_rn(hi[i], r), w[e + half]) : hi[i];
        o[e] = __fmaf_rn(a, cs[e].x, -__fmul_rn(b, cs[e].y));
        o[e + half] = __fmaf_rn(a, cs[e].y, __fmul_rn(b, cs[e].x));
      }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
      const int e = p.n_dims + lane + 32 * i;
      if (e < p.D) o[e] = w ? __fmul_rn(__fmul_rn(rest[i], r), w[e]) : rest[i];
    }
  }
}

// base^(-2p / n) / (2 pi) for every pair: the last shape's are kept (a model's
// calls all have one).
std::mutex g_turns_mu;
int32_t g_turns_dims = 0;
float g_turns_base = 0.0f;
double g_turns[kRopeMaxDim / 2];

}  // namespace

cudaError_t launch_qk_norm_rope(QkRopeParams& p, float freq_base, cudaStream_t s) {
  if (p.n_tokens == 0) return cudaSuccess;
  {
    std::lock_guard<std::mutex> lock(g_turns_mu);
    if (g_turns_dims != p.n_dims || g_turns_base != freq_base) {
      for (int i = 0; i < p.n_dims / 2; i++)
        g_turns[i] = std::pow((double)freq_base, -2.0 * i / p.n_dims) / 6.283185307179586476925287;
      g_turns_dims = p.n_dims;
      g_turns_base = freq_base;
    }
    for (int i = 0; i < p.n_dims / 2; i++) p.turns[i] = g_turns[i];
  }
  const uintptr_t all = (uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.wq | (uintptr_t)p.wk | (uintptr_t)p.q_out | (uintptr_t)p.k_out;
  if (p.D % 4 == 0 && p.n_dims % 8 == 0 && all % 16 == 0 && p.q_stride % 4 == 0 && p.k_stride % 4 == 0) {
    int group = 1;
    while (group * 8 < p.D) group *= 2;
    qk_norm_rope_vec_kernel<<<(unsigned)p.n_tokens, kRopeNT, 0, s>>>(p, group);
  } else {
    qk_norm_rope_kernel<<<(unsigned)p.n_tokens, kRopeNT, 0, s>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace mi
