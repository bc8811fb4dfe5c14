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
// it to 0.004, so the angles are formed and reduced to one turn in 64 bits and
// only the remainder in (-pi, pi] is rounded to a float (2e-7 at most).
#include <cmath>

#include "mi_device.cuh"

namespace mi {

namespace {

constexpr int kRopeNT = 256;

// cos and sin of every pair of the CTA's token, in shared memory.
__device__ __forceinline__ void token_angles(const QkRopeParams& p, int64_t t, float2* cs) {
  const double pos = p.pos ? (double)p.pos[t] : (double)p.n_past + (double)t;
  for (int i = threadIdx.x; i < p.n_dims / 2; i += kRopeNT) {
    const double a = pos * p.freq[i];
    // one turn as a float64 and the rest of it: the remainder is good to 2^-53 of a
    const double turns = rint(a * 0.15915494309189535);
    double r = fma(turns, -6.283185307179586, a);
    r = fma(turns, -2.4492935982947064e-16, r);
    float s, c;
    sincosf((float)r, &s, &c);
    cs[i] = make_float2(c, s);
  }
}

// One CTA per token; a warp per head. A lane holds both elements of its pairs,
// so a head is read once, before any of it is written (in place is safe).
__global__ void __launch_bounds__(kRopeNT) qk_norm_rope_kernel(const __grid_constant__ QkRopeParams p) {
  constexpr int NP = kRopeMaxDim / 64, NR = kRopeMaxDim / 32;
  __shared__ float2 cs[kRopeMaxDim / 2];
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
      r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)p.D), p.eps)));
    }
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

}  // namespace

cudaError_t launch_qk_norm_rope(QkRopeParams& p, float freq_base, cudaStream_t s) {
  if (p.n_tokens == 0) return cudaSuccess;
  for (int i = 0; i < p.n_dims / 2; i++) p.freq[i] = std::pow((double)freq_base, -2.0 * i / p.n_dims);
  qk_norm_rope_kernel<<<(unsigned)p.n_tokens, kRopeNT, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace mi
