// The Q8_0 key/value cache: quantised as it is written, read back as F32. No
// counterpart in the reference, whose cache is F32 (ref src/model_qwen2.cpp:557-596).
//
// One buffer holds the keys (or the values) of one layer:
//   int8 quants [n_head_kv][n_ctx][D], then fp16 scales [n_head_kv][n_ctx][D / 32].
// A KV head's positions are contiguous in both planes, so attention streams any
// run of positions as two contiguous ranges; 34/32 bytes per value.
//
// Block of 32 values of a row:
//   d = fp16(min(max|x| / 127, 65504)),  q = clamp(rint(x / d), -127, 127),  q = 0 where d = 0.
// q rounds against the d that is stored, so a value is off by d / 2 at most (a
// fp16 below amax / 127 makes |x| / d pass 127 by 2^-11 of it, which rounds to
// 127; only subnormal scales reach the clamp). An infinity or a NaN makes d NaN
// and q 0: the whole block reads back as NaN.
//
// The float32 quotients give exactly the integers that 64-bit ones give: a
// rounding border is (k + 1/2) d with at most 20 significant bits, a float x
// beside it is at least one of its own ulps away, and that moves the quotient by
// more than half an ulp of k + 1/2. The same holds for amax / 127 and the
// borders between two fp16 values.
#include <algorithm>

#include "mi_device.cuh"

namespace mi {

namespace {

constexpr int kKvNT = 256;
constexpr int kKvTokens = 8;  // tokens per CTA of the append

// Eight lanes hold a block, four values each.
__device__ __forceinline__ void quantise_block(const float (&x)[4], bool store, int8_t* q, __half* d, int lane8) {
  float m = 0.0f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    m = fmaxf(m, fabsf(x[i]));
    bad |= !(fabsf(x[i]) <= 3.402823466e38f);
  }
  if (bad) m = INFINITY;
#pragma unroll
  for (int s = 4; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  const bool finite = m <= 3.402823466e38f;
  const __half dh = finite ? __float2half_rn(fminf(__fdiv_rn(m, 127.0f), 65504.0f)) : __ushort_as_half(0x7e00);
  const float df = __half2float(dh);
  uint32_t word = 0;
  if (df > 0.0f) {  // (NaN: no)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float r = fminf(fmaxf(rintf(__fdiv_rn(x[i], df)), -127.0f), 127.0f);
      word |= ((uint32_t)(int32_t)r & 0xffu) << (8 * i);
    }
  }
  if (store) {
    *(uint32_t*)(q + 4 * lane8) = word;
    if (lane8 == 0) *d = dh;
  }
}

// VEC: rows are 16-byte aligned (float4 loads).
template <bool VEC>
__global__ void __launch_bounds__(kKvNT) kv_append_q8_kernel(const KvAppendParams p) {
  __shared__ int32_t row[kKvTokens];
  const int64_t t0 = (int64_t)blockIdx.x * kKvTokens;
  const int nt = (int)min((int64_t)kKvTokens, p.n_tokens - t0);
  if (threadIdx.x < nt) {
    const int64_t t = t0 + threadIdx.x;
    int32_t r = p.slots ? p.slots[t] : (int32_t)(p.n_past + t);
    if (r >= p.n_ctx) {
      atomicExch(p.err, 1 /* MI_CUDA_ERR_ARG */);
      r = -1;
    }
    row[threadIdx.x] = r;
  }
  __syncthreads();
  if (p.slots) {  // a later token with the same slot wins
    for (int64_t j = t0 + 1 + threadIdx.x; j < p.n_tokens; j += kKvNT) {
      const int32_t r = p.slots[j];
      if (r >= 0)
        for (int i = 0; i < nt; i++)
          if (t0 + i < j && p.slots[t0 + i] == r) row[i] = -1;
    }
    __syncthreads();
  }
  const int nb = p.D / 32, per_row = p.HKV * nb;  // blocks of a token's row
  const int items = nt * per_row * 2;
  const int lane8 = threadIdx.x & 7;
  const int64_t plane = (int64_t)p.HKV * p.n_ctx * p.D;
  for (int i0 = 0; i0 < items; i0 += kKvNT / 8) {  // (whole warps stay for the shuffles)
    const int it = i0 + (threadIdx.x >> 3);
    const bool live = it < items;
    const int which = live ? it / (nt * per_row) : 0, rem = live ? it - which * nt * per_row : 0;
    const int i = rem / per_row, blk = rem - i * per_row, h = blk / nb, b = blk - h * nb;
    const float* src = (which ? p.v + (t0 + i) * p.v_stride : p.k + (t0 + i) * p.k_stride) + blk * 32 + lane8 * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    const int32_t r = live ? row[i] : -1;
    if (r >= 0) {
      if (VEC) {
        const float4 f = *(const float4*)src;
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = src[e];
      }
    }
    uint8_t* c = which ? p.cache_v : p.cache_k;
    const int64_t at = (int64_t)h * p.n_ctx + (r < 0 ? 0 : r);
    quantise_block(x, r >= 0, (int8_t*)c + at * p.D + b * 32, (__half*)(c + plane) + at * nb + b, lane8);
  }
}

__global__ void __launch_bounds__(kKvNT) kv_read_q8_kernel(const KvReadParams p) {
  const int nb = p.D / 32;
  const int64_t plane = (int64_t)p.HKV * p.n_ctx * p.D;
  const uint8_t* c = blockIdx.y ? p.cache_v : p.cache_k;
  float* out = blockIdx.y ? p.v : p.k;
  const int64_t n4 = p.n_rows * p.HKV * p.D / 4, row4 = (int64_t)p.HKV * p.D / 4;
  for (int64_t i = (int64_t)blockIdx.x * kKvNT + threadIdx.x; i < n4; i += (int64_t)gridDim.x * kKvNT) {
    const int64_t r = i / row4;
    const int e = (int)(i - r * row4) * 4, h = e / p.D, o = e - h * p.D;
    const int64_t at = (int64_t)h * p.n_ctx + p.first + r;
    const char4 q = *(const char4*)(c + at * p.D + o);
    const float d = __half2float(((const __half*)(c + plane))[at * nb + (o >> 5)]);
    *(float4*)(out + 4 * i) = make_float4(__fmul_rn((float)q.x, d), __fmul_rn((float)q.y, d), __fmul_rn((float)q.z, d),
                                          __fmul_rn((float)q.w, d));
  }
}

}  // namespace

cudaError_t launch_kv_append_q8(const KvAppendParams& p, cudaStream_t s) {
  if (p.n_tokens == 0) return cudaSuccess;
  const unsigned grid = (unsigned)((p.n_tokens + kKvTokens - 1) / kKvTokens);
  const bool vec = ((uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0 && p.k_stride % 4 == 0 && p.v_stride % 4 == 0;
  if (vec) kv_append_q8_kernel<true><<<grid, kKvNT, 0, s>>>(p);
  else kv_append_q8_kernel<false><<<grid, kKvNT, 0, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv_read_q8(const KvReadParams& p, cudaStream_t s) {
  if (p.n_rows == 0) return cudaSuccess;
  const int64_t n4 = p.n_rows * p.HKV * p.D / 4;
  const dim3 grid((unsigned)std::min<int64_t>((n4 + kKvNT - 1) / kKvNT, 148 * 8), 2);
  kv_read_q8_kernel<<<grid, kKvNT, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace mi
