// The Q8_0 key/value cache: quantised as it is written, read back as F32. No
// counterpart in the reference, whose cache is F32 (ref src/model_qwen2.cpp:557-596).
//
// One buffer holds the keys (or the values) of one layer:
//   int8 quants [n_head_kv][n_ctx][D], then fp16 scales [n_head_kv][n_ctx][D / 32].
// A KV head's positions are contiguous in both planes, so attention streams any
// run of positions as two contiguous ranges; 34/32 bytes per value.
//
// Block of 32 values of a row:
//   d = fp16(min(max|x| * fl(1 / 127), 65504)),  q = clamp(rint(x / d), -127, 127),  q = 0 where d = 0.
// (The product with the float nearest 1 / 127 is off by 2^-23 of the quotient at
// most, which picks the other neighbour of d only where both are as good to that.) q rounds
// against the d that is stored, so a value is off by d / 2 at most: a d below
// max|x| / 127 makes |x| / d pass 127 by 2^-11 of it, which rounds to 127; only
// subnormal and saturated scales reach the clamp. An infinity or a NaN makes d NaN
// and q 0: the whole block reads back as NaN.
//
// The float32 quotient x / d gives exactly the integer that a 64-bit one gives: a
// rounding border is (k + 1/2) d with at most 20 significant bits, a float x beside
// it is at least one of its own ulps away, and that moves the quotient by more than
// half an ulp of k + 1/2.
//
// Both kernels pass over their data once. For many rows HBM bounds the read (16384 rows of
// 4 heads of 128 13.9 us, 6.1 TB/s); the append, with four divisions a 16-byte piece, runs
// at half of that (27.4 us). Few rows are launch and latency. Each thread has four 16-byte
// pieces of four rows under way.
#include <algorithm>

#include "mi_device.cuh"

namespace mi {

namespace {

constexpr int kKvNT = 256;
constexpr int kKvAhead = 4;  // rows that a thread has under way

// A CTA's threads are tiled over a row's 16-byte pieces (`width` of them, all of the
// row where it has no more than the CTA has threads) and over rows.
struct KvTiling {
  int32_t pieces, width, rows;  // of a row; of a CTA; rows of a CTA at a time
};

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
  const __half dh = finite ? __float2half_rn(fminf(__fmul_rn(m, 1.0f / 127.0f), 65504.0f)) : __ushort_as_half(0x7e00);
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

// Where a later token names the same slot, an earlier one must leave the row alone. Few
// tokens are compared in pairs. Many leave tags instead: the first word of what a CTA
// writes of a row becomes 0x80 << 24 | t for the last token t that names the row. No
// quants are such a word (none is -128), so a token that finds its own tag is the last
// one, also while others' rows are being written over their tags. (Pairs cost the square
// of the tokens, tags two launches: 512 slots of 2 heads of 64 7.2 us with pairs, 513 7.0
// with tags; 2048 17.6 and 7.2, 65536 2 ms and 36 us, of which 27 without slots.)
constexpr uint32_t kKvTag = 0x80000000u;
constexpr int64_t kKvTags = 1 << 24;    // tokens that tags can tell apart
constexpr int64_t kKvPairs = 16384;     // tokens times those of a CTA that are compared in pairs, at most
__device__ __forceinline__ uint32_t* kv_tag(const KvAppendParams& p, bool is_v, int first_piece, int32_t slot) {
  const int nb = p.D / 32, blk = first_piece >> 3, h = blk / nb, b = blk - h * nb;
  return (uint32_t*)((is_v ? p.cache_v : p.cache_k) + ((int64_t)h * p.n_ctx + slot) * p.D + b * 32);
}
// Grid (tokens, pieces of a row, keys / values) as below: the tags' words as 0, then the tags.
template <bool SET>
__global__ void __launch_bounds__(kKvNT) kv_tag_kernel(const KvAppendParams p, const KvTiling g) {
  const int64_t t = (int64_t)blockIdx.x * kKvNT + threadIdx.x;
  const int32_t s = t < p.n_tokens ? p.slots[t] : -1;
  if (s < 0 || s >= p.n_ctx) return;
  uint32_t* tag = kv_tag(p, blockIdx.z, blockIdx.y * g.width, s);
  if (SET) atomicMax(tag, kKvTag | (uint32_t)t);
  else *tag = 0;
}

// VEC: rows are 16-byte aligned (float4 loads). Grid (rows, pieces of a row, keys /
// values); eight threads hold a block of 32. tagged: see above.
template <bool VEC>
__global__ void __launch_bounds__(kKvNT) kv_append_q8_kernel(const KvAppendParams p, const KvTiling g, const bool tagged) {
  extern __shared__ int32_t row[];  // cache row of each of the CTA's tokens, -1: none
  const int nt_cta = g.rows * kKvAhead;
  const int64_t t0 = (int64_t)blockIdx.x * nt_cta;
  const int nt = (int)min((int64_t)nt_cta, p.n_tokens - t0);
  const bool is_v = blockIdx.z;
  const int tid = threadIdx.x, r = tid / g.width, piece = blockIdx.y * g.width + tid - r * g.width;
  const bool live = r < g.rows && piece < g.pieces;
  const float* src = (is_v ? p.v : p.k) + (int64_t)piece * 4;
  const int64_t stride = is_v ? p.v_stride : p.k_stride;
  float x[kKvAhead][4];
#pragma unroll
  for (int u = 0; u < kKvAhead; u++) {
    const int i = r + u * g.rows;
    if (live && i < nt) {
      if (VEC) {
        const float4 f = *(const float4*)(src + (t0 + i) * stride);
        x[u][0] = f.x, x[u][1] = f.y, x[u][2] = f.z, x[u][3] = f.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[u][e] = src[(t0 + i) * stride + e];
      }
    } else {
      x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.0f;
    }
  }
  for (int i = tid; i < nt; i += kKvNT) {
    int32_t s = p.slots ? p.slots[t0 + i] : (int32_t)(p.n_past + t0 + i);
    if (s >= p.n_ctx) {
      atomicExch(p.err, 1 /* MI_CUDA_ERR_ARG */);
      s = -1;
    }
    if (tagged && s >= 0 && *(volatile uint32_t*)kv_tag(p, is_v, blockIdx.y * g.width, s) != (kKvTag | (uint32_t)(t0 + i))) s = -1;
    row[i] = s;
  }
  __syncthreads();
  if (p.slots && !tagged) {  // a later token with the same slot wins
    for (int64_t j = t0 + 1 + tid; j < p.n_tokens; j += kKvNT) {
      const int32_t s = p.slots[j];
      if (s >= 0)
        for (int i = 0; i < nt && t0 + i < j; i++)
          if (p.slots[t0 + i] == s) row[i] = -1;
    }
    __syncthreads();
  }
  const int nb = p.D / 32, blk = piece >> 3, h = blk / nb, b = blk - h * nb, lane8 = tid & 7;
  const int64_t plane = (int64_t)p.HKV * p.n_ctx * p.D;
  uint8_t* c = is_v ? p.cache_v : p.cache_k;
#pragma unroll
  for (int u = 0; u < kKvAhead; u++) {  // (whole warps stay for the shuffles)
    const int i = r + u * g.rows;
    const int32_t s = live && i < nt ? row[i] : -1;
    const int64_t at = (int64_t)h * p.n_ctx + (s < 0 ? 0 : s);
    quantise_block(x[u], s >= 0, (int8_t*)c + at * p.D + b * 32, (__half*)(c + plane) + at * nb + b, lane8);
  }
}

__global__ void __launch_bounds__(kKvNT) kv_read_q8_kernel(const KvReadParams p, const KvTiling g) {
  const bool is_v = blockIdx.z;
  const int tid = threadIdx.x, r = tid / g.width, piece = blockIdx.y * g.width + tid - r * g.width;
  if (r >= g.rows || piece >= g.pieces) return;
  const int nb = p.D / 32, blk = piece >> 3, h = blk / nb, b = blk - h * nb;
  const int64_t plane = (int64_t)p.HKV * p.n_ctx * p.D, at = (int64_t)h * p.n_ctx + p.first;
  const uint8_t* c = is_v ? p.cache_v : p.cache_k;
  const uint8_t* qs = c + at * p.D + b * 32 + (piece & 7) * 4;
  const __half* ds = (const __half*)(c + plane) + at * nb + b;
  float* out = (is_v ? p.v : p.k) + (int64_t)piece * 4;
  const int64_t i0 = (int64_t)blockIdx.x * g.rows * kKvAhead + r;
  // (loads only, from a row that is there: a use or a branch between them would make
  // each wait for the one before it)
  char4 q[kKvAhead];
  __half dh[kKvAhead];
#pragma unroll
  for (int u = 0; u < kKvAhead; u++) {
    const int64_t i = min(i0 + u * g.rows, p.n_rows - 1);
    q[u] = *(const char4*)(qs + i * p.D);
    dh[u] = ds[i * nb];
  }
#pragma unroll
  for (int u = 0; u < kKvAhead; u++) {
    const int64_t i = i0 + u * g.rows;
    const float d = __half2float(dh[u]);
    if (i < p.n_rows)
      *(float4*)(out + i * g.pieces * 4) = make_float4(__fmul_rn((float)q[u].x, d), __fmul_rn((float)q[u].y, d),
                                                       __fmul_rn((float)q[u].z, d), __fmul_rn((float)q[u].w, d));
  }
}

KvTiling kv_tiling(int32_t HKV, int32_t D) {
  KvTiling g{};
  g.pieces = HKV * (D / 4);
  g.width = std::min(g.pieces, kKvNT);
  g.rows = kKvNT / g.width;
  return g;
}
dim3 kv_grid(const KvTiling& g, int64_t n) {
  const int64_t per = g.rows * kKvAhead;
  return dim3((unsigned)((n + per - 1) / per), (unsigned)((g.pieces + g.width - 1) / g.width), 2);
}

}  // namespace

cudaError_t launch_kv_append_q8(const KvAppendParams& p, cudaStream_t s) {
  if (p.n_tokens == 0) return cudaSuccess;
  const KvTiling g = kv_tiling(p.HKV, p.D);
  const size_t smem = (size_t)g.rows * kKvAhead * 4;
  const bool vec = ((uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0 && p.k_stride % 4 == 0 && p.v_stride % 4 == 0;
  const bool tagged = p.slots && p.n_tokens * (g.rows * kKvAhead) > kKvPairs;
  const int64_t n = tagged ? kKvTags : p.n_tokens;
  for (int64_t t = 0; t < p.n_tokens; t += n) {  // (later tokens write last)
    KvAppendParams c = p;
    c.n_tokens = std::min(n, p.n_tokens - t);
    c.k += t * p.k_stride;
    c.v += t * p.v_stride;
    if (tagged) {
      c.slots += t;
      const dim3 grid((unsigned)((c.n_tokens + kKvNT - 1) / kKvNT), kv_grid(g, 1).y, 2);
      kv_tag_kernel<false><<<grid, kKvNT, 0, s>>>(c, g);
      kv_tag_kernel<true><<<grid, kKvNT, 0, s>>>(c, g);
    }
    if (vec) kv_append_q8_kernel<true><<<kv_grid(g, c.n_tokens), kKvNT, smem, s>>>(c, g, tagged);
    else kv_append_q8_kernel<false><<<kv_grid(g, c.n_tokens), kKvNT, smem, s>>>(c, g, tagged);
  }
  return cudaGetLastError();
}

cudaError_t launch_kv_read_q8(const KvReadParams& p, cudaStream_t s) {
  if (p.n_rows == 0) return cudaSuccess;
  const KvTiling g = kv_tiling(p.HKV, p.D);
  kv_read_q8_kernel<<<kv_grid(g, p.n_rows), kKvNT, 0, s>>>(p, g);
  return cudaGetLastError();
}

}  // namespace mi
