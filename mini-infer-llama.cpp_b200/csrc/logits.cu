// Penalties for repeated tokens, biases and grammar masks on logits, with the
// greedy token of what is left. No counterpart in the reference, which picks the
// first maximum of the raw logits (ref src/model_qwen2.cpp:690-700).
//
// Row r, token j with logit l, c = how often j is in the row's history:
//   x = l;                          c > 0: x = (l > 0 ? l / repeat : l * repeat) - (c * frequency + presence)
//   x += sum of the biases of j (in the list's order);   x = -inf where the allowed bit of j is 0
// token = the lowest j of the largest x, -1 where no x is above -inf.
//
// A row is one thread-block cluster: CTA c takes a contiguous part of the
// vocabulary and counts the history's tokens that fall into it in shared memory
// (integer adds: their order does not matter), so the counts never exist in
// global memory and a row is one pass, 8 bytes per token; the CTAs' winners meet
// in the first CTA's shared memory.
#include <algorithm>

#include "mi_device.cuh"

namespace mi {

namespace {

constexpr int kLgNT = 512;
constexpr int kLgCluster = 8;
constexpr int kLgSlice = 2048;  // tokens counted at a time

__global__ void __launch_bounds__(kLgNT) logits_process_kernel(const LogitsParams p) {
  __shared__ int32_t cnt[kLgSlice];
  __shared__ float bias[kLgSlice];
  __shared__ int32_t owner[kLgSlice];
  __shared__ float wv[kLgNT / 32];
  __shared__ int32_t wi[kLgNT / 32];
  __shared__ float cv[kLgCluster];
  __shared__ int32_t ci[kLgCluster];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_ctarank();
  cluster_arrive_relaxed();  // (every CTA runs before any stores into another's shared memory)
  const int64_t row = blockIdx.x / kLgCluster;
  const int64_t V = p.n_vocab;
  const int64_t per = ((V + kLgCluster - 1) / kLgCluster + 31) / 32 * 32;
  const int64_t v0 = min(V, (int64_t)rank * per), v1 = min(V, v0 + per);
  const float* x = p.logits + row * p.stride;
  float* y = p.out + row * V;
  const int32_t* hist = p.hist + row * p.hist_stride;
  const uint32_t* allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  float best = -INFINITY;
  int32_t best_i = -1;
  for (int64_t s0 = v0; s0 < v1; s0 += kLgSlice) {
    const int n = (int)min((int64_t)kLgSlice, v1 - s0);
    for (int i = tid; i < n; i += kLgNT) {
      cnt[i] = 0;
      bias[i] = 0.0f;
      owner[i] = 0x7fffffff;
    }
    __syncthreads();
    for (int64_t i = tid; i < p.n_hist; i += kLgNT) {
      const int64_t u = (int64_t)hist[i] - s0;
      if (u >= 0 && u < n) atomicAdd(&cnt[u], 1);
    }
    // biases in the list's order: of the entries for one token in a chunk the
    // first adds, then the next (one round where no token is named twice)
    for (int64_t b0 = 0; b0 < p.n_bias; b0 += kLgNT) {
      const int64_t i = b0 + tid;
      const int64_t u = i < p.n_bias ? (int64_t)p.bias_ids[i] - s0 : -1;
      bool todo = u >= 0 && u < n;
      while (__syncthreads_or(todo)) {
        if (todo) atomicMin(&owner[u], tid);
        __syncthreads();
        const bool mine = todo && owner[u] == tid;
        __syncthreads();
        if (mine) {
          bias[u] = __fadd_rn(bias[u], p.bias[i]);
          owner[u] = 0x7fffffff;
          todo = false;
        }
      }
    }
    __syncthreads();
    for (int i = tid; i < n; i += kLgNT) {
      const int64_t j = s0 + i;
      float v = x[j];
      const int c = cnt[i];
      if (c > 0)
        v = __fsub_rn(v > 0.0f ? __fdiv_rn(v, p.repeat) : __fmul_rn(v, p.repeat),
                      __fadd_rn(__fmul_rn((float)c, p.frequency), p.presence));
      if (p.n_bias) v = __fadd_rn(v, bias[i]);
      if (allowed && !((allowed[j >> 5] >> (j & 31)) & 1u)) v = -INFINITY;
      y[j] = v;
      if (v > best) {
        best = v;
        best_i = (int32_t)j;
      }
    }
    __syncthreads();
  }
  cluster_wait_acquire();
  if (!p.tokens) return;
  auto take = [&](float v, int32_t i) {
    if (i >= 0 && (v > best || best_i < 0 || (v == best && i < best_i))) {
      best = v;
      best_i = i;
    }
  };
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, s);
    const int32_t i = __shfl_xor_sync(0xffffffffu, best_i, s);
    take(v, i);
  }
  if (lane == 0) {
    wv[warp] = best;
    wi[warp] = best_i;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kLgNT / 32; w++) take(wv[w], wi[w]);
    // into the first CTA's shared memory
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dsmem_addr(&cv[rank], 0)), "f"(best) : "memory");
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(dsmem_addr(&ci[rank], 0)), "r"(best_i) : "memory");
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0 && tid == 0) {
    best_i = -1;
    best = -INFINITY;
    for (int c = 0; c < kLgCluster; c++) take(cv[c], ci[c]);
    p.tokens[row] = best_i;
  }
}

}  // namespace

cudaError_t launch_logits_process(const LogitsParams& p, int64_t n_rows, cudaStream_t s) {
  if (n_rows == 0) return cudaSuccess;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_rows * kLgCluster));
  cfg.blockDim = dim3(kLgNT);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kLgCluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logits_process_kernel, p);
}

}  // namespace mi
