// Penalties for repeated tokens, biases and grammar masks on logits, with the
// greedy token of what is left. No counterpart in the reference, which picks the
// first maximum of the raw logits (ref src/model_qwen2.cpp:690-700).
//
// Row r, token j with logit l, c = how often j is in the row's history:
//   x = l;  c > 0: x = (l > 0 ? l / repeat : l * repeat) - (c * frequency + presence)
//   x += sum of the biases of j (in the list's order);  x = -inf where the allowed bit of j is 0
// token = the lowest j of the largest x, -1 where no x is above -inf.
//
// A row is one thread-block cluster: CTA c takes a contiguous part of the
// vocabulary and counts the history's tokens that fall into it in shared memory
// (integer adds: their order does not matter), so the counts never exist in global
// memory. The tokens with a count or a bias are few: they are listed when they are
// first met, computed from the list, and left out of the dense pass. (Computed
// inside it they cost every warp that met one the divisions of all its lanes, 60 us
// for 64 rows of 152064 with 4093 ids of history; computed by the thread of their
// history entry, 48 us.) The CTAs' winners meet in the first CTA's shared memory.
// A row is one pass, 8 bytes per token.
//
// Bound for many rows by HBM (8.1 bytes per token of the vocabulary: 64 rows of 152064
// without history or biases take 14 us, 5.6 TB/s) and by the phases before the dense
// pass (4093 ids of history and 300 biases: 23 us; as many biases as are listed, 2048: 66),
// for few rows by the latency of all phases.
#include <algorithm>

#include "mi_device.cuh"

namespace mi {

namespace {

constexpr int kLgNT = 512;
constexpr int kLgMaxCluster = 16;
constexpr int kLgBias = 2048;    // biases of a CTA's part that are kept in shared memory
constexpr int kLgList = 2048;    // tokens of a part with a count or a bias that are listed
constexpr int kLgAhead = 4;      // 16-byte pieces that a thread has under way

// Count words: 16 bits, or 32 for histories that 15 bits do not count. The top bit
// marks a token with a bias. add() and mark() give the word as it was.
constexpr int64_t kLgNarrow = 32767;  // the longest history for 16-bit words
template <bool WIDE>
struct Counts;
template <>
struct Counts<false> {
  static constexpr int bytes = 2;
  static constexpr uint32_t count = 0x7fffu, biased = 0x8000u;
  static __device__ __forceinline__ uint32_t add(uint32_t* w, int i) {
    return atomicAdd(w + (i >> 1), 1u << (16 * (i & 1))) >> (16 * (i & 1)) & 0xffffu;
  }
  static __device__ __forceinline__ uint32_t mark(uint32_t* w, int i) {
    return atomicOr(w + (i >> 1), biased << (16 * (i & 1))) >> (16 * (i & 1)) & 0xffffu;
  }
  static __device__ __forceinline__ uint32_t word(const uint32_t* w, int i) { return ((const uint16_t*)w)[i]; }
  // bit k: whether word i + k is not 0 (i a multiple of 4)
  static __device__ __forceinline__ uint32_t any4(const uint32_t* w, int i) {
    const uint2 v = *(const uint2*)((const uint16_t*)w + i);
    if ((v.x | v.y) == 0) return 0;
    return (v.x & 0xffffu ? 1u : 0u) | (v.x >> 16 ? 2u : 0u) | (v.y & 0xffffu ? 4u : 0u) | (v.y >> 16 ? 8u : 0u);
  }
};
template <>
struct Counts<true> {
  static constexpr int bytes = 4;
  static constexpr uint32_t count = 0x7fffffffu, biased = 0x80000000u;
  static __device__ __forceinline__ uint32_t add(uint32_t* w, int i) { return atomicAdd(w + i, 1u); }
  static __device__ __forceinline__ uint32_t mark(uint32_t* w, int i) { return atomicOr(w + i, biased); }
  static __device__ __forceinline__ uint32_t word(const uint32_t* w, int i) { return w[i]; }
  static __device__ __forceinline__ uint32_t any4(const uint32_t* w, int i) {
    const uint4 v = *(const uint4*)(w + i);
    return (v.x ? 1u : 0u) | (v.y ? 2u : 0u) | (v.z ? 4u : 0u) | (v.w ? 8u : 0u);
  }
};
// tokens counted at a time (a multiple of 32), at most; where their biases have sums, what
// lets two CTAs share an SM (64 rows, 4093 ids of history, 5000 biases: 140 us, 160 with
// one CTA; 40000 ids: 265 and 343)
constexpr int kLgSlice = 40960;
template <bool WIDE, bool MANY>
constexpr int kLgPer = MANY ? (WIDE ? 9600 : 12800) : kLgSlice;
template <bool WIDE, bool MANY>
constexpr int kLgBytes = Counts<WIDE>::bytes + (MANY ? 4 : 0);  // shared memory of a token

struct LgSmem {
  float cv[kLgMaxCluster], wv[kLgNT / 32];
  int32_t ci[kLgMaxCluster], wi[kLgNT / 32];
  int32_t bias_of[kLgNT / 32];
  int32_t n_list;
  int32_t list[kLgList];
};

// VEC: rows are 16-byte aligned, so four tokens a thread at a time. MANY: there are more
// than kLgBias biases, so that a part's may not fit; each token then has a sum beside its
// count, and when the list is full its biases are added there, a token's by one thread
// (in order). Otherwise each biased token goes through the part's list by itself: 64 rows
// with 2048 biases take 66 us so, 81 with 2049 and sums. (Tokens that went through the
// caller's list in global memory took 290 us there, 10 ms with 5000.)
template <bool WIDE, bool VEC, bool MANY>
__global__ void __launch_bounds__(kLgNT) logits_process_kernel(const LogitsParams p, const int cluster, const int slice) {
  using C = Counts<WIDE>;
  constexpr int NT = kLgNT;
  extern __shared__ __align__(16) uint32_t cnt[];
  // behind the counts: MANY, the tokens' sums; the part's biases, token (less s0) and value
  float* sums = (float*)((uint8_t*)cnt + slice * C::bytes);
  const int room = (int)min((int64_t)kLgBias, (p.n_bias + 3) / 4 * 4);
  int32_t* bias_id = (int32_t*)(sums + (MANY ? slice : 0));
  float* bias = (float*)(bias_id + room);
  __shared__ LgSmem sm;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_ctarank();
  if (p.tokens) cluster_arrive_relaxed();  // (every CTA runs before any stores into another's shared memory)
  const int64_t row = blockIdx.x / cluster, V = p.n_vocab;
  const int64_t per = ((V + cluster - 1) / cluster + 31) / 32 * 32;
  const int64_t v0 = min(V, (int64_t)rank * per), v1 = min(V, v0 + per);
  const float* x = p.logits + row * p.stride;
  float* y = p.out + row * V;
  const int32_t* hist = p.hist + (p.n_hist ? row * p.hist_stride : 0);
  const uint32_t* allowed = p.allowed ? p.allowed + row * p.allowed_stride : nullptr;
  const bool special = p.n_hist > 0 || p.n_bias > 0;
  float best = -INFINITY, best_s = -INFINITY;  // of the dense pass, which goes up, and of the others
  int32_t best_i = -1, best_si = -1;
  for (int64_t s0 = v0; s0 < v1; s0 += slice) {
    const int n = (int)min((int64_t)slice, v1 - s0);
    // the dense pass's first pieces are under way while the special tokens are seen to
    constexpr int W = VEC ? 4 : 1;
    const int np = n / W;  // (VEC: V is a multiple of 4, and so is n)
    float f[kLgAhead][W];
    uint32_t a[kLgAhead];
    // (loads only, from a place that is always there: a use or a branch between them
    // made each wait for the one before it, 6 of 19 us for 64 rows with masks)
    auto load = [&](int i0) {
#pragma unroll
      for (int u = 0; u < kLgAhead; u++) {
        const int i = min(i0 + u * NT, np - 1);
        if (VEC) {
          const float4 v = *(const float4*)(x + s0 + 4 * i);
          f[u][0] = v.x, f[u][W > 1 ? 1 : 0] = v.y, f[u][W > 2 ? 2 : 0] = v.z, f[u][W > 3 ? 3 : 0] = v.w;
        } else {
          f[u][0] = x[s0 + i];
        }
        a[u] = allowed ? allowed[(s0 + W * i) >> 5] : ~0u;
      }
    };
    load(tid);
    if (special) {
      int32_t h[8];
      auto history = [&](int64_t i0) {
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = i0 + e * NT < p.n_hist ? hist[i0 + e * NT] : -1;
      };
      history(tid);
      for (int i = tid; i < (n * C::bytes + 15) / 16; i += NT) ((uint4*)cnt)[i] = make_uint4(0, 0, 0, 0);
      if (tid == 0) sm.n_list = 0;
      __syncthreads();
      auto met = [&](int u) {  // the first entry of token s0 + u
        const int at = atomicAdd(&sm.n_list, 1);
        if (at < kLgList) sm.list[at] = u;
      };
      for (int64_t i0 = tid; i0 < p.n_hist; i0 += 8 * NT) {
        if (i0 != tid) history(i0);
        uint32_t old[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int64_t u = (int64_t)h[e] - s0;
          old[e] = u >= 0 && u < n ? C::add(cnt, (int)u) : 1u;
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (old[e] == 0) met((int)(h[e] - s0));
      }
      // the part's biases in the list's order
      int n_bias = 0;
      bool summed = false;
      auto sum = [&]() {
        for (int e = 0; e < n_bias; e += 4) {
          const int4 id = *(const int4*)(bias_id + e);
          auto add = [&](int k, int32_t u) {
            if (e + k < n_bias && (u & (NT - 1)) == tid) sums[u] = __fadd_rn(sums[u], bias[e + k]);
          };
          add(0, id.x);
          add(1, id.y);
          add(2, id.z);
          add(3, id.w);
        }
        summed = true;
      };
      int64_t u = tid < p.n_bias ? (int64_t)p.bias_ids[tid] - s0 : -1;
      for (int64_t b0 = 0; b0 < p.n_bias; b0 += NT) {
        const bool in = u >= 0 && u < n;
        const float v = in ? p.bias[b0 + tid] : 0.0f;
        const int64_t next = b0 + NT + tid < p.n_bias ? (int64_t)p.bias_ids[b0 + NT + tid] - s0 : -1;
        const uint32_t m = __ballot_sync(0xffffffffu, in);
        if (lane == 0) sm.bias_of[warp] = __popc(m);
        if (MANY && n_bias > kLgBias - NT) {
          sum();
          n_bias = 0;
        }
        __syncthreads();
        int at = n_bias + __popc(m & ((1u << lane) - 1)), all = 0;
        for (int w = 0; w < NT / 32; w++) {
          if (w < warp) at += sm.bias_of[w];
          all += sm.bias_of[w];
        }
        if (in) {
          const uint32_t old = C::mark(cnt, (int)u);
          if (old == 0) met((int)u);
          if (MANY && !(old & C::biased)) sums[u] = 0.0f;
          bias_id[at] = (int32_t)u;
          bias[at] = v;
        }
        u = next;
        n_bias += all;
        __syncthreads();
      }
      __syncthreads();
      const int n_list = sm.n_list;
      // (one thread's tokens after one another go through the list as often)
      if (MANY && n_bias > 0 && (summed || n_list > NT)) {
        sum();
        __syncthreads();
      }
      auto one = [&](int u) {  // token s0 + u
        const uint32_t c = C::word(cnt, u);
        const int64_t j = s0 + u;
        float v = x[j];
        if (c & C::count)
          v = __fsub_rn(v > 0.0f ? __fdiv_rn(v, p.repeat) : __fmul_rn(v, p.repeat),
                        __fadd_rn(__fmul_rn((float)(c & C::count), p.frequency), p.presence));
        if (c & C::biased) {
          float b = 0.0f;
          if (MANY && summed) {
            b = sums[u];
          } else {
            for (int e = 0; e < n_bias; e += 4) {
              const int4 id = *(const int4*)(bias_id + e);
              if (id.x == u) b = __fadd_rn(b, bias[e]);
              if (id.y == u && e + 1 < n_bias) b = __fadd_rn(b, bias[e + 1]);
              if (id.z == u && e + 2 < n_bias) b = __fadd_rn(b, bias[e + 2]);
              if (id.w == u && e + 3 < n_bias) b = __fadd_rn(b, bias[e + 3]);
            }
          }
          v = __fadd_rn(v, b);
        }
        if (allowed && !((allowed[j >> 5] >> (j & 31)) & 1u)) v = -INFINITY;
        y[j] = v;
        if (v > best_s || (v == best_s && (int32_t)j < best_si)) best_s = v, best_si = (int32_t)j;
      };
      if (n_list <= kLgList) {
        for (int i = tid; i < n_list; i += NT) one(sm.list[i]);
      } else {  // more than the list holds: every word is looked at
        for (int i = tid; i < n; i += NT)
          if (C::word(cnt, i)) one(i);
      }
    }
    for (int i0 = tid; i0 < np; i0 += NT * kLgAhead) {
      if (i0 != tid) load(i0);
#pragma unroll
      for (int u = 0; u < kLgAhead; u++) {
        const int i = i0 + u * NT;
        if (i >= np) continue;
        const int32_t j = (int32_t)(s0 + W * i);
        uint32_t skip = 0;  // tokens that are done
        if (special) skip = VEC ? C::any4(cnt, 4 * i) : (C::word(cnt, i) ? 1u : 0u);
#pragma unroll
        for (int k = 0; k < W; k++) {
          if (!((a[u] >> ((j + k) & 31)) & 1u)) f[u][k] = -INFINITY;
          if (f[u][k] > best && !((skip >> k) & 1u)) best = f[u][k], best_i = j + k;
        }
        if (VEC && skip == 0) {
          *(float4*)(y + j) = make_float4(f[u][0], f[u][W > 1 ? 1 : 0], f[u][W > 2 ? 2 : 0], f[u][W > 3 ? 3 : 0]);
        } else {
#pragma unroll
          for (int k = 0; k < W; k++)
            if (!((skip >> k) & 1u)) y[j + k] = f[u][k];
        }
      }
    }
    __syncthreads();
  }
  if (!p.tokens) return;
  auto take = [&](float v, int32_t i) {
    if (i >= 0 && (v > best || best_i < 0 || (v == best && i < best_i))) {
      best = v;
      best_i = i;
    }
  };
  take(best_s, best_si);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, s);
    const int32_t i = __shfl_xor_sync(0xffffffffu, best_i, s);
    take(v, i);
  }
  if (lane == 0) {
    sm.wv[warp] = best;
    sm.wi[warp] = best_i;
  }
  __syncthreads();
  cluster_wait_acquire();
  if (tid == 0) {
    for (int w = 1; w < NT / 32; w++) take(sm.wv[w], sm.wi[w]);
    // into the first CTA's shared memory
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dsmem_addr(&sm.cv[rank], 0)), "f"(best) : "memory");
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(dsmem_addr(&sm.ci[rank], 0)), "r"(best_i) : "memory");
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank == 0 && tid == 0) {
    best_i = -1;
    best = -INFINITY;
    for (int c = 0; c < cluster; c++) take(sm.cv[c], sm.ci[c]);
    p.tokens[row] = best_i;
  }
}

template <bool WIDE, bool VEC, bool MANY>
cudaError_t launch_logits(const LogitsParams& p, int64_t n_rows, cudaStream_t s) {
  // CTAs of a row: 16 while the rows are few, 8, and 4 where all of them still run at
  // once (us for 4 / 13 / 24 / 64 rows of 152000: 7.5 / 10.0 / 18.2 / 50.1 with 16,
  // 9.0 / 9.1 / 12.4 / 29.4 with 8, 11.6 / 11.9 / 12.0 / 22.7 with 4; every CTA of a row
  // reads all of its history).
  const int cluster = n_rows <= 6 ? 16 : n_rows <= 20 ? 8 : 4;
  const int64_t per = ((p.n_vocab + cluster - 1) / cluster + 31) / 32 * 32;
  const int64_t slices = (per + kLgPer<WIDE, MANY> - 1) / kLgPer<WIDE, MANY>;
  const int slice = (int)((per + slices - 1) / slices + 31) / 32 * 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_rows * cluster));
  cfg.blockDim = dim3(kLgNT);
  cfg.dynamicSmemBytes = p.n_hist || p.n_bias ? (size_t)slice * kLgBytes<WIDE, MANY> + (std::min<int64_t>(p.n_bias, kLgBias) + 3) / 4 * 4 * 8 : 0;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logits_process_kernel<WIDE, VEC, MANY>, p, cluster, slice);
}
template <bool WIDE, bool VEC>
cudaError_t launch_logits(const LogitsParams& p, int64_t n_rows, cudaStream_t s) {
  return p.n_bias > kLgBias ? launch_logits<WIDE, VEC, true>(p, n_rows, s) : launch_logits<WIDE, VEC, false>(p, n_rows, s);
}

template <bool WIDE, bool VEC, bool MANY>
cudaError_t prepare_logits() {
  cudaError_t e = cudaFuncSetAttribute(logits_process_kernel<WIDE, VEC, MANY>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kLgPer<WIDE, MANY> * kLgBytes<WIDE, MANY> + kLgBias * 8);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(logits_process_kernel<WIDE, VEC, MANY>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}
template <bool WIDE>
cudaError_t prepare_logits_of() {
  cudaError_t e = prepare_logits<WIDE, false, false>();
  if (e == cudaSuccess) e = prepare_logits<WIDE, true, false>();
  if (e == cudaSuccess) e = prepare_logits<WIDE, false, true>();
  return e == cudaSuccess ? prepare_logits<WIDE, true, true>() : e;
}

}  // namespace

// (the counts' shared memory and clusters of 16 CTAs need attributes; per device, at init)
cudaError_t prepare_logits_kernels() {
  const cudaError_t e = prepare_logits_of<false>();
  return e == cudaSuccess ? prepare_logits_of<true>() : e;
}

cudaError_t launch_logits_process(const LogitsParams& p, int64_t n_rows, cudaStream_t s) {
  if (n_rows == 0) return cudaSuccess;
  const bool vec = ((uintptr_t)p.logits | (uintptr_t)p.out) % 16 == 0 && p.stride % 4 == 0 && p.n_vocab % 4 == 0;
  if (p.n_hist <= kLgNarrow) return vec ? launch_logits<false, true>(p, n_rows, s) : launch_logits<false, false>(p, n_rows, s);
  return vec ? launch_logits<true, true>(p, n_rows, s) : launch_logits<true, false>(p, n_rows, s);
}

}  // namespace mi
