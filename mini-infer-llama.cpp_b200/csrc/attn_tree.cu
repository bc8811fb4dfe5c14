// Attention of a tree of drafted tokens over a cache. No counterpart in the
// reference, whose attention knows only a causal run of tokens
// (ref src/ops_cpu.cpp:304-410).
//
// Token i of T attends to cache rows [0, n_past) and to row n_past + j (drafted
// token j's) where bit j of its mask is set; without a mask to j <= i.
//   s = scale q.k,  p = e^(s - max s),  out = sum p v / sum p
// over the attended rows, and zeros where there is none. The cache is F32
// ([n_ctx][n_head_kv][D]) or Q8_0 (kv_q8.cu).
//
// The n_rep query heads of a KV head times T tokens are the rows of two matrix
// products over the KV head's positions, S = Q K^T and O = P V, and run on the
// tensor cores (tcgen05) at float precision:
//
//   * every operand is split into two fp16 planes, x = hi + lo, after its row was
//     scaled by a power of two (so that neither half leaves fp16's range): hi + lo
//     is x to 22 bits, and for a Q8_0 value exactly (11 bits of scale times 7 of
//     quant: hi = fl(d q) and lo = fma(d, q, -hi) is the whole rest). A product
//     takes three MMAs (hi hi, hi lo, lo hi); what is left out is 2^-22 of it.
//   * the rows' powers of two leave the products as factors: the keys' exponent
//     multiplies S, the values' exponent e is added to the score that makes P
//     (P = 2^(s + e - M)), and the sum of the weights takes it out again. The 64
//     positions of a step share both exponents unless their rows' magnitudes are
//     more than 2^10 apart or one holds an infinity or a NaN; only then does every
//     position have its own (a masked row's value then takes nothing from the
//     others' precision).
//
// One CTA: 128 rows (a TMEM lane each) over one range of positions, 128 a step.
// Warps 0-15 softmax: four threads per row, 32 positions each; 16-19 convert keys
// and 20-23 values into the MMAs' layout in shared memory; 24 issues the MMAs; 25 and
// 26 ask for the cache ahead (Q8_0: into L2; F32: its rows into shared memory). The
// queries' planes are copied into TMEM: as a shared-memory operand they are 4 KB a
// product beside the keys' 4, and shared memory, not the tensor core, set the pace.
// S, P's planes, O and the queries' planes fill TMEM's 512 columns at D = 128. The
// next step's scores run under a step's exponentials and its P V under the next
// one's.
//
// What bounds it: the softmax threads (of some 3450 cycles a step at D = 64 the
// exponentials are 1400, the rest round trips between its phases; steps of 64 positions
// took nearly as long as steps of 128), the converters close behind at D = 128. 64
// tokens, 28 / 4 heads of 128 over 8175 positions: 33 us; 14 / 2 heads of 64 over
// 32764: 39 us.
//
// More than one tile of rows: two CTAs of a cluster take two tiles over the same
// positions as one pair (cta_group::2). One of them issues the MMAs of both, 256 rows
// each; B is split between their shared memories, so each converts half of a step's
// keys (64 positions) and half of its values (half of the dims). With a CTA by itself
// the conversion is 40 % of the issued instructions and, at D = 128, there is no room
// for a second step's values; stores or bulk copies of converted planes into the
// other CTAs' shared memory took longer than converting them again.
//
// A step's O is a product of its own, added to the softmax threads' registers
// (O = O 2^(M_old - M_new) + O_step): the MMA's accumulation cuts instead of
// rounding, by half an ulp of the accumulator each time, and over a thousand
// positions accumulated in TMEM that came to 7e-6 of the result, one-signed. For
// the same reason the small products (hi lo, lo hi) come first in each step.
//
// The positions are split over CTAs to fill the GPU; a second kernel joins the
// splits' (M, sum, O) records.
#include <algorithm>
#include <type_traits>

#include "attn_tree.cuh"
#include "mi_tc.cuh"

namespace mi {

namespace {

constexpr int kTrTile = 128;     // positions per step
constexpr int kTrHalf = 64;      // ... that share their exponents
constexpr int kTrParts = 4;      // softmax threads per row: 32 positions each, and a quarter of O's dims
constexpr int kTrRows = 128;     // rows per CTA (MMA M)
constexpr int kTrWarpK = 16, kTrWarpV = 20, kTrWarpMma = 24;
constexpr int kTrThreads = 28 * 32;  // (the last warp completes the MMA warp's group for setmaxnreg)
constexpr int kTrChunk = 16;     // F32: rows of a cache that are copied at a time
constexpr int kTrSlots = 8;      // steps whose exponents are kept (see the roles' waits)
constexpr uint32_t kTrCols = 512;  // all of TMEM: its base is 0
constexpr uint32_t kTmem = 0;
// TMEM columns: S, P's planes (64 + 64), O, the queries' planes (D / 2 each)
constexpr uint32_t kColS = 0, kColP = 128, kColO = 256, kColQ = 384;
// Registers per thread of the roles: launched with 72 x 896 = 64512, of which
// 88 x 512 + 56 x 256 + 40 x 128 = 64512 are given out again.
constexpr int kRegsSoftmax = 88, kRegsConvert = 56, kRegsMma = 40;

// PAIR: two CTAs share the products' B operand.
template <int D, bool Q8, bool PAIR>
struct TrSmem {
  // steps whose planes there is room for
  static constexpr int n_v = PAIR || D <= 64 ? 2 : 1, n_k = Q8 ? 2 : n_v;
  static constexpr int plane = kTrTile * D * 2 / (PAIR ? 2 : 1);  // of a CTA's share of the keys or the values
  static constexpr int k = 0;                      // [step % n_k][hi, lo]; at the end float [128][D + 4], the rows' records
  static constexpr int v = k + n_k * 2 * plane;    // [step % n_v][hi, lo]; before the first step the queries
  static constexpr int col = v + n_v * 2 * plane;  // float [kTrSlots][half][2][64]: key factor, value exponent
  static constexpr int info = col + kTrSlots * 2 * 2 * kTrHalf * 4;  // float [kTrSlots][half][4]: key factor, whether the positions have
                                                                     // their own, value exponent, whether they have their own
  static constexpr int ends = info + kTrSlots * 2 * 16;  // int2 [keys, values][step & 1][half][4 warps]: largest and least exponent
  static constexpr int mx = ends + 2 * 2 * 2 * 4 * 8;    // float [2][part][128]: the parts' maxima (at the end their sums)
  // F32: rows as they are, in chunks of 16 (8 where there is room for them)
  static constexpr int n_rows = Q8 ? 0 : D <= 96 ? 8 : 5, pitch = D + 4;  // chunks of each cache; floats between rows (a
                                                                         // column of eight rows in all banks)
  static constexpr int rows = mx + 2 * kTrParts * kTrRows * 4;           // float [keys, values][n_rows][16][pitch]
  static constexpr int bars = rows + 2 * n_rows * kTrChunk * pitch * 4;
  static constexpr int n_bars = 2 * n_k + 2 * n_v + 2 * kTrSlots + 8 + 4 * n_rows;
  static constexpr int misc = bars + n_bars * 8;   // TMEM base, abort flag
  static constexpr int used = misc + 16;
  // above half of an SM's shared memory: two CTAs must not share its TMEM
  static constexpr int total = used > 120 * 1024 ? used : 120 * 1024;
  static_assert(kTrRows * (D + 4) * 4 <= v + n_v * 2 * plane, "the records fit where the planes were");
  static_assert(kTrRows * D * 4 <= n_v * 2 * plane, "the queries fit where the values will be");
  static_assert(total <= 227 * 1024, "shared memory of one CTA");
};

// Arrives on a barrier of the CTA that issues (its shared::cluster address). What the
// barrier stands for is in TMEM, behind tcgen05.wait and fence, or in this CTA's own
// shared memory, behind the fence to the async proxy: it has been performed before
// this, and nothing else has to be made visible (a release for the whole cluster
// waited for the loads in flight as well, 900 to 1250 cycles each time).
__device__ __forceinline__ void arrive_lead(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// True in one lane of a converged warp (always the same one).
__device__ __forceinline__ bool elect_one() {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(y));
  return y != 0;
}

// D (+)= A B, f32 += f16 x f16; A from TMEM, B from shared memory (of both CTAs).
template <bool PAIR>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0u)
        : "memory");
}
// Arrives on `bar` (of both CTAs) when the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  if (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    umma_commit(bar);
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
      "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(addr));
}
// tcgen05.wait::ld with the loaded registers threaded through it, so that none
// of their uses is scheduled before it.
__device__ __forceinline__ void tmem_wait_ld(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                 "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]),
                 "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]),
                 "+f"(r[30]), "+f"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_ld8f(uint32_t addr, float* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld8(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t addr, uint4 a) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Eight floats (scaled) as the two fp16 planes' 16-byte pieces.
__device__ __forceinline__ void split8(const float* x, float f, uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float a = __fmul_rn(x[2 * i], f), b = __fmul_rn(x[2 * i + 1], f);
    const __half2 hh = __floats2half2_rn(a, b);
    const float2 back = __half22float2(hh);
    h[i] = h2_bits(hh);
    l[i] = h2_bits(__floats2half2_rn(__fsub_rn(a, back.x), __fsub_rn(b, back.y)));
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// A CTA's share of one cache (keys or values) of one KV head, by four warps: of a
// step's 128 positions NK * 4 row groups of eight, of their dims CH pieces of eight
// (all of both by itself; in a pair half the groups of the keys, half the pieces of
// the values). A warp takes groups w + 4 k, k < NK; lane = position % 8 + 8 g, and
// pieces g + 4 i. A piece is 16 bytes of each plane: core matrices of 8 positions x
// 8 dims.
//
// The exponent of a row (planes = row * 2^-e brings it to fp16's range) is that of
// its largest scale, or for F32 of its largest value.
// Q8_0: two of a warp's rows are in registers; a row that has been converted makes
// room for the one after the next.
template <int D, int NK, int CH>
struct KvRows {
  static constexpr int NC = D / 32, ND = (NC + 1) / 2, NI = (CH + 3) / 4;
  uint2 q[2][NI];
  uint32_t d[2][ND];    // two scales a word
  uint32_t all[4][ND];  // the scales of the step's positions lane + 32 k: every warp finds the exponents itself
  const uint8_t* qs;    // the head's quants (this share's dims) and scales from this CTA's first position on
  const uint16_t* ds;
  int64_t left;         // positions from there on
  int row0, ch0;        // this share's first position of a step, first piece

  static __device__ __forceinline__ void scales(const uint16_t* s, bool in, uint32_t (&o)[ND]) {
#pragma unroll
    for (int i = 0; i < ND; i++)
      o[i] = !in ? 0u : NC % 2 == 0 ? *(const uint32_t*)(s + 2 * i) : s[2 * i] | (2 * i + 1 < NC ? (uint32_t)s[2 * i + 1] << 16 : 0u);
  }
  // the largest scale becomes 1..2 (below it for subnormal ones); false for a NaN scale
  static __device__ __forceinline__ bool exponent(const uint32_t (&s)[ND], int& e, bool& any) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < ND; i++) m = max(m, max(s[i] & 0x7fffu, (s[i] >> 16) & 0x7fffu));
    e = max((int)(m >> 10), 1) - 15;
    any = m != 0;
    return m < 0x7c00u;
  }
  __device__ __forceinline__ void load_all(int at, int lane) {
#pragma unroll
    for (int k = 0; k < 4; k++) scales(ds + (int64_t)(at + lane + 32 * k) * NC, at + lane + 32 * k < left, all[k]);
  }
  // row k of the step at `at` into buffer b
  __device__ __forceinline__ void load_row(int k, int b, int at, int w, int lane) {
    const int pos = at + row0 + (w + 4 * k) * 8 + (lane & 7), g = lane >> 3;
    const bool in = pos < left;
    const uint8_t* src = qs + (int64_t)pos * D + 8 * g;
    scales(ds + (int64_t)pos * NC, in, d[b]);
#pragma unroll
    for (int i = 0; i < NI; i++) q[b][i] = in && g + 4 * i < CH ? *(const uint2*)(src + 32 * i) : make_uint2(0u, 0u);
  }
  __device__ __forceinline__ void begin(const TreeAttnParams& p, const void* cache, int kvh, int64_t pos0, int64_t n_kv, int w, int lane,
                                        int first_row, int first_piece) {
    const int64_t at = (int64_t)kvh * p.n_ctx + pos0;
    row0 = first_row;
    ch0 = first_piece;
    qs = (const uint8_t*)cache + at * D + 8 * ch0;
    ds = (const uint16_t*)((const uint8_t*)cache + (int64_t)p.HKV * p.n_ctx * D) + at * NC;
    left = n_kv - pos0;
    load_all(0, lane);
    load_row(0, 0, 0, w, lane);
    load_row(1, 1, 0, w, lane);
  }
  // The largest and least exponent of each half's rows that have a value but 0
  // (least is -2000 where a row has a NaN scale); those of rows that have their own
  // go to put(half, position in it, exponent, whether it is no NaN).
  template <class Own, class Put>
  __device__ __forceinline__ void exponents(int at, int w, int lane, int (&most)[2], bool (&own)[2], Own judge, Put put) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      bool bad = false;
      int e[2], hi = -1000, lo = 1000;
      bool fine[2];
#pragma unroll
      for (int k = 0; k < 2; k++) {
        bool any;
        fine[k] = exponent(all[2 * h + k], e[k], any);
        bad |= !fine[k];
        if (fine[k] && any) {
          hi = max(hi, e[k]);
          lo = min(lo, e[k]);
        }
      }
      hi = __reduce_max_sync(0xffffffffu, hi);
      lo = __reduce_min_sync(0xffffffffu, lo);
      if (__any_sync(0xffffffffu, bad)) lo = -2000;
      most[h] = hi;
      own[h] = judge(hi, lo);
      if (own[h] && (lane >> 3) == w) {
#pragma unroll
        for (int k = 0; k < 2; k++) put(h, lane + 32 * k, e[k], fine[k]);
      }
    }
    load_all(at + kTrTile, lane);
  }
  // row k, in buffer b
  __device__ __forceinline__ void convert(int k, int b, uint8_t* planes, int w, int lane, const int (&most)[2], const bool (&own)[2]) const {
    const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
    const int g = lane >> 3;
    const bool second = row0 + 32 * k >= kTrHalf;  // of the step's halves
    int e = second ? most[1] : most[0];
    bool fine = true, any;
    if (second ? own[1] : own[0]) fine = exponent(d[b], e, any);
    // 2^-e: fp16 holds 2^14 down to 2^-15
    const __half down = __float2half_rn(fine ? pow2f(-e) : 0.0f);
    uint8_t* dst = planes + (w + 4 * k) * (CH * 128) + g * 128 + (lane & 7) * 16;
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int blk = (ch0 + g + 4 * i) >> 2;
      uint32_t sd = d[b][0];
#pragma unroll
      for (int u = 1; u < ND; u++) sd = (blk >> 1) == u ? d[b][u] : sd;
      const __half s = __ushort_as_half(fine ? (uint16_t)(blk & 1 ? sd >> 16 : sd) : (uint16_t)0);
      const __half2 f = __half2half2(__hmul_rn(s, down));
      uint32_t h[4], l[4];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const uint32_t x = (j < 2 ? q[b][i].x : q[b][i].y) ^ 0x80808080u;
        // two signed bytes as fp16: 1024 + (byte + 128) - 1152
        const uint32_t t = __byte_perm(x, 0x64646464u, j & 1 ? 0x7362 : 0x5140);
        const __half2 n = __hsub2_rn(*reinterpret_cast<const __half2*>(&t), off);
        const __half2 hh = __hmul2_rn(n, f);
        h[j] = h2_bits(hh);
        l[j] = h2_bits(__hfma2(n, f, __hneg2(hh)));
      }
      if (CH % 4 == 0 || g + 4 * i < CH) {
        *(uint4*)(dst + i * 512) = make_uint4(h[0], h[1], h[2], h[3]);
        *(uint4*)(dst + NK * 4 * CH * 128 + i * 512) = make_uint4(l[0], l[1], l[2], l[3]);
      }
    }
  }
  __device__ __forceinline__ void store(int at, uint8_t* planes, int w, int lane, const int (&most)[2], const bool (&own)[2]) {
#pragma unroll 1
    for (int u = 0; u < NK; u += 2) {
      // (the row that a buffer takes next: two on, or this one of the next step)
      const int next = NK == 4 ? u ^ 2 : u, to = NK == 4 && u == 0 ? at : at + kTrTile;
      convert(u, 0, planes, w, lane, most, own);
      load_row(next, 0, to, w, lane);
      convert(u + 1, 1, planes, w, lane, most, own);
      load_row(next + 1, 1, to, w, lane);
    }
  }
};

// What a converting warp needs of its CTA.
struct TrConvert {
  int64_t pos0, n_kv;
  int kvh, n, w, lane, rank;
  const void* cache;
  uint8_t* planes;  // [n_buf][hi, lo]
  uint64_t *empty, *col_full;
  uint32_t full;    // shared::cluster address of the issuing CTA's barriers
  float *col, *info;
  volatile int* abort_flag;
  // F32
  float* rows;      // [n_rows][kTrChunk][D + 4]
  uint64_t *rows_full, *rows_empty;
  int2* ends;       // [step & 1][half][4 warps]: largest and least exponent
};

// Where 64 positions have magnitudes too far apart for one exponent (or one that is
// not finite).
__device__ __forceinline__ bool too_far_apart(int hi, int lo) { return lo < 1000 && hi - lo > 10; }

// One position's own exponent.
template <bool IS_V>
__device__ __forceinline__ void put_own(const TrConvert& r, int slot, int half, int at, int e, bool fine) {
  float* c = r.col + (slot * 2 + half) * 2 * kTrHalf;
  const float nan = __int_as_float(0x7fffffff);
  if (IS_V) c[kTrHalf + at] = fine ? (float)e : nan;
  else c[at] = fine ? pow2f(e) : nan;
}
template <bool IS_V>
__device__ __forceinline__ void put_info(const TrConvert& r, int slot, int half, int most, bool own) {
  if (r.w == 0 && r.lane == 0)
    *(float2*)(r.info + (slot * 2 + half) * 4 + (IS_V ? 2 : 0)) = make_float2(IS_V ? (float)most : pow2f(most), own ? 1.0f : 0.0f);
}

// The keys (or values) of every step. A step's exponents go out before its planes,
// which wait for the products that read the planes there before. Their slot is
// written again eight steps later: after the planes of seven, for which the scores of
// five were done, for which the softmax had read those of four, and so had long left
// the step itself.
template <int D, bool PAIR, bool IS_V, int n_buf>
__device__ __forceinline__ void convert_q8_0(const TreeAttnParams& p, const TrConvert& r, uint64_t* queries_done, bool wait_queries) {
  constexpr int NK = PAIR && !IS_V ? 2 : 4, CH = PAIR && IS_V ? D / 16 : D / 8, plane = NK * 4 * CH * 128;
  KvRows<D, NK, CH> kv;
  kv.begin(p, r.cache, r.kvh, r.pos0, r.n_kv, r.w, r.lane, PAIR && !IS_V ? r.rank * kTrHalf : 0, PAIR && IS_V ? r.rank * CH : 0);
  bool ok = true;
  for (int j = 0; j < r.n; j++) {
    const int slot = j & (kTrSlots - 1), b = j % n_buf;
    int most[2];
    bool own[2];
    kv.exponents(j * kTrTile, r.w, r.lane, most, own, too_far_apart,
                 [&](int h, int at, int e, bool fine) { put_own<IS_V>(r, slot, h, at, e, fine); });
#pragma unroll
    for (int h = 0; h < 2; h++) {
      if (most[h] < -999) most[h] = 0;  // (nothing but zeros)
      put_info<IS_V>(r, slot, h, most[h], own[h]);
    }
    __syncwarp();
    if (r.lane < 2) mbar_arrive_one(&r.col_full[slot * 2 + r.lane]);
    ok = ok && (j < n_buf || tc_wait_ready(&r.empty[b], (uint32_t)(j / n_buf - 1) & 1u, r.abort_flag, p.err));
    // (the first values lie where the queries were)
    if (IS_V && j == 0 && wait_queries) ok = ok && tc_wait_ready(queries_done, 0, r.abort_flag, p.err);
    if (ok) {
      kv.store(j * kTrTile, r.planes + b * 2 * plane, r.w, r.lane, most, own);
      fence_proxy_async_smem();
      __syncwarp();
      if (r.lane == 0) arrive_lead(r.full + 8 * b);
    }
  }
}

// The same from an F32 cache, whose rows the copying warps leave in shared memory,
// 64 positions at a time: read there for their exponents, and again for their planes.
// (Both times from global memory, a step took 15 us at D = 128, 5 times the softmax.)
template <int D, bool PAIR, bool IS_V, int n_buf, int n_rows>
__device__ __forceinline__ void convert_f32(const TreeAttnParams& p, const TrConvert& r, uint64_t* queries_done, bool wait_queries) {
  constexpr int NK = PAIR && !IS_V ? 2 : 4, CH = PAIR && IS_V ? D / 16 : D / 8, plane = NK * 4 * CH * 128, pitch = D + 4;
  const int ch0 = PAIR && IS_V ? r.rank * CH : 0, w = r.w, lane = r.lane, g = lane >> 3;
  const int64_t left = r.n_kv - r.pos0;
  bool ok = true;
  for (int j = 0; j < r.n; j++) {
    const int slot = j & (kTrSlots - 1), b = j % n_buf;
#pragma unroll 1
    for (int h = 0; h < 2; h++) {
      // row groups w + 4 k of the step, k = 2 h and 2 h + 1: half a chunk each
      const float* src[2];
      int e[2], hi = -1000, lo = 1000;
      bool fine[2], in[2], bad = false;
      uint64_t* done[2];
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int k = 2 * h + u, c = j * (kTrTile / kTrChunk) + (w >> 1) + 2 * k, at = c % n_rows;
        ok = ok && tc_wait_ready(&r.rows_full[at], (uint32_t)(c / n_rows) & 1u, r.abort_flag, p.err);
        done[u] = &r.rows_empty[at];
        src[u] = r.rows + (at * kTrChunk + (w & 1) * 8 + (lane & 7)) * pitch;
        in[u] = (int64_t)j * kTrTile + (w + 4 * k) * 8 + (lane & 7) < left;
        uint32_t m = 0;  // the largest magnitude's bits (those of an infinity or a NaN are above all others)
        if (ok && in[u]) {
#pragma unroll
          for (int i = 0; i < D / 32; i++) {
            const uint4* x = (const uint4*)(src[u] + (g + 4 * i) * 8);
            const uint4 a = x[0], c4 = x[1];
            m = max(max(max(m, a.x & 0x7fffffffu), max(a.y & 0x7fffffffu, a.z & 0x7fffffffu)), a.w & 0x7fffffffu);
            m = max(max(max(m, c4.x & 0x7fffffffu), max(c4.y & 0x7fffffffu, c4.z & 0x7fffffffu)), c4.w & 0x7fffffffu);
          }
        }
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
        // The row's largest magnitude becomes 2^14..2^15. Rows below 2^-100 keep -100:
        // their halves lose bits below 2^-138, nothing that a float sum of products shows.
        fine[u] = m < 0x7f800000u;
        e[u] = max((int)(m >> 23) - 127, -100);
        bad |= !fine[u];
        const bool any = m != 0;
        e[u] -= 14;
        if (fine[u] && any) {
          hi = max(hi, e[u]);
          lo = min(lo, e[u]);
        }
      }
      hi = __reduce_max_sync(0xffffffffu, hi);
      lo = __reduce_min_sync(0xffffffffu, lo);
      if (__any_sync(0xffffffffu, bad)) lo = -2000;
      int2* ends = r.ends + ((j & 1) * 2 + h) * 4;
      if (lane == 0) ends[w] = make_int2(hi, lo);
      // (also warps that have given up)
      asm volatile("bar.sync %0, 128;" ::"r"(IS_V ? 6 : 5) : "memory");
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int2 o = ends[k];
        hi = max(hi, o.x);
        lo = min(lo, o.y);
      }
      const bool own = too_far_apart(hi, lo);
      const int most = hi < -999 ? 0 : hi;
      if (own && lane < 8) {
#pragma unroll
        for (int u = 0; u < 2; u++) put_own<IS_V>(r, slot, h, (w + 4 * u) * 8 + lane, e[u], fine[u]);
      }
      put_info<IS_V>(r, slot, h, most, own);
      __syncwarp();
      if (lane == 0) mbar_arrive_one(&r.col_full[slot * 2 + h]);
      const bool share = !PAIR || IS_V || h == r.rank;  // whether these rows' planes are this CTA's
      if (share && (h == 0 || (PAIR && !IS_V))) {       // (the step's first)
        ok = ok && (j < n_buf || tc_wait_ready(&r.empty[b], (uint32_t)(j / n_buf - 1) & 1u, r.abort_flag, p.err));
        // (the first values lie where the queries were)
        if (IS_V && j == 0 && wait_queries) ok = ok && tc_wait_ready(queries_done, 0, r.abort_flag, p.err);
      }
      if (ok && share) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const bool take = in[u] && (!own || fine[u]);
          const float f = pow2f(own ? -e[u] : -most);
          uint8_t* dst = r.planes + b * 2 * plane + (w + 4 * (NK == 2 ? u : 2 * h + u)) * (CH * 128) + g * 128 + (lane & 7) * 16;
#pragma unroll
          for (int i = 0; i < (CH + 3) / 4; i++) {
            if (CH % 4 != 0 && g + 4 * i >= CH) continue;
            uint4 up = make_uint4(0, 0, 0, 0), down = up;
            if (take) {
              const float4* from = (const float4*)(src[u] + (ch0 + g + 4 * i) * 8);
              const float4 a = from[0], c4 = from[1];
              const float x[8] = {a.x, a.y, a.z, a.w, c4.x, c4.y, c4.z, c4.w};
              split8(x, f, up, down);
            }
            *(uint4*)(dst + i * 512) = up;
            *(uint4*)(dst + plane + i * 512) = down;
          }
        }
      }
      __syncwarp();
      if (ok && lane < 2) mbar_arrive_one(lane == 0 ? done[0] : done[1]);
    }
    if (ok) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) arrive_lead(r.full + 8 * b);
    }
  }
}

// One warp copies the rows of an F32 cache into shared memory, as far ahead as there
// is room. (In 16-byte pieces: a bulk copy a row took some 45 cycles each whatever its
// size, 11 us a step.) It leaves only when its copies have arrived.
template <int D, int n_rows>
__device__ __forceinline__ void copy_rows(const TreeAttnParams& p, const float* cache, int kvh, int64_t pos0, int64_t n_kv, int n, int lane,
                                          float* rows, uint64_t* full, uint64_t* empty, volatile int* abort_flag) {
  constexpr int pitch = D + 4, pieces = D / 4;
  const int64_t row = (int64_t)p.HKV * D;
  const float* src = cache + pos0 * row + (int64_t)kvh * D;
  const int64_t left = n_kv - pos0;
  for (int c = 0; c < n * (kTrTile / kTrChunk); c++) {
    const int at = c % n_rows;
    if (c >= n_rows && !tc_wait_ready(&empty[at], (uint32_t)(c / n_rows - 1) & 1u, abort_flag, p.err)) break;
    const uint32_t to = smem_addr(rows + at * kTrChunk * pitch);
    const float* from = src + (int64_t)c * kTrChunk * row;
    const int here = (int)max((int64_t)0, min((int64_t)kTrChunk, left - (int64_t)c * kTrChunk));
#pragma unroll
    for (int i = 0; i < kTrChunk * pieces / 32; i++) {
      const int e = lane + 32 * i, r = e / pieces, k = e - r * pieces;
      if (r < here)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (r * pitch + 4 * k) * 4), "l"(from + r * row + 4 * k) : "memory");
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_addr(&full[at])) : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int D, bool Q8, bool PAIR>
__global__ void __launch_bounds__(kTrThreads, 1) attn_tree_kernel(const __grid_constant__ TreeAttnParams p,
                                                                  const TreeSplit sp, const int vec_q) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using L = TrSmem<D, Q8, PAIR>;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.z, kvh = blockIdx.y, r0 = blockIdx.x * kTrRows;
  const int rep = p.H / p.HKV;
  const int64_t n_kv = (int64_t)p.n_past + p.T;
  const int64_t pos0 = (int64_t)split * sp.per * kTrTile;
  const int n = (int)min((int64_t)sp.per, (n_kv - pos0 + kTrTile - 1) / kTrTile);  // steps of this CTA, at least one
  const int rank = PAIR ? (int)cluster_ctarank() : 0;  // CTA 0 of a pair issues the MMAs
  // quadrants of 32 rows in use, kTrParts softmax warps each: here (none, where a pair
  // has no second tile) and in the pair
  const int nq = max(0, min(4, (sp.R - r0 + 31) / 32));
  const int nq_all = PAIR ? max(0, min(8, (sp.R - (r0 - rank * kTrRows) + 31) / 32)) : nq;
  float* col = (float*)(smem + L::col);
  float* info = (float*)(smem + L::info);
  float* mxs = (float*)(smem + L::mx);
  uint64_t* k_full = (uint64_t*)(smem + L::bars);  // [step % n_k]
  uint64_t* k_empty = k_full + L::n_k;
  uint64_t* v_full = k_empty + L::n_k;  // [step % n_v]
  uint64_t* v_empty = v_full + L::n_v;
  uint64_t* col_full = v_empty + L::n_v;  // [kTrSlots][half]
  uint64_t* s_full = col_full + 2 * kTrSlots;
  uint64_t* s_empty = s_full + 1;
  uint64_t* p_full = s_full + 2;
  uint64_t* o_full = s_full + 3;
  uint64_t* t_full = s_full + 4;  // TMEM is there
  uint64_t* q_full = s_full + 5;  // the queries are in TMEM (of both CTAs)
  uint64_t* drain = s_full + 6;
  uint64_t* q_here = s_full + 7;  // ... of this one
  uint64_t* rows_full = s_full + 8;               // F32: [keys, values][chunk % n_rows]
  uint64_t* rows_empty = rows_full + 2 * L::n_rows;
  uint32_t* tmem_base = (uint32_t*)(smem + L::misc);
  volatile int* abort_flag = (volatile int*)(smem + L::misc + 4);

  // Barriers that the issuing warp waits on lie in CTA 0 and count both CTAs' warps;
  // its commits arrive in both.
  if (tid == 0) {
    for (int i = 0; i < L::n_k; i++) {
      mbar_init(&k_full[i], PAIR ? 8 : 4);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < L::n_v; i++) {
      mbar_init(&v_full[i], PAIR ? 8 : 4);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2 * kTrSlots; i++) mbar_init(&col_full[i], 8);
    mbar_init(s_full, 1);
    mbar_init(s_empty, kTrParts * nq_all);
    mbar_init(p_full, kTrParts * nq_all);
    mbar_init(o_full, 1);
    mbar_init(t_full, 1);
    mbar_init(q_full, kTrParts * nq_all + (PAIR ? 2 : 1));
    mbar_init(drain, 1);
    mbar_init(q_here, max(1, kTrParts * nq));
    for (int i = 0; i < 2 * L::n_rows; i++) {
      mbar_init(&rows_full[i], 32);
      mbar_init(&rows_empty[i], 2);  // (a chunk is read by two warps)
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (PAIR) cluster_sync_all();
  else __syncthreads();
  auto lead = [](uint64_t* bar) { return dsmem_addr(bar, 0); };
  const uint32_t s_empty0 = lead(s_empty), p_full0 = lead(p_full), q_full0 = lead(q_full);

  if (warp >= kTrWarpMma) {
    // ---------------- MMA issue ----------------
    // The whole warp runs the loop and one elected lane issues: descriptors then
    // stay in uniform registers (in a branch of one lane each MMA cost 100 cycles
    // to issue, three times what it takes to run).
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
    if (warp == kTrWarpMma) {
      if (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_base)), "r"(kTrCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
      } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_base)), "r"(kTrCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_one(t_full);
        arrive_lead(q_full0);
      }
      constexpr uint32_t M = kTrRows * (PAIR ? 2 : 1);
      constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(kTrTile >> 3) << 17) | ((M >> 4) << 24);
      // (bit 16: B, the values, is dims-major)
      constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((M >> 4) << 24);
      // bytes between the values' groups of eight positions
      constexpr uint32_t v_group = (uint32_t)(D / 8) * 128 / (PAIR ? 2 : 1);
      const uint32_t qh = kTmem + kColQ, ql = qh + D / 2;
      const uint64_t kd = umma_desc(smem_addr(smem + L::k), 128, 16 * D);
      const uint64_t vd = umma_desc(smem_addr(smem + L::v), v_group, 128);
      constexpr uint64_t plane = L::plane >> 4;
      // step j's scores, once the step before's have been read
      auto scores = [&](int j) {
        const int b = j % L::n_k;
        if (!tc_wait_ready(&k_full[b], (uint32_t)(j / L::n_k) & 1u, abort_flag, p.err)) return false;
        if (j > 0 && !tc_wait_ready(s_empty, (uint32_t)(j - 1) & 1u, abort_flag, p.err)) return false;
        tc_fence_after();
        if (elect_one()) {
          constexpr uint32_t d = kTmem + kColS;
          uint64_t kh = kd + 2 * plane * b;
          asm volatile("" : "+l"(kh));  // (the 24 descriptors are formed here, not kept in registers)
          const uint64_t kl = kh + plane;
#pragma unroll
          for (int s = 0; s < D / 16; s++) mma_ts<PAIR>(d, ql + 8 * s, kh + 16 * s, idesc_s, s > 0);
#pragma unroll
          for (int s = 0; s < D / 16; s++) mma_ts<PAIR>(d, qh + 8 * s, kl + 16 * s, idesc_s, 1);
#pragma unroll
          for (int s = 0; s < D / 16; s++) mma_ts<PAIR>(d, qh + 8 * s, kh + 16 * s, idesc_s, 1);
          mma_commit<PAIR>(s_full);
          mma_commit<PAIR>(&k_empty[b]);
        }
        __syncwarp();
        return true;
      };
      bool ok = rank == 0 && tc_wait_ready(q_full, 0, abort_flag, p.err) && scores(0);
      for (int j = 0; j < n && ok; j++) {
        if (j + 1 < n && !(ok = scores(j + 1))) break;
        const int b = j % L::n_v;
        if (!(ok = tc_wait_ready(&v_full[b], (uint32_t)(j / L::n_v) & 1u, abort_flag, p.err))) break;
        if (!(ok = tc_wait_ready(p_full, (uint32_t)j & 1u, abort_flag, p.err))) break;
        tc_fence_after();
        if (elect_one()) {
          constexpr uint32_t o = kTmem + kColO, p_hi = kTmem + kColP, p_lo = p_hi + kTrTile / 2;
          uint64_t vh = vd + 2 * plane * b;
          asm volatile("" : "+l"(vh));
          const uint64_t vl = vh + plane;
#pragma unroll
          for (int s = 0; s < kTrTile / 16; s++) mma_ts<PAIR>(o, p_lo + 8 * s, vh + (v_group >> 3) * s, idesc_o, s > 0);
#pragma unroll
          for (int s = 0; s < kTrTile / 16; s++) mma_ts<PAIR>(o, p_hi + 8 * s, vl + (v_group >> 3) * s, idesc_o, 1);
#pragma unroll
          for (int s = 0; s < kTrTile / 16; s++) mma_ts<PAIR>(o, p_hi + 8 * s, vh + (v_group >> 3) * s, idesc_o, 1);
          mma_commit<PAIR>(o_full);
          mma_commit<PAIR>(&v_empty[b]);
        }
        __syncwarp();
      }
      // every MMA has finished before TMEM and shared memory are given back
      if (rank == 0 && elect_one()) mma_commit<PAIR>(drain);
      __syncwarp();
      for (uint32_t it = 0; it < kSpinLimit && !__all_sync(0xffffffffu, mbar_try_wait_sleep(drain, 0)); it++) {
      }
    } else if (warp < kTrWarpMma + 3) {
      const int v = warp - kTrWarpMma - 1;  // keys, values
      const void* cache = v ? p.cache_v : p.cache_k;
      if constexpr (Q8) {
        // Two of the other warps of the group ask for the whole range, keys and values,
        // ahead of the converters (whose first read of a line from HBM takes 2 us).
        const int64_t pend = min(n_kv, pos0 + (int64_t)n * kTrTile);
        const uint8_t* src = (const uint8_t*)cache + ((int64_t)kvh * p.n_ctx + pos0) * D;
        for (int64_t o = (int64_t)lane * 4096; o < (pend - pos0) * D; o += 32 * 4096)
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src + o),
                       "r"((uint32_t)min((int64_t)4096, (pend - pos0) * D - o))
                       : "memory");
      } else {
        copy_rows<D, L::n_rows>(p, (const float*)cache, kvh, pos0, n_kv, n, lane, (float*)(smem + L::rows) + v * L::n_rows * kTrChunk * L::pitch,
                                rows_full + v * L::n_rows, rows_empty + v * L::n_rows, abort_flag);
      }
    }
  } else if (warp >= kTrWarpK) {
    // ---------------- keys (warps 16-19) and values (20-23) ----------------
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
    auto convert = [&](auto which) {
      constexpr bool is_v = decltype(which)::value;
      TrConvert r;
      r.pos0 = pos0;
      r.n_kv = n_kv;
      r.kvh = kvh;
      r.n = n;
      r.w = warp & 3;
      r.lane = lane;
      r.rank = rank;
      r.cache = is_v ? p.cache_v : p.cache_k;
      r.planes = smem + (is_v ? L::v : L::k);
      r.empty = is_v ? v_empty : k_empty;
      r.full = lead(is_v ? v_full : k_full);
      r.col_full = col_full;
      r.col = col;
      r.info = info;
      r.abort_flag = abort_flag;
      r.rows = (float*)(smem + L::rows) + is_v * L::n_rows * kTrChunk * L::pitch;
      r.rows_full = rows_full + is_v * L::n_rows;
      r.rows_empty = rows_empty + is_v * L::n_rows;
      r.ends = (int2*)(smem + L::ends) + is_v * 16;
      if constexpr (Q8) convert_q8_0<D, PAIR, is_v, is_v ? L::n_v : L::n_k>(p, r, q_here, is_v && nq > 0);
      else convert_f32<D, PAIR, is_v, is_v ? L::n_v : L::n_k, L::n_rows>(p, r, q_here, is_v && nq > 0);
    };
    if (warp < kTrWarpV) convert(std::false_type{});
    else convert(std::true_type{});
  } else {
    // ---------------- softmax: four threads per row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int quad = warp & 3, part = warp >> 2;
    if (quad < nq) {
      constexpr int NA = D / kTrParts, HT = kTrTile / kTrParts;
      const int lr = quad * 32 + lane, r = r0 + lr, i = min(r, sp.R - 1) / rep;
      const uint32_t base = kTmem + ((uint32_t)(32 * quad) << 16);
      // The row's other parts have come as far: twice before the steps, once in each and
      // twice behind them, also by warps that have given up (so that none waits for another).
      auto meet = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + quad) : "memory"); };
      bool ok = true;
      // the row's query planes into TMEM (this thread's quarter of the dims)
      float rf;  // |scale| * log2(e) * the row's factor
      {
        float x[NA], m = 0.0f;
        bool fine = true;
        // read along the rows (a row a lane would be 32 lines a request), turned where
        // the first values will be: this warp's 32 rows x NA floats
        constexpr int NP = NA / 4;
        float4* turn = (float4*)(smem + L::v) + (part * 4 + quad) * 32 * NP;
        auto place = [](int row, int c) { return row * NP + (NP == 8 || NP == 4 ? c ^ (row & (NP - 1)) : c); };
        float4 got[NP];
#pragma unroll
        for (int u = 0; u < NP; u++) {
          const int e = lane + 32 * u, row = e / NP, c = e - row * NP, rr = min(r0 + quad * 32 + row, sp.R - 1), ti = rr / rep;
          const float* src = p.q + ti * p.q_stride + (int64_t)(kvh * rep + rr - ti * rep) * D + NA * part + 4 * c;
          got[u] = vec_q ? *(const float4*)src : make_float4(src[0], src[1], src[2], src[3]);
        }
#pragma unroll
        for (int u = 0; u < NP; u++) {
          const int e = lane + 32 * u, row = e / NP;
          turn[place(row, e - row * NP)] = got[u];
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < NP; c++) {
          const float4 a = turn[place(lane, c)];
          x[4 * c] = a.x, x[4 * c + 1] = a.y, x[4 * c + 2] = a.z, x[4 * c + 3] = a.w;
        }
#pragma unroll
        for (int k = 0; k < NA; k++) {
          m = fmaxf(m, fabsf(x[k]));
          fine &= fabsf(x[k]) <= 3.402823466e38f;
        }
        float* ex = mxs + lr;
        ex[part * kTrRows] = fine ? m : INFINITY;
        meet();
        m = fmaxf(fmaxf(ex[0], ex[kTrRows]), fmaxf(ex[2 * kTrRows], ex[3 * kTrRows]));
        meet();
        fine = m <= 3.402823466e38f;
        const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 127);
        rf = __fmul_rn(__fmul_rn(fabsf(p.scale), 1.4426950408889634f), pow2f(e - 14));
        ok = tc_wait_ready(t_full, 0, abort_flag, p.err);
        if (ok) {
          tc_fence_after();
          const float f = p.scale < 0.0f ? -pow2f(14 - e) : pow2f(14 - e);
#pragma unroll
          for (int k = 0; k < NA; k += 8) {
            // (a query with an infinity or a NaN becomes NaN: so do its scores)
            uint4 hi = make_uint4(0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u), lo = make_uint4(0, 0, 0, 0);
            if (fine) split8(&x[k], f, hi, lo);
            tmem_st4(base + kColQ + part * (NA / 2) + k / 2, hi);
            tmem_st4(base + kColQ + D / 2 + part * (NA / 2) + k / 2, lo);
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive_one(q_here);
            arrive_lead(q_full0);
          }
        }
      }
      float M = -INFINITY;                   // the row's maximum
      float l = 0.0f;                        // this part's weights (Q8_0: relative to M - 14, F32: to ml)
      float ml = -INFINITY, f_prev = 1.0f;
      float acc[NA];
#pragma unroll
      for (int k = 0; k < NA; k++) acc[k] = 0.0f;
      // step j's O into the registers
      auto take_o = [&](int j, float f) {
        if (!tc_wait_ready(o_full, (uint32_t)j & 1u, abort_flag, p.err)) return false;
        tc_fence_after();
        const float2 f2 = make_float2(f, f);
        float y[NA];
#pragma unroll
        for (int o = 0; o < NA; o += 8) tmem_ld8f(base + kColO + NA * part + o, y + o);
#pragma unroll
        for (int o = 0; o < NA; o += 8) tmem_wait_ld8(y + o);
#pragma unroll
        for (int k = 0; k < NA; k += 2) {
          const float2 a = __ffma2_rn(make_float2(acc[k], acc[k + 1]), f2, make_float2(y[k], y[k + 1]));
          acc[k] = a.x;
          acc[k + 1] = a.y;
        }
        return true;
      };
      for (int j = 0; j < n; j++) {
        const int slot = (j & (kTrSlots - 1)) * 2 + (part >> 1);
        const int64_t pt = pos0 + (int64_t)j * kTrTile + part * HT;
        const float* c = col + slot * 2 * kTrHalf + (part & 1) * HT;
        // (a masked position's weight is 0 whatever its row holds)
        auto finite = [](float e) { return e == e ? e : 0.0f; };
        ok = ok && tc_wait_ready(&col_full[slot], (uint32_t)(j / kTrSlots) & 1u, abort_flag, p.err) &&
             tc_wait_ready(s_full, (uint32_t)j & 1u, abort_flag, p.err);
        if (!ok) {
          meet();
          continue;
        }
        tc_fence_after();
        float x[HT];
        tmem_ld32(base + kColS + part * HT, x);
        tmem_wait_ld(x);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_lead(s_empty0);
        // (two elements an instruction where the hardware has one)
        float2* x2 = (float2*)x;
        const float4 in = *(const float4*)(info + slot * 4);
        const bool own = in.y != 0.0f || in.w != 0.0f;  // the positions have exponents of their own
        // score + exponent = x * fac + off; the factor stays above 0, so that a masked -inf does, and
        // finite, so that a product of 0 stays 0
        auto factor = [](float f) { return fminf(fmaxf(f, 1e-37f), 3.4e38f); };
        float fac = factor(__fmul_rn(in.x, rf)), off = in.z;
        if (own) {
          const float kc = in.y != 0.0f ? 0.0f : in.x, vc = in.z;
#pragma unroll
          for (int k = 0; k < HT; k++) {
            const float kf = in.y != 0.0f ? c[k] : kc, ve = in.w != 0.0f ? c[kTrHalf + k] : vc;
            x[k] = __fmaf_rn(x[k], kf == kf ? factor(__fmul_rn(kf, rf)) : kf, ve);
          }
          fac = 1.0f;
          off = 0.0f;
        }
        if (pt + HT > p.n_past) {
          const uint32_t m = attended32(p, i, pt, n_kv);
#pragma unroll
          for (int k = 0; k < HT; k++)
            if (!((m >> k) & 1u)) x[k] = -INFINITY;
        }
        float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int k = 4; k < HT; k += 8)
#pragma unroll
          for (int u = 0; u < 4; u++) mx[u] = k + 4 < HT ? fmaxf(fmaxf(mx[u], x[k + u]), x[k + 4 + u]) : fmaxf(mx[u], x[k + u]);
        mx[0] = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        // The references are whole numbers not below the maximum, so that their
        // differences and those with the exponents are exact (NaN where there is
        // nothing else: as if nothing were attended, the weights bring it back).
        mx[0] = mx[0] == mx[0] ? ceilf(__fmaf_ru(mx[0], fac, off)) : -INFINITY;
        // the row's maximum over its parts
        float* ex = mxs + (j & 1) * kTrParts * kTrRows + lr;
        ex[part * kTrRows] = mx[0];
        meet();
        const float Mn = fmaxf(fmaxf(fmaxf(M, ex[0]), fmaxf(ex[kTrRows], ex[2 * kTrRows])), ex[3 * kTrRows]);
        // (2^14: the largest weight that fp16 still holds with room; rounded up, and
        // the sum below down, so that no score of any size gets past it)
        const float Mr = Mn == -INFINITY ? 0.0f : Mn, Ms = __fsub_ru(Mr, 14.0f);
        const float f = exp2_approx(__fsub_rn(M, Mr));
        M = Mn;
        float lr0 = Ms;  // what the weights' sum is relative to
        if (Q8) {
          l = __fmul_rn(l, f);
        } else {
          // the values' exponents reach over all of a float's range: the sum has a
          // reference of its own, the largest score of this part without them
          float ms = -INFINITY;
          if (own) {
#pragma unroll
            for (int k = 0; k < HT; k++) ms = fmaxf(ms, __fsub_rn(x[k], in.w != 0.0f ? finite(c[kTrHalf + k]) : in.z));
            ms = ceilf(ms);
          } else {
            ms = __fsub_rn(mx[0], in.z);
          }
          if (ms > ml) {
            l = __fmul_rn(l, exp2_approx(__fsub_rn(ml, ms)));
            ml = ms;
          }
          lr0 = ml == -INFINITY ? 0.0f : ml;
        }
        // the factor that takes a value exponent out of a weight and brings it to lr0
        const float ls = __fsub_rn(Ms, lr0), lf = __fsub_rn(ls, in.z);
        const bool apart = own || lf > 100.0f;  // (above: weights that count may be below a float's range)
        if (apart) {
#pragma unroll
          for (int k = 0; k < HT; k++) {
            const float ve = in.w != 0.0f ? finite(c[kTrHalf + k]) : in.z, g = __fsub_rn(ls, ve);
            const float s = own ? x[k] : __fmaf_rn(x[k], fac, off);
            l = g > 100.0f ? __fadd_rn(l, exp2_approx(__fsub_rn(__fsub_rn(s, ve), lr0)))
                           : __fmaf_rn(exp2_approx(__fsub_rn(s, Ms)), exp2_approx(g), l);
          }
        }
        const float2 fac2 = make_float2(fac, fac), off2 = make_float2(__fsub_rd(off, Ms), __fsub_rd(off, Ms));
        const float2 minus = make_float2(-1.0f, -1.0f);
        float2 sum = make_float2(0.0f, 0.0f);
        uint32_t hi[HT / 2], lo[HT / 2];
#pragma unroll
        for (int k = 0; k < HT / 2; k++) {
          const float2 d = __ffma2_rn(x2[k], fac2, off2);
          const float2 pe = make_float2(exp2_approx(d.x), exp2_approx(d.y));
          sum = __fadd2_rn(sum, pe);
          // the upper half by cutting to fp16's 11 bits (below 2^-14, a weight of
          // 2^-28 of the row's largest, its conversion rounds instead)
          const float2 top = make_float2(__uint_as_float(__float_as_uint(pe.x) & 0xffffe000u),
                                         __uint_as_float(__float_as_uint(pe.y) & 0xffffe000u));
          const float2 rest = __ffma2_rn(top, minus, pe);
          hi[k] = h2_bits(__floats2half2_rn(top.x, top.y));
          lo[k] = h2_bits(__floats2half2_rn(rest.x, rest.y));
        }
        if (!apart) l = __fmaf_rn(__fadd_rn(sum.x, sum.y), exp2_approx(lf), l);
        // the step before's O; with it P's columns are free
        if (j > 0) ok = take_o(j - 1, f_prev);
        f_prev = f;
        tmem_st16(base + kColP + part * (HT / 2), hi);
        tmem_st16(base + kColP + kTrTile / 2 + part * (HT / 2), lo);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_lead(p_full0);
      }
      if (ok) ok = take_o(n - 1, f_prev);
      // the parts' sums
      float m = M == -INFINITY ? -INFINITY : __fsub_ru(M, 14.0f);  // what l is relative to
      float* ex = mxs + (n & 1) * kTrParts * kTrRows + lr;  // (not the last step's)
      ex[part * kTrRows] = ml;
      meet();
      if (!Q8) {
        m = fmaxf(fmaxf(ex[0], ex[kTrRows]), fmaxf(ex[2 * kTrRows], ex[3 * kTrRows]));
        if (ml != -INFINITY) l = __fmul_rn(l, exp2_approx(__fsub_rn(ml, m)));
      }
      ex = mxs + ((n + 1) & 1) * kTrParts * kTrRows + lr;
      ex[part * kTrRows] = l;
      meet();
      l = __fadd_rn(__fadd_rn(ex[0], ex[kTrRows]), __fadd_rn(ex[2 * kTrRows], ex[3 * kTrRows]));
      // The rows into shared memory (every product that read the planes there is done:
      // O has been taken), as records or, with one split, as results; a token that
      // attends to nothing has l = 0.
      const float Ms = M == -INFINITY ? -INFINITY : __fsub_ru(M, 14.0f);
      float* rec = (float*)(smem + L::k) + lr * (D + 4);
      if (sp.S == 1) {
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l), down = Ms == -INFINITY ? 0.0f : __fsub_rn(Ms, m);
#pragma unroll
        for (int k = 0; k < NA; k++) {
          acc[k] = __fmul_rn(acc[k], inv);
          if (!Q8) acc[k] = times_pow2(acc[k], down);  // (Q8_0: 0)
        }
      }
      if (ok) {
        if (part == 0) *(float4*)rec = make_float4(Ms, m, l, 0.0f);
#pragma unroll
        for (int k = 0; k < NA; k += 4)
          *(float4*)(rec + 4 + NA * part + k) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
      }
    }
  }
  tc_fence_before();
  if (PAIR) cluster_sync_all();  // (neither CTA leaves, or gives up its TMEM, before the other has finished)
  else __syncthreads();
  if (*abort_flag == 0) {
    // out of it in rows: the records of a CTA's rows are contiguous
    const int rows = min(kTrRows, sp.R - r0);
    const float* rec = (const float*)(smem + L::k);
    if (sp.S == 1) {
      for (int e = tid; e < rows * (D / 4); e += kTrThreads) {
        const int lr = e / (D / 4), d = (e - lr * (D / 4)) * 4, r = r0 + lr, i = r / rep;
        const float4 v = *(const float4*)(rec + lr * (D + 4) + 4 + d);
        float* out = p.out + ((int64_t)i * p.H + kvh * rep + (r - i * rep)) * D + d;
        out[0] = v.x, out[1] = v.y, out[2] = v.z, out[3] = v.w;
      }
    } else {
      float4* dst = (float4*)((float*)p.scratch + (((int64_t)kvh * sp.S + split) * sp.R + r0) * (D + 4));
      for (int e = tid; e < rows * (D / 4 + 1); e += kTrThreads) dst[e] = ((const float4*)rec)[e];
    }
  }
  if (warp == kTrWarpMma) {
    __syncwarp();
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(*tmem_base), "r"(kTrCols));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_base), "r"(kTrCols));
  }
}

// Splits of a KV head's positions: one CTA (or pair) per SM (or two).
int64_t most_splits(int64_t H, int64_t HKV, int64_t n_kv, int64_t T) {
  const int64_t RG = (T * (H / HKV) + kTrRows - 1) / kTrRows, steps = (n_kv + kTrTile - 1) / kTrTile;
  const int64_t ctas = RG == 1 ? 1 : (RG + 1) / 2 * 2;
  return std::min(steps, std::max<int64_t>(1, kTrSms / std::max<int64_t>(1, HKV * ctas)));
}

template <int D, bool Q8, bool PAIR>
cudaError_t launch_tiles(const TreeAttnParams& p, const TreeSplit& sp, cudaStream_t s) {
  const int vec_q = (uintptr_t)p.q % 16 == 0 && p.q_stride % 4 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(PAIR ? (sp.RG + 1) / 2 * 2 : sp.RG), (unsigned)p.HKV, (unsigned)sp.S);
  cfg.blockDim = dim3(kTrThreads);
  cfg.dynamicSmemBytes = TrSmem<D, Q8, PAIR>::total;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : 1;  // (a pair lies along x: along z the launch is refused)
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn_tree_kernel<D, Q8, PAIR>, p, sp, vec_q);
}

template <int D, bool Q8>
cudaError_t launch_tree(const TreeAttnParams& p, cudaStream_t s) {
  TreeSplit sp{};
  sp.R = p.T * (p.H / p.HKV);
  sp.RG = (sp.R + kTrRows - 1) / kTrRows;
  const int64_t n_kv = (int64_t)p.n_past + p.T, steps = (n_kv + kTrTile - 1) / kTrTile;
  const int64_t most = most_splits(p.H, p.HKV, n_kv, p.T);
  sp.per = (int32_t)((steps + most - 1) / most);
  sp.S = (int32_t)((steps + sp.per - 1) / sp.per);
  const cudaError_t e = sp.RG == 1 ? launch_tiles<D, Q8, false>(p, sp, s) : launch_tiles<D, Q8, true>(p, sp, s);
  if (e != cudaSuccess || sp.S == 1) return e;
  return launch_tree_join<D>(p, sp, s);
}

template <int D, bool Q8, bool PAIR>
cudaError_t prepare_tiles() {
  // A build that gave the kernel fewer registers than its roles share out would wait
  // for them for good.
  cudaFuncAttributes a;
  const cudaError_t e = cudaFuncGetAttributes(&a, attn_tree_kernel<D, Q8, PAIR>);
  if (e != cudaSuccess) return e;
  if (a.numRegs * kTrThreads < kRegsSoftmax * 512 + kRegsConvert * 256 + kRegsMma * 128) return cudaErrorInvalidConfiguration;
  return cudaFuncSetAttribute(attn_tree_kernel<D, Q8, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, TrSmem<D, Q8, PAIR>::total);
}
template <int D>
cudaError_t prepare_tree() {
  cudaError_t e = prepare_tiles<D, false, false>();
  if (e == cudaSuccess) e = prepare_tiles<D, false, true>();
  if (e == cudaSuccess) e = prepare_tiles<D, true, false>();
  return e == cudaSuccess ? prepare_tiles<D, true, true>() : e;
}

}  // namespace

bool attn_tree_fits(int64_t D, int64_t H, int64_t HKV, int64_t T) {
  return (D == 32 || D == 64 || D == 96 || D == 128) && H > 0 && HKV > 0 && H % HKV == 0 && H <= 4096 && T >= 0 &&
         T <= kTreeMaxTokens;
}

// Records of all splits, for up to n_kv rows and T tokens: a KV head's groups of
// 128 rows times its splits pass kTrSms / HKV only where one group alone does.
size_t attn_tree_scratch_bytes(int64_t H, int64_t HKV, int64_t n_kv, int64_t T, int64_t D) {
  const int64_t R = T * (H / HKV), steps = (n_kv + kTrTile - 1) / kTrTile;
  const int64_t rows = std::min(steps * R, std::max(R, (kTrSms + HKV - 1) / HKV * kTrRows));
  return (size_t)(16 + HKV * rows * (D + 4) * 4);
}

cudaError_t prepare_attn_tree_kernels() {
  cudaError_t e = prepare_tree<32>();
  if (e == cudaSuccess) e = prepare_tree<64>();
  if (e == cudaSuccess) e = prepare_tree<96>();
  if (e == cudaSuccess) e = prepare_tree<128>();
  return e;
}

// Whether attn_few.cu is the faster one for R rows of a KV head. Q8_0: up to 8 rows it
// always is (one token, us there / here: 5.2 / 10.0 at 500 positions, 11.5 / 18.1 at
// 32000 with 14 / 2 heads of 64, 24.4 / 42.5 with 28 / 4 heads of 128); each further
// 16 rows are another pass over the cache there, which 14 rows repay up to some
// 16000 positions (heads of 128 16.9 / 19.1 at 8000, 52 / 42 at 32000; of 64 11.4 / 14.4 at
// 16000, 20.3 / 18.2 at 32000) and 28 up to some 8000 of 64 dims (11.2 / 12.2 at 8000, 19.7 /
// 14.3 at 16000; heads of 128 10.5 / 13.3 at 500, 14.9 / 13.9 at 2000, 21.2 / 19.3 at 8000).
//
// Over an F32 cache: up to 8 rows always (14 / 2 heads of 64: 7.6 / 13.2 at 2000
// positions, 21 / 25 at 32000), up to 16 nearly always (14 rows 12.0 / 14.3 at 8000; 12
// of 96 dims 34 / 41 at 32000) but at 128 dims, where they no longer fit the registers
// (14 rows 13.2 / 17.5 at 500, 19.5 / 16.1 at 2000), and with more passes of 16 rows
// while the cache is small (63 rows of 64 over 2000 11.8 / 13.5, 91 rows 20.2 / 13.7).
static bool few_rows(bool q8, int64_t R, int64_t n_kv, int64_t HKV, int64_t D) {
  if (q8) return R <= 8 || (R <= 16 && n_kv <= 16384) || (R <= 32 && n_kv * D <= (1 << 19));
  const int64_t most = D > 96 ? 1 << 19 : R <= 16 ? 1 << 23 : R <= 64 ? 1 << 20 : 1 << 19;
  return R <= 8 || (R <= 128 && (R + 15) / 16 * n_kv * HKV * D <= most);
}

cudaError_t launch_attn_tree(const TreeAttnParams& p, cudaStream_t s) {
  if (p.T == 0) return cudaSuccess;
  if (few_rows(p.q8, (int64_t)p.T * (p.H / p.HKV), (int64_t)p.n_past + p.T, p.HKV, p.D)) return launch_attn_few(p, s);
  switch (p.D) {
    case 32: return p.q8 ? launch_tree<32, true>(p, s) : launch_tree<32, false>(p, s);
    case 64: return p.q8 ? launch_tree<64, true>(p, s) : launch_tree<64, false>(p, s);
    case 96: return p.q8 ? launch_tree<96, true>(p, s) : launch_tree<96, false>(p, s);
    case 128: return p.q8 ? launch_tree<128, true>(p, s) : launch_tree<128, false>(p, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace mi
