// Matrix products of the loss over a vocabulary (sa_loss.cu): D = A B^T with 16-bit operands and fp32 sums, a persistent kernel
// with four epilogues.  A CTA, or the two CTAs of a cluster on one tile (CTAS = 2), own 128 rows each of a tile of up to
// 128 * CTAS columns; TMA fills a ring of stages 64 deep, one thread issues the MMAs, and two accumulators in tensor memory let
// the epilogue of a tile run under the products of the next.
//
// Either operand may stand with the contraction contiguous ("K-major": rows of x or W) or with its own index contiguous
// ("MN-major": W, x and the probabilities as the gradients' products read them), so nothing is transposed in memory.
// fp32 operands come as three bf16 parts of 8 bits each, x = hi + mid + lo, and a product is the six products of parts that reach
// 2^-16 of it or more, smallest first: six times the work of a bf16 product.
#pragma once

#include <type_traits>

#include "sa_tc_ptx.cuh"

namespace sa {
namespace product {

using namespace tc;

constexpr int kRows = 128;                 // of a CTA
constexpr int kDepth = 64;                 // of a stage: 128 bytes of a 16-bit operand
constexpr int kOperand = kRows * kDepth * 2;
constexpr int kStages = 6;
constexpr int kThreads = 384;              // warp 0 loads, warp 1 issues, warp 2 has the tensor memory, warps 4 to 11 read it
constexpr int kEpilogueWarps = 8;
constexpr size_t kSmem = (size_t)kStages * 2 * kOperand + 1024;
constexpr int kTurnPitch = 33;               // words of 32 columns that a warp turns
constexpr size_t kSmemResult = kSmem + (size_t)kEpilogueWarps * 32 * kTurnPitch * 4;
constexpr int kTerms = 6;                  // of an fp32 product
// The tensor cores' additions round towards zero: 2^-23.4 a group of 16 products of what is summed, all one way, so a long sum loses in
// proportion to its length (logits of a width of 4,096: 2.8e-6 of the loss; the mean of 50,304 rows of a table: 2.9e-4 of it).  So an
// epilogue adds the sums of a few stages at a time in its registers, with rounding to nearest: of fp32 operands of 256 of the contraction
// (1.5e-7 of the loss); of 16-bit ones of 512 in logits, up to a width of 1,024 of all (3e-7, 6.9e-7), and of 8,192 in gradients, which are
// rounded to 16 bits themselves.
constexpr int kSegment = 4, kSegmentLogits = 8, kUncutLogits = 16, kSegmentResult = 128;
constexpr int kSegmentChunks = 4;          // chunks of 32 columns of a tile that a thread of an epilogue has, at most

// The work of a launch: tiles of rows x columns, each a walk over `blocks` stages of the contraction.  The first `whole` tiles are
// walked by one cluster each, round by round.  Of what is left, less than half a round, every tile is cut into `slabs` equal parts of
// the contraction with a cluster and a sum (a slab) each; the parts of all tiles at one depth are walked side by side, so what tiles
// share is still read once.
struct Walk {
  int m, n;                                // rows and columns of the result
  int bn;                                  // columns of a tile, a multiple of 32
  int m_tiles, n_tiles, whole;
  int depth_blocks, blocks;                // stages of one term, of all terms
  int clusters;
  int slabs;                               // of a cut tile
  int segment;                             // stages that are summed in tensor memory at a time, `blocks` without SEGMENTS
  int group;                               // row tiles that are walked side by side
  __host__ __device__ int tiles() const { return m_tiles * n_tiles; }
  __host__ __device__ void place(int tile, int* tm, int* tn) const {
    const int per = group * n_tiles, g = tile / per, r = tile - g * per;
    const int rows = m_tiles - g * group < group ? m_tiles - g * group : group;
    *tn = r / rows;
    *tm = g * group + (r - *tn * rows);
  }
  __host__ __device__ int columns(int tn) const {                 // of a tile, in 32s
    const int left = (n - tn * bn + 31) / 32 * 32;
    return left < bn ? left : bn;
  }
};

// A cluster's walk, the same in every role of its CTAs: units of at most `segment` stages.
struct Units {
  int at, k, share1;                       // the next item: a whole tile, or a part of one behind them
  int tile, tm, tn, k0, k1, slab;
  bool last;                               // of this cluster's sums of the tile
  __host__ __device__ void begin(int c) {
    at = c;
    k = share1 = 0;
  }
  __host__ __device__ bool next(const Walk& w) {
    while (k >= share1) {
      const int left = w.tiles() - w.whole;
      if (at >= w.whole + left * w.slabs) return false;
      tile = at;
      slab = 0;
      k = 0;
      share1 = w.blocks;
      if (at >= w.whole && w.slabs > 1) {
        slab = (at - w.whole) / left;
        tile = at - slab * left;
        k = (int)((int64_t)w.blocks * slab / w.slabs);
        share1 = (int)((int64_t)w.blocks * (slab + 1) / w.slabs);
      }
      at += w.clusters;
      w.place(tile, &tm, &tn);
    }
    k0 = k;
    k1 = k = k + w.segment < share1 ? k + w.segment : share1;
    last = k == share1;
    return true;
  }
};

// Where an operand's tiles start: offsets of its own index and of the contraction, in elements.
struct Origin {
  int own, depth;
};

// SEGMENTS of the kernel: sums leave tensor memory every `segment` stages, of which every tile has several.
enum Kind { kStats, kProbabilities, kBoth, kResult };

struct Epilogue {
  // kStats: of every row and half tile, the maximum and the sum of exponentials above it (see base_of); the targets' logits
  float2* stats;                           // [2 * n_tiles][m]
  float* at_target;                        // [m]
  float* e_target;                         // kBoth: [m], the exponential
  const int64_t* targets;
  int column0;                             // of the vocabulary, that the launch's first column is
  unsigned int* zeroed;                    // kStats: a counter to be cleared for the kernel behind
  // kBoth: exp(z - ref) (see base_of) in `parts` parts, with their sum (and the maximum of z) in the place of the others'; 0 where
  // ref is +inf
  const float* ref;
  const int* only;                         // rows that are not marked stay as they are; null: all are meant
  const int* any;                          // nothing is done where this is 0; null: it is done
  // kProbabilities: (exp2((z - lse.x) log2 e - lse.y) - [target]) * factor, in `parts` 16-bit parts
  const float2* lse;
  const float* factor;
  float* less;                             // of one or two parts: [m], what the first one's rounding takes from the target's column, times `scale`
  uint16_t* p;
  int64_t p_pitch, p_part;                 // elements of a row, of a part
  int parts;
  int half;                                // fp16, not bf16
  // kResult: of whole tiles (sums + addend) * scale + table_factor * [a row of `table`]; cut tiles keep their sums in slabs of a tile each
  void* out;
  int dtype;
  int64_t out_pitch;
  int aligned;                             // its rows start where whole vectors are stored: set with the launch
  const float* addend;                     // fp32, may be null
  int64_t addend_pitch;
  int cut_addend;                          // cut tiles have it too; otherwise what is added to them stands in their slabs
  int addend_first;                        // its rows start at 32 bytes; others have no scale and no table beside them.  Set with the launch
  const float* scale;                      // may be null
  int scale_rows;                          // one for every row
  float* slabs;
  int later;                               // cut tiles add to what their slabs hold
  const void* table;                       // whose rows that `targets` names are added, `table_factor` times; may be null
  int table_dtype;
  int64_t table_stride;
  const float* table_factor;               // of a row of the result
  int vocab;
};

// ---- PTX of CTA pairs ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t address_in(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Relaxed: what it tells of are loads from tensor memory whose values are there.  A release to the cluster would also wait for the warp's
// stores to global memory.
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  if constexpr (CTAS == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
template <int CTAS>
__device__ __forceinline__ void mma(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "n"(kDescHigh)
        : "memory");
}
// Arrives on the barrier at this offset in every CTA of the tile once the MMAs issued so far are complete.
template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3)
                 : "memory");
  else
    mma_commit(bar);
}
template <int CTAS>
__device__ __forceinline__ void tensor_memory_alloc(uint32_t* dst, uint32_t cols) {
  if constexpr (CTAS == 2) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, cols);
  }
}
template <int CTAS>
__device__ __forceinline__ void tensor_memory_free(uint32_t addr, uint32_t cols) {
  if constexpr (CTAS == 2) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
  } else {
    tmem_dealloc(addr, cols);
  }
}
// 32 bytes a thread: a whole sector of memory.
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// The same of what is not read again before much else has been written: it leaves L2 first.
__device__ __forceinline__ void store32_once(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.L1::no_allocate.L2::evict_first.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void load32(const void* p, uint32_t (&v)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Waits for the loads from tensor memory; the values are there behind it, for the compiler too.
__device__ __forceinline__ void tmem_loaded(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// ---- epilogues: 32 columns of a row in registers ----------------------------------------------------------------------------------

// Two values in a register pair: one instruction for both.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float lo, float hi) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 both(Pair x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float most_of(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The largest of 32 columns and of `than`, by four chains.
__device__ __forceinline__ float most_of(const uint32_t (&r)[32], float than) {
  float m[4] = {than, __uint_as_float(r[1]), __uint_as_float(r[2]), __uint_as_float(r[3])};
  m[0] = fmaxf(m[0], __uint_as_float(r[0]));
#pragma unroll
  for (int i = 4; i < 32; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      m[k] = i + 4 + k < 32 ? most_of(m[k], __uint_as_float(r[i + k]), __uint_as_float(r[i + 4 + k])) : fmaxf(m[k], __uint_as_float(r[i + k]));
  return fmaxf(most_of(m[0], m[1], m[2]), m[3]);
}
// Exponentials of logits relative to another one, exp(z - top), are exp2(z log2 e - base) for the base of `top`: top * log2 e, rounded once
// and taken from the exact product, so that only what the base is relative to moves (a rounded z log2 e of 100 would move its exponential
// by 2^-18).  The rounding is up to 8 where |top| is kHuge, far less than an exponential can bear, and anything beyond, where logits
// mask words or stand for nothing else that is useful: there the difference comes first and the base is `top` itself.  (That by a branch of
// 32 columns: the forward of 4,736 tokens of 56,832 words 129 -> 132 us at a width of 64, 179 -> 184 at 512; by a vote of the warp 143, 188.)
constexpr float kHuge = 134217728.f;                        // 2^27
__device__ __forceinline__ bool is_huge(float top) { return fabsf(top) >= kHuge; }
__device__ __forceinline__ float base_of(float top) { return __fmul_rn(top, kLog2e); }
// log2 of exponentials that are relative to the base of `top`, were they relative to that of `other`.
__device__ __forceinline__ float between(float top, float other) {
  return is_huge(top) || is_huge(other) ? (top - other) * kLog2e : base_of(top) - base_of(other);
}
// log2 of a sum relative to the base of `top`, above top itself.
__device__ __forceinline__ float log2_above(float sum, float top) {
  return log2f(sum) - (is_huge(top) ? 0.f : __fmaf_rn(top, kLog2e, -base_of(top)));
}
// Of 32 columns, and their sum: relative to the base `from`, or with HUGE to the logit `from`.
template <bool HUGE>
__device__ __forceinline__ float exponentials(const uint32_t (&r)[32], float from, float (&p)[32]) {
  const Pair by = pair(kLog2e, kLog2e), less = pair(-from, -from);
  Pair sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const Pair z = pair(__uint_as_float(r[i]), __uint_as_float(r[i + 1]));
    const float2 x = both(HUGE ? fma2(add2(z, less), by, pair(0.f, 0.f)) : fma2(z, by, less));
    p[i] = ex2(x.x);
    p[i + 1] = ex2(x.y);
    sums[(i >> 1) & 1] = add2(sums[(i >> 1) & 1], pair(p[i], p[i + 1]));
  }
  const float2 a = both(sums[0]), b = both(sums[1]);
  return (a.x + a.y) + (b.x + b.y);
}
__device__ __forceinline__ float exponential(float z, float top) {           // one, as it stands in the sum
  return ex2(is_huge(top) ? (z - top) * kLog2e : __fmaf_rn(z, kLog2e, -base_of(top)));
}

// Running maximum and sum of exponentials above it.
struct RowStats {
  float top = -INFINITY, base = -INFINITY, sum = 0.f;       // base: of top
  __device__ __forceinline__ void add(uint32_t (&r)[32], int valid) {
    if (valid < 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = i < valid ? r[i] : __float_as_uint(-INFINITY);
    }
    const float best = most_of(r, top), to = base_of(best);
    float p[32];
    if (__builtin_expect(!is_huge(best), 1)) {
      sum = sum * ex2(base - to) + exponentials<false>(r, to, p);
    } else if (best != -INFINITY) {
      sum = (top == -INFINITY ? 0.f : sum * ex2((top - best) * kLog2e)) + exponentials<true>(r, best, p);
    }
    top = best;
    base = to;
  }
  __device__ __forceinline__ float2 result() const { return make_float2(top, sum); }
};

// 32 columns rounded to the parts; exactly nothing of a token that does not count, whatever they are.
__device__ __forceinline__ void store_parts(const Epilogue& e, float (&p)[32], bool counts, int64_t at) {
  for (int part = 0; part < e.parts; ++part) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = e.half ? pack_half(p[2 * i], p[2 * i + 1]) : pack_bf16(p[2 * i], p[2 * i + 1]);
    uint16_t* dst = e.p + part * e.p_part + at;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = counts ? w[8 * h + i] : 0u;
      store32_once(dst + 16 * h, v);
    }
    if (part + 1 < e.parts) {                                                // what is left for the next part: exact
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 kept = e.half ? __half22float2(*reinterpret_cast<const __half2*>(&w[i]))
                                   : make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
        p[2 * i] -= kept.x;
        p[2 * i + 1] -= kept.y;
      }
    }
  }
}

__device__ __forceinline__ float select(const uint32_t (&r)[32], int i) {
  float v = 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) v = j == i ? __uint_as_float(r[j]) : v;
  return v;
}

// (exp2((z - lse.x) log2 e - lse.y) - [target]) * factor of 32 columns, rounded to the parts.
__device__ __forceinline__ void store_probabilities(const Epilogue& e, const uint32_t (&r)[32], int row, int64_t at, float2 lse, float factor,
                                                    int target) {
  const Pair by = pair(kLog2e, kLog2e), top = pair(-lse.x, -lse.x), rest = pair(-lse.y, -lse.y);
  float p[32];
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const float2 x = both(fma2(add2(pair(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), top), by, rest));
    p[i] = ex2(x.x);
    p[i + 1] = ex2(x.y);
  }
  if (target >= 0) {
#pragma unroll
    for (int i = 0; i < 32; ++i) p[i] = i == target ? p[i] - 1.f : p[i];
    if (e.parts < 3 && factor != 0.f) {                                      // the largest column by far, most often
      float d = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) d = i == target ? p[i] * factor : d;
      e.less[row] = (d - (e.half ? __half2float(__float2half_rn(d)) : __bfloat162float(__float2bfloat16_rn(d)))) * (e.scale != nullptr ? *e.scale : 1.f);
    }
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) p[i] *= factor;
  store_parts(e, p, factor != 0.f, at);
}

// 32 columns of a row in fp32, `valid` of them inside.
__device__ __forceinline__ void add_row(const float* p, uint32_t (&r)[32], int valid) {
  if (valid >= 32 && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      uint32_t v[8];
      load32(p + 8 * h, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[8 * h + i] = __float_as_uint(__uint_as_float(r[8 * h + i]) + __uint_as_float(v[i]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < valid) r[i] = __float_as_uint(__uint_as_float(r[i]) + p[i]);
  }
}
__device__ __forceinline__ void store_row(float* p, const uint32_t (&r)[32], int valid) {
  if (valid >= 32 && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r[8 * h + i];
      store32(p + 8 * h, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < valid) p[i] = __uint_as_float(r[i]);
  }
}
__device__ __forceinline__ void store_row(uint16_t* p, const uint32_t (&r)[32], int valid, bool half) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    w[i] = half ? pack_half(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])) : pack_bf16(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
  if (valid >= 32 && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = w[8 * h + i];
      store32(p + 16 * h, v);
    }
  } else if (valid >= 32 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int h = 0; h < 4; ++h) reinterpret_cast<uint4*>(p)[h] = make_uint4(w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < valid) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  }
}

// Eight values of a row of any type from column `col` on, zeros behind the width.
__device__ __forceinline__ void load_columns(const void* base, int dtype, int64_t row_at, int col, int width, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  const int64_t at = row_at + col;
  const char* src = static_cast<const char*>(base) + at * (dtype == SA_F32 ? 4 : 2);
  if (col + 8 <= width && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    if (dtype == SA_F32) {
      const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      return;
    }
    const uint4 a = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (dtype == SA_BF16) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (col + i < width) {
      if (dtype == SA_F32) v[i] = static_cast<const float*>(base)[at + i];
      else if (dtype == SA_BF16) v[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at + i]);
      else v[i] = __half2float(static_cast<const __half*>(base)[at + i]);
    }
}

// Stores 32 columns of a warp's `rows` rows, `valid` of them inside, where rows start anywhere: turned in shared memory, so that a store runs
// along a row (two tokens' gradient of 93,968 words of 2,926, in bf16: 352 us, a row a thread 2,140).
template <typename T>
__device__ __forceinline__ void store_across(T* out, int64_t pitch, const float* addend, int64_t addend_pitch, const uint32_t (&r)[32], int rows,
                                             int valid, int lane, float* turn) {
  constexpr int kBatch = 8;                // rows whose values and addends are in flight
#pragma unroll
  for (int j = 0; j < 32; ++j) turn[lane * kTurnPitch + j] = __uint_as_float(r[j]);
  __syncwarp();
  if (lane < valid) {
    out += lane;
    for (int i0 = 0; i0 < rows; i0 += kBatch) {
      float v[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) v[k] = turn[(i0 + k) * kTurnPitch + lane];
      if (addend != nullptr) {
        float also[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) also[k] = i0 + k < rows ? addend[(i0 + k) * addend_pitch + lane] : 0.f;
#pragma unroll
        for (int k = 0; k < kBatch; ++k) v[k] += also[k];
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (i0 + k < rows) {
          if constexpr (sizeof(T) == 4) *out = v[k];
          else if constexpr (std::is_same<T, __half>::value) *out = __float2half_rn(v[k]);
          else *out = __float2bfloat16_rn(v[k]);
        }
        out += pitch;
      }
    }
  }
  __syncwarp();
}

// 32 columns of a warp's 32 rows of the result, or of a slab; a thread's row is `row0` and its lane.  Rows that start anywhere go across.
__device__ __forceinline__ void store_result(const Epilogue& e, const Walk& w, const Units& u, uint32_t (&r)[32], int row0, int lane, int in_tile,
                                             int tile_rows, int chunk, float* turn) {
  const int col = u.tn * w.bn + chunk * 32, valid = w.n - col, row = row0 + lane;
  const bool across = !e.aligned && u.tile < w.whole, inside = row < w.m;
  if (valid <= 0 || row0 >= w.m || (!inside && !across)) return;
  if (u.tile >= w.whole) {
    float* const slab = e.slabs + (((int64_t)(u.tile - w.whole) * w.slabs + u.slab) * tile_rows + in_tile) * w.bn + chunk * 32;
    if (e.later) add_row(slab, r, 32);
    store_row(slab, r, 32);
    return;
  }
  if (inside) {
    if (e.addend != nullptr && (!across || e.addend_first)) add_row(e.addend + (int64_t)row * e.addend_pitch + col, r, valid);
    if (e.scale != nullptr) {
      const float scale = e.scale[e.scale_rows ? row : 0];
#pragma unroll
      for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * scale);
    }
    if (e.table != nullptr && e.table_factor[row] != 0.f) {
      const int64_t t = e.targets[row];
      const float factor = e.table_factor[row];
      if (t >= 0 && t < e.vocab) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v[8];
          load_columns(e.table, e.table_dtype, t * e.table_stride, col + 8 * k, w.n, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) r[8 * k + j] = __float_as_uint(fmaf(factor, v[j], __uint_as_float(r[8 * k + j])));
        }
      }
    }
  }
  if (!across) {
    const int64_t at = (int64_t)row * e.out_pitch + col;
    if (e.dtype == SA_F32) store_row(static_cast<float*>(e.out) + at, r, valid);
    else store_row(static_cast<uint16_t*>(e.out) + at, r, valid, e.dtype == SA_F16);
    return;
  }
  const int64_t at = (int64_t)row0 * e.out_pitch + col;
  const float* const addend = e.addend != nullptr && !e.addend_first ? e.addend + (int64_t)row0 * e.addend_pitch + col : nullptr;
  const int rows = min(32, w.m - row0);
  if (e.dtype == SA_F32) store_across(static_cast<float*>(e.out) + at, e.out_pitch, addend, e.addend_pitch, r, rows, valid, lane, turn);
  else if (e.dtype == SA_BF16) store_across(static_cast<__nv_bfloat16*>(e.out) + at, e.out_pitch, addend, e.addend_pitch, r, rows, valid, lane, turn);
  else store_across(static_cast<__half*>(e.out) + at, e.out_pitch, addend, e.addend_pitch, r, rows, valid, lane, turn);
}

// ---- the kernel ---------------------------------------------------------------------------------------------------------------

// `a_bytes`: of the left operand in a stage, less than a whole one where its box has fewer rows; what stands in the others' place makes
// rows of the tile that nothing reads.
template <int CTAS, Kind KIND, bool A_MN, bool B_MN, bool SEGMENTS>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Walk w, const Origin at_a,
               const Origin at_b, const int a_bytes, const Epilogue e, const WaitCtx status) {
  constexpr int kColumns = kRows * CTAS;                            // of an accumulator
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * kStages + 4];
  __shared__ uint32_t tmem_base_s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 ? cluster_rank() : 0u;
  const int c = blockIdx.x / CTAS;
  const uint32_t full = smem_u32(bars), empty = full + 8 * kStages, done = empty + 8 * kStages, read = done + 16;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kStages; ++i) mbar_init(&bars[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bars[2 * kStages + i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bars[2 * kStages + 2 + i], kEpilogueWarps * CTAS);
    mbar_init_fence();
  }
  if (warp == 2) tensor_memory_alloc<CTAS>(&tmem_base_s, 2 * kColumns);
  tc_fence_before_sync();
  if constexpr (CTAS == 2) cluster_barrier();
  else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_base_s;
  after_previous_kernel();
  Waiter wait;
  wait.begin(status);
  Units u;
  u.begin(c);
  if (KIND == kBoth && e.any != nullptr && *e.any == 0) u.at = w.tiles();    // nothing to do: tiles are all whole here

  if (warp == 0) {
    if (lane == 0) {
      // ---- loads.  Both CTAs count on the first one's barrier: its thread issues the MMAs of both.
      const uint32_t full_there = CTAS == 2 ? address_in(full, 0) : full;
      const uint32_t ring = smem_u32(smem);
      // parts of the terms: of one (0,0), of two (1,0) (0,0), of six (2,0) (1,1) (0,2) (1,0) (0,1) (0,0)
      const int terms = w.blocks / w.depth_blocks, parts_a = terms == 1 ? 0 : terms == 2 ? 0x01 : 0x001012, parts_b = terms < 6 ? 0 : 0x010210;
      int stage = 0, round = 0;
      while (u.next(w)) {
        const int a0 = at_a.own + u.tm * kColumns + (int)rank * kRows;
        const int b0 = at_b.own + u.tn * w.bn + (int)rank * (w.columns(u.tn) / CTAS);
        int term = u.k0 / w.depth_blocks, block = u.k0 - term * w.depth_blocks;
        for (int k = u.k0; k < u.k1; ++k) {
          if (round > 0) wait(empty + 8 * stage, (round - 1) & 1, 1000);
          if (rank == 0) expect_tx(full + 8 * stage, (a_bytes + kOperand) * CTAS);
          const int pa = (parts_a >> (4 * term)) & 3, pb = (parts_b >> (4 * term)) & 3;
          const uint32_t a = ring + stage * 2 * kOperand, b = a + kOperand, bar = full_there + 8 * stage;
          const int ka = at_a.depth + block * kDepth, kb = at_b.depth + block * kDepth;
          if constexpr (A_MN) {
            load_3d<CTAS>(a, &map_a, bar, a0, ka, pa);
            load_3d<CTAS>(a + kOperand / 2, &map_a, bar, a0 + 64, ka, pa);
          } else {
            load_3d<CTAS>(a, &map_a, bar, ka, a0, pa);
          }
          if constexpr (B_MN) {
            load_3d<CTAS>(b, &map_b, bar, b0, kb, pb);
            load_3d<CTAS>(b + kOperand / 2, &map_b, bar, b0 + 64, kb, pb);
          } else {
            load_3d<CTAS>(b, &map_b, bar, kb, b0, pb);
          }
          if (++block == w.depth_blocks) {
            block = 0;
            ++term;
          }
          if (++stage == kStages) {
            stage = 0;
            ++round;
          }
        }
      }
      for (int i = 0; i < kStages; ++i) {                            // what was loaded has been read
        if (round > 0) wait(empty + 8 * stage, (round - 1) & 1, 1001);
        if (++stage == kStages) {
          stage = 0;
          ++round;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---- products.  The whole warp walks: an MMA issued in a divergent branch takes longer.
      const uint32_t format = e.half ? 0u : (1u << 7) | (1u << 10);
      const uint32_t a_low = desc_low(smem_u32(smem), A_MN ? kOperand / 2 : 16), b_low = desc_low(smem_u32(smem) + kOperand, B_MN ? kOperand / 2 : 16);
      constexpr uint32_t kStepA = (A_MN ? 2048 : 32) >> 4, kStepB = (B_MN ? 2048 : 32) >> 4;
      int stage = 0, round = 0, n = 0;
      while (u.next(w)) {
        const uint32_t idesc = (1u << 4) | format | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16) |
                               ((uint32_t)(w.columns(u.tn) >> 3) << 17) | ((uint32_t)(kColumns >> 4) << 24);
        const uint32_t acc = tmem + (n & 1) * kColumns;
        if (n >= 2) wait(read + 8 * (n & 1), ((n >> 1) - 1) & 1, 1002);
        for (int k = u.k0; k < u.k1; ++k) {
          wait(full + 8 * stage, round & 1, 1003);
          __syncwarp();
          tc_fence_after_sync();
          const uint32_t at = (uint32_t)(stage * 2 * kOperand) >> 4;
          if (elect_one()) {
#pragma unroll
            for (int s = 0; s < kDepth / 16; ++s) mma<CTAS>(acc, a_low + at + s * kStepA, b_low + at + s * kStepB, idesc, k > u.k0 || s > 0);
            commit<CTAS>(empty + 8 * stage);
            if (k + 1 == u.k1) commit<CTAS>(done + 8 * (n & 1));
          }
          if (++stage == kStages) {
            stage = 0;
            ++round;
          }
        }
        ++n;
      }
    }
  } else if (warp >= 4) {
    // ---- epilogues: a warp reads the 32 rows that its place in the CTA allows, two warps share their columns
    const int half = (warp - 4) >> 2;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;              // 32 lanes, in bits 16 on
    const uint32_t read_there = CTAS == 2 ? address_in(read, 0) : read;
    if (KIND == kStats && blockIdx.x == 0 && threadIdx.x == 128 && e.zeroed != nullptr) *e.zeroed = 0u;
    float* const turn = reinterpret_cast<float*>(smem + kStages * 2 * kOperand) + (warp - 4) * 32 * kTurnPitch;    // kResult
    uint32_t sums[SEGMENTS ? kSegmentChunks : 1][32];
    auto clear = [&] {                                               // behind a tile, so that its epilogue has the registers
#pragma unroll
      for (int i = 0; i < kSegmentChunks; ++i)
#pragma unroll
        for (int j = 0; j < 32; ++j) sums[i][j] = 0u;
    };
    if constexpr (SEGMENTS) clear();
    int n = 0;
    while (u.next(w)) {
      const int row = u.tm * kColumns + (int)rank * kRows + (warp & 3) * 32 + lane;
      const bool inside = row < w.m;
      const int columns = w.columns(u.tn), chunks = columns >> 5;
      const int from = half == 0 ? 0 : (chunks + 1) >> 1, to = half == 0 ? (chunks + 1) >> 1 : chunks;
      const uint32_t acc = tmem + (n & 1) * kColumns + lanes;
      wait(done + 8 * (n & 1), (n >> 1) & 1, 1004);
      __syncwarp();
      tc_fence_after_sync();
      auto release = [&] {                                           // all that this warp reads of the accumulator has been read
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CTAS == 2) arrive_cluster(read_there + 8 * (n & 1));
          else mbar_arrive(read + 8 * (n & 1));
        }
      };
      // The chunks in turn; the accumulator goes back before the last one's arithmetic.  (The next chunk's load before a chunk's arithmetic:
      // +4 to +10 % at widths up to 512.  Sixteen warps: -8 % at 64, +2 % from 768 on.)
      auto each_chunk = [&](auto f) {
        if (from == to) release();
        for (int i = from; i < to; ++i) {
          uint32_t r[32];
          tmem_ld32(acc + i * 32, r);
          tmem_loaded(r);
          if (i + 1 == to) release();
          f(i, r);
        }
      };
      if constexpr (SEGMENTS) {
        // the last one's sums and the others' meet in tensor memory, where they take no registers of what follows
#pragma unroll
        for (int i = 0; i < kSegmentChunks; ++i) {
          if (from + i >= to) break;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[16];
            tmem_ld16(acc + (from + i) * 32 + 16 * h, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[i][16 * h + j] = __float_as_uint(__uint_as_float(sums[i][16 * h + j]) + __uint_as_float(r[j]));
          }
          if (u.last) tmem_st32(acc + (from + i) * 32, sums[i]);
        }
        if (u.last) {
          tmem_st_wait();
        } else {
          release();
          ++n;
          continue;
        }
      }
      if constexpr (KIND == kStats) {
        const int64_t target = inside ? e.targets[row] : -1;
        RowStats stats;
        each_chunk([&](int i, uint32_t (&r)[32]) {
          const int col = u.tn * w.bn + i * 32;
          stats.add(r, w.n - col);
          const int64_t mine = target - e.column0 - col;
          if (mine >= 0 && mine < 32 && col + mine < w.n) e.at_target[row] = select(r, (int)mine);
        });
        if (inside) e.stats[(int64_t)(2 * u.tn + half) * w.m + row] = stats.result();
      } else if constexpr (KIND == kBoth) {
        const int64_t target = inside ? e.targets[row] : -1;
        const float ref = inside ? e.ref[row] : INFINITY, relative_to = ref == INFINITY ? 0.f : ref;
        const bool store = inside && (e.only == nullptr || e.only[row] != 0);
        const float base = base_of(relative_to);
        float top = -INFINITY, sum = 0.f;
        auto chunk = [&](int i, uint32_t (&r)[32], auto huge) {
          constexpr bool HUGE = decltype(huge)::value;
          const int col = u.tn * w.bn + i * 32, valid = w.n - col;
          const int64_t mine = target - e.column0 - col;
          float p[32];
          if (valid < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = j < valid ? r[j] : __float_as_uint(-INFINITY);
          }
          top = most_of(r, top);
          sum += HUGE && is_huge(relative_to) ? exponentials<true>(r, relative_to, p) : exponentials<false>(r, base, p);
          if (store && mine >= 0 && mine < 32 && mine < valid) {
            const float z = select(r, (int)mine);
            e.at_target[row] = z;
            e.e_target[row] = exponential(z, ref);
          }
          if (store) store_parts(e, p, ref != INFINITY, (int64_t)row * e.p_pitch + col);
        };
        if (__any_sync(~0u, is_huge(relative_to))) each_chunk([&](int i, uint32_t (&r)[32]) { chunk(i, r, std::true_type()); });
        else each_chunk([&](int i, uint32_t (&r)[32]) { chunk(i, r, std::false_type()); });
        if (store) e.stats[(int64_t)(2 * u.tn + half) * w.m + row] = make_float2(top, ref != INFINITY ? sum : 0.f);
      } else if constexpr (KIND == kProbabilities) {
        const float2 lse = inside ? e.lse[row] : make_float2(0.f, 0.f);
        const float factor = inside ? e.factor[row] : 0.f;
        const int64_t target = inside ? e.targets[row] : -1;
        each_chunk([&](int i, uint32_t (&r)[32]) {
          const int col = u.tn * w.bn + i * 32;
          const int64_t mine = target - e.column0 - col;
          if (inside) store_probabilities(e, r, row, (int64_t)row * e.p_pitch + col, lse, factor, mine >= 0 && mine < 32 ? (int)mine : -1);
        });
      } else {
        const int in_tile = (int)rank * kRows + (warp & 3) * 32 + lane;
        each_chunk([&](int i, uint32_t (&r)[32]) {
          store_result(e, w, u, r, row - lane, lane, in_tile, kColumns, i, turn);
        });
      }
      if constexpr (SEGMENTS) clear();
      ++n;
    }
  }
  wait.end(status);
  tc_fence_before_sync();
  __syncwarp();
  if constexpr (CTAS == 2) cluster_barrier();
  else __syncthreads();
  if (warp == 2) tensor_memory_free<CTAS>(tmem, 2 * kColumns);
}

}  // namespace product
}  // namespace sa
