// Selective Attention of one new token of every row over a paged cache, or of a few (FEW, up to kFewTokens) (sm_100a).
//
// What sa_misc.cu's decode step does for one contiguous cache, for rows of any length whose keys and values lie in pages: a row
// has z_j = q.k_j / sqrt(D) - selected[j], y = softmax(z) v, and then selected[j] += relu(q0.k0_j / sqrt(D)) for exempt <= j < t.
// A few tokens: z_ij has what the tokens before i of the same row select taken off, too.
//
// The plan of the step has the rows' keys cut into pieces of equal length.  A CTA takes a (piece, head): a warp streams its keys of K
// and V through a ring of stages of 64 keys; a page, or the part of it that fits a stage, is one TMA box, so a page outside the
// pool reads as zeros and not as somebody's memory.  Four warps have 16 keys of a stage each, as rows of a 16 x 8 matrix product
// (mma.sync): logits = K q, with q in every column so that each lane has the logits of two keys, or with a token a column; y += V^T p
// with p as two bf16 numbers, which keeps 16 bits of it: in neighbouring columns, or in two products.  The warps have softmax sums of
// their own, merged at the end; pieces of a row are merged by the CTA that finishes last, in the order of the pieces.  The CTAs whose
// keys have new tokens among them take those from k, v and write them to their pages.
//
// A few tokens: the CTAs of a head that does not select for itself stream the selecting head's K too (from L2: one of the heads that
// share it has just read it) and make its logits again.  A lane has those of two neighbouring tokens; what is selected by the tokens
// before is a prefix sum over two tokens of a lane and the four lanes of a key.
//
// Bound by HBM (2 D 2 bytes a key and head).  16 heads of head_dim 64: a row of 131,000 tokens 86.5 us, 96 % of the measured
// copy rate (89 in pages of 16); 64 rows of 1 to 7,000 tokens 142 us, 93 %.  With p in 32 bits on the CUDA cores and a lane
// group a key, which is 28 instructions a key, they took 105 and 190 us.  Several tokens of each of the 64 rows: 2, 4, 8 163, 166, 172 us
// (as tiles of 128 queries 383, 384, 391), 5 after 131,000 97 us (207); 16 rows of 1 to 6,000 66 us, 40 % more instructions than for
// one token and a second K through L2.  8 heads of head_dim 128 (as many bytes as 16 of 64): a row of 131,000 91 us, 102 with four
// tokens; 64 rows of 226,000 tokens in all 145 us (16 heads of 64: 145), 168 with four tokens of each.
// Pieces: one wave of CTAs over all heads, or four where the rows alone fill half of one.  131,000 tokens in 1, 1.5, 2, 4 waves:
// 86.5, 91.7, 90.6, 99.7 us; the 64 rows in 1, 2, 4, 8: 159, 159, 139, 140; 16 rows of 1 to 6,000 in 1, 2, 4: 37, 39, 43.
#include <float.h>
#include <type_traits>

#include "sa_paged.cuh"
#include "sa_tc_host.cuh"
#include "sa_tc_ptx.cuh"

namespace sa {
namespace paged {
namespace {

constexpr int kWarps = 4;                       // of arithmetic; one more loads
constexpr int kThreads = 32 * kWarps, kAllThreads = kThreads + 32;
constexpr int kStageKeys = 16 * kWarps;
constexpr int kTileBytes = kStageKeys * 128;    // 64 keys of 64 columns
constexpr int kBarrier = 1;                     // hardware barrier of the arithmetic warps
// The ring: three stages of 64 keys of K and V, or two that have the selecting head's K too.  An SM has four CTAs of head_dim 64, or
// two of 128.
template <int D> constexpr int kRingTiles = 6 * (D / 64);
template <int D> constexpr size_t smem_bytes() { return (size_t)kRingTiles<D> * kTileBytes + 1024; }

struct Strides { int64_t token, head; };

__device__ __forceinline__ void ldmatrix(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose(uint32_t x) {      // of an 8 x 8 matrix, two neighbours of a row a lane
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// p as two bf16 numbers: the rounded one below, what it leaves above
__device__ __forceinline__ uint32_t split(float p) {
  const uint32_t hi = tc::pack_bf16(p, 0.f);
  return (hi & 0xffffu) | (tc::pack_bf16(0.f, p - __uint_as_float(hi << 16)) & 0xffff0000u);
}

template <int D, bool FEW>
__global__ void __launch_bounds__(kAllThreads, D == 64 ? 4 : 2) decode_pages_kernel(
    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __nv_bfloat16* q,
    Strides q_str, const __nv_bfloat16* k_new, Strides k_str, const __nv_bfloat16* v_new, Strides v_str,
    __nv_bfloat16* k_pages, __nv_bfloat16* v_pages, float* selected, int64_t sel_stride, const int* tables, int max_pages,
    int num_pages, int page_shift, int box_rows, const int* header, const DecodeItem* items, int items_max,
    float* partial, int partial_tokens, float* sel_new, int64_t new_stride, unsigned int* tickets, int heads, int groups, int exempt,
    float scale, const int64_t* slots, int total, __nv_bfloat16* __restrict__ y, tc::WaitCtx status, bool beside) {
  constexpr int DK = D / 64, KB = D / 16;
  constexpr int kTokens = FEW ? kFewTokens : 1;                   // of a row, at most
  if (!beside) {
    tc::after_previous_kernel();
  } else {
    // The kernel before is that of the same call's tiles, which this one needs nothing of: each of its blocks has let this one
    // begin after its own wait, when the plan, the pages and the histories that earlier kernels wrote were performed in device
    // memory.  This grid has not waited for those itself, so every thread fences before its first load: none of them is served by
    // a line that was read before.  One block more waits for the tiles' end, so that what comes after both waits for both.
    asm volatile("griddepcontrol.launch_dependents;");
    __threadfence();
    if (blockIdx.x == (unsigned)items_max * heads) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      return;
    }
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[3], empty[3];
  __shared__ float part_s[FEW ? 1 : kWarps * D];
  float* part = FEW ? reinterpret_cast<float*>(ring) : part_s;    // [warp][token][D]; FEW: in the ring, when that has been read
  __shared__ float warp_max[kWarps][kTokens], warp_den[kWarps][kTokens];
  __shared__ unsigned int ticket_s[2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // tokens that no row was given: zeros
  for (int i = blockIdx.x; i < total && !beside; i += gridDim.x) {
    if (slots[i] >= 0) continue;
    for (int u = tid; u < heads * D / 8; u += kAllThreads) reinterpret_cast<uint4*>(y + (int64_t)i * heads * D)[u] = make_uint4(0u, 0u, 0u, 0u);
  }
  const int item = blockIdx.x / (unsigned)heads, h = blockIdx.x - item * heads;
  if (item >= header[kDecodeItems]) return;
  const DecodeItem w = items[item];
  const int per = heads / groups, g = h / per, h0 = g * per;
  const bool selector = h == h0;
  const int t = w.length, c0 = w.c0, c1 = w.c1;
  const int count = FEW ? w.count : 1, a0 = t - count;            // new tokens, from position a0 on
  const bool other = FEW && count > 1 && !selector;               // what the new tokens select among themselves takes another head's logits
  const int tiles = (other ? 3 : 2) * DK;                         // of a stage: K, then V, then K of the head that selects
  const int stages = kRingTiles<D> / tiles, stage_bytes = tiles * kTileBytes;
  const int n_stages = (c1 - c0 + kStageKeys - 1) / kStageKeys;
  float* selb = selected + ((int64_t)w.row * groups + g) * sel_stride;
  float* selnb = per > 1 ? sel_new + ((int64_t)w.row * groups + g) * new_stride : nullptr;

  if (tid == 0) {
    for (int st = 0; st < 3; ++st) {
      tc::mbar_init(&full[st], 1);
      tc::mbar_init(&empty[st], kWarps);
    }
    tc::mbar_init_fence();
  }
  __syncthreads();
  if (warp == kWarps) {
    // ---- loads: a lane a box of 64 columns; its page of the stage after is fetched meanwhile ------------------------------------
    const int boxes = kStageKeys / box_rows, mine = lane % boxes, tile = lane / boxes;      // tile: 64 columns, in the order of a stage
    const int head = tile < 2 * DK ? h : h0;
    const CUtensorMap* map = tile >= DK && tile < 2 * DK ? &map_v : &map_k;
    const int* table = tables + (int64_t)w.row * max_pages;
    auto page_of = [&](int st) {
      const int j = c0 + st * kStageKeys + mine * box_rows;
      return tile < tiles && j < c1 ? __ldg(table + (j >> page_shift)) : -1;
    };
    int page = page_of(0), slot = 0;
    uint32_t phase = 0;
#pragma unroll 1
    for (int st = 0; st < n_stages; ++st) {
      const int j0 = c0 + st * kStageKeys;
      if (st >= stages) tc::mbar_wait(&empty[slot], phase ^ 1u, status, 611);
      const int used = min(boxes, (c1 - j0 + box_rows - 1) / box_rows);
      if (lane == 0) tc::mbar_expect_tx(&full[slot], (uint32_t)(tiles * used * box_rows * 128));
      __syncwarp();
      if (tile < tiles && mine < used)
        tc::tma_load_4d(ring + slot * stage_bytes + tile * kTileBytes + mine * box_rows * 128, map, &full[slot], (tile % DK) * 64,
                        (j0 + mine * box_rows) & ((1 << page_shift) - 1), head, page);
      page = page_of(st + 1);
      if (++slot == stages) slot = 0, phase ^= 1u;
    }
  } else {
    // ---- arithmetic: keys 16 warp .. of every stage; this lane has the logits of keys r and r + 8 of them, with kMany of tokens
    // 2c and 2c + 1
    auto walk = [&](auto many) {
      constexpr bool kMany = decltype(many)::value;
      constexpr int kOwn = kMany ? 2 : 1;                           // tokens whose logits a lane has
      const int r = lane >> 2, c = lane & 3;
      uint32_t qb[KB][2], q0b[kMany ? KB : 1][2];                     // q in every column; kMany: a token a column (the last in the others)
      {
        const int64_t token = w.token + (kMany ? min(r, count - 1) : 0);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(q + token * q_str.token + h * q_str.head);
  #pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          qb[kb][0] = src[kb * 8 + c];
          qb[kb][1] = src[kb * 8 + 4 + c];
        }
        if constexpr (kMany) {
          src = reinterpret_cast<const uint32_t*>(q + token * q_str.token + h0 * q_str.head);
  #pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            q0b[kb][0] = other ? src[kb * 8 + c] : 0u;
            q0b[kb][1] = other ? src[kb * 8 + 4 + c] : 0u;
          }
        }
      }
      // row and 16-byte chunk that this lane gives ldmatrix: of K (keys x dims), and of V to be transposed (dims x keys)
      const int k_row = warp * 16 + (lane & 15), k_chunk = lane >> 4;
      const int v_row = warp * 16 + (lane & 7) + ((lane >> 4) << 3), v_chunk = (lane >> 3) & 1;
      const uint32_t ring0 = tc::smem_u32(ring);
      const uint32_t pick = (r & 1) ? 0x7632u : 0x5410u;            // odd columns take the lower parts of p
      float acc[KB][4];
  #pragma unroll
      for (int kb = 0; kb < KB; ++kb)
  #pragma unroll
        for (int e = 0; e < 4; ++e) acc[kb][e] = 0.f;
      float m[kOwn], den[kOwn];                                     // (a key whose history is infinite has no weight: -inf - (-inf))
  #pragma unroll
      for (int e = 0; e < kOwn; ++e) m[e] = -FLT_MAX, den[e] = 0.f;
      int slot = 0;
      uint32_t phase = 0;
  #pragma unroll 1
      for (int st = 0; st < n_stages; ++st) {
        const int j0 = c0 + st * kStageKeys, ja = j0 + warp * 16 + r, jb = ja + 8;
        // the history sums arrive while the stage is awaited; a new key has none, whatever an earlier row left there
        const float sa = ja < a0 && ja < c1 ? selb[ja] : 0.f, sb = jb < a0 && jb < c1 ? selb[jb] : 0.f;
        tc::mbar_wait(&full[slot], phase, status, 610);
        const uint32_t ks = ring0 + slot * stage_bytes, vs = ks + DK * kTileBytes;
        if (j0 + kStageKeys > a0) {
          // the new keys and values into their rows of the stage and the pool; values behind them become zeros, whatever stands there
          uint8_t* stage = ring + slot * stage_bytes;
          const int row0 = max(a0 - j0, 0), rows = min(t - j0, kStageKeys) - row0;
          for (int u = tid; u < rows * (other ? 3 : 2) * DK * 8; u += kThreads) {
            const int col = u % (DK * 8), which = u / (DK * 8) % (other ? 3 : 2), row = row0 + u / (DK * 8 * (other ? 3 : 2));
            const int64_t token = w.token + (j0 + row - a0), token_slot = slots[token];
            const __nv_bfloat16* from = which == 1 ? v_new + token * v_str.token + h * v_str.head
                                                   : k_new + token * k_str.token + (which == 0 ? h : h0) * k_str.head;
            const uint4 x = reinterpret_cast<const uint4*>(from)[col];
            *reinterpret_cast<uint4*>(stage + (which * DK + (col >> 3)) * kTileBytes + tc::swz_off(row, col & 7)) = x;
            if (which < 2 && token_slot >= 0 && token_slot < ((int64_t)num_pages << page_shift)) {
              const int64_t at = (((token_slot >> page_shift) * heads + h) << page_shift) + (token_slot & ((1 << page_shift) - 1));
              reinterpret_cast<uint4*>((which == 1 ? v_pages : k_pages) + at * D)[col] = x;
            }
          }
          for (int u = tid; u < (kStageKeys - (t - j0)) * DK * 8; u += kThreads) {
            const int row = t - j0 + u / (DK * 8), col = u % (DK * 8);
            *reinterpret_cast<uint4*>(stage + (DK + (col >> 3)) * kTileBytes + row * 128 + (col & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          tc::named_barrier(kBarrier, kThreads);
        }
        float x[4] = {0.f, 0.f, 0.f, 0.f};
  #pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t a[4];
          ldmatrix(ks + (kb >> 2) * kTileBytes + tc::swz_off(k_row, (kb & 3) * 2 + k_chunk), a);
          mma(x, a, qb[kb][0], qb[kb][1]);
        }
        float za[kOwn], zb[kOwn];
        if constexpr (!kMany) {
          const float raw_a = x[0] * scale, raw_b = x[2] * scale;
          if (selector && c == 0) {
            const float ta = ja >= exempt && ja != a0 && raw_a > 0.f ? raw_a : 0.f, tb = jb >= exempt && jb != a0 && raw_b > 0.f ? raw_b : 0.f;
            float* to = per > 1 ? selnb : selb;                     // of its own history nobody else reads this key's
            if (ja < c1) to[ja] = per > 1 ? ta : sa + ta;
            if (jb < c1) to[jb] = per > 1 ? tb : sb + tb;
          }
          za[0] = ja < c1 ? (raw_a - sa) * kLog2e : -INFINITY;
          zb[0] = jb < c1 ? (raw_b - sb) * kLog2e : -INFINITY;
        } else {
          // what each token selects, and the sum of what those before it have: along the tokens that this lane has, then the four lanes
          float x0[4] = {x[0], x[1], x[2], x[3]};
          if (other) {
  #pragma unroll
            for (int e = 0; e < 4; ++e) x0[e] = 0.f;
  #pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              uint32_t a[4];
              ldmatrix(vs + (DK + (kb >> 2)) * kTileBytes + tc::swz_off(k_row, (kb & 3) * 2 + k_chunk), a);
              mma(x0, a, q0b[kb][0], q0b[kb][1]);
            }
          }
          float ta[2], tb[2];
  #pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int token = 2 * c + e, end = token < count ? a0 + token : 0;     // it selects among the keys before its own
            ta[e] = ja >= exempt && ja < end && x0[e] > 0.f ? x0[e] * scale : 0.f;
            tb[e] = jb >= exempt && jb < end && x0[2 + e] > 0.f ? x0[2 + e] * scale : 0.f;
          }
          float upto_a = ta[0] + ta[1], upto_b = tb[0] + tb[1];
  #pragma unroll
          for (int s = 1; s < 4; s <<= 1) {
            const float below_a = __shfl_up_sync(0xffffffffu, upto_a, s, 4), below_b = __shfl_up_sync(0xffffffffu, upto_b, s, 4);
            if (c >= s) upto_a += below_a, upto_b += below_b;
          }
          const float below_a = __shfl_up_sync(0xffffffffu, upto_a, 1, 4), below_b = __shfl_up_sync(0xffffffffu, upto_b, 1, 4);
          float fa = sa + (c > 0 ? below_a : 0.f), fb = sb + (c > 0 ? below_b : 0.f);
          if (selector && c == 3) {                                 // all of the tokens'
            float* to = per > 1 ? selnb : selb;
            if (ja < c1) to[ja] = per > 1 ? upto_a : sa + upto_a;
            if (jb < c1) to[jb] = per > 1 ? upto_b : sb + upto_b;
          }
  #pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int end = 2 * c + e < count ? min(a0 + 2 * c + e + 1, c1) : 0;
            za[e] = ja < end ? (x[e] * scale - fa) * kLog2e : -INFINITY;
            zb[e] = jb < end ? (x[2 + e] * scale - fb) * kLog2e : -INFINITY;
            fa += ta[e];
            fb += tb[e];
          }
        }
        float mx[kOwn];
        bool grew = false;
  #pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          mx[e] = fmaxf(za[e], zb[e]);
          grew = grew || mx[e] > m[e];
        }
        if (__any_sync(0xffffffffu, grew)) {                        // a maximum of the warp grew: rescale its sums
          float f[2];
  #pragma unroll
          for (int e = 0; e < kOwn; ++e) {
            float top = fmaxf(mx[e], m[e]);
  #pragma unroll
            for (int s = 4; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
            f[e] = tc::ex2(m[e] - top);
            m[e] = top;
            den[e] *= f[e];
          }
  #pragma unroll
          for (int kb = 0; kb < KB; ++kb)
  #pragma unroll
            for (int e = 0; e < 4; ++e) acc[kb][e] *= f[e & (kOwn - 1)];
        }
        float pa[kOwn], pb[kOwn];
  #pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          pa[e] = tc::ex2(za[e] - m[e]);
          pb[e] = tc::ex2(zb[e] - m[e]);
          den[e] += pa[e] + pb[e];
        }
        // p as the product wants it: keys 2c, 2c + 1 and 2c + 8, 2c + 9 of column r
        uint32_t p0, p1, low0 = 0u, low1 = 0u;
        if constexpr (!kMany) {
          const uint32_t wa = split(pa[0]), wb = split(pb[0]);
          const uint32_t a0_ = __shfl_sync(0xffffffffu, wa, 8 * c), a1_ = __shfl_sync(0xffffffffu, wa, 8 * c + 4);
          const uint32_t b0_ = __shfl_sync(0xffffffffu, wb, 8 * c), b1_ = __shfl_sync(0xffffffffu, wb, 8 * c + 4);
          p0 = __byte_perm(a0_, a1_, pick);
          p1 = __byte_perm(b0_, b1_, pick);
        } else {
          const uint32_t wa[2] = {split(pa[0]), split(pa[1])}, wb[2] = {split(pb[0]), split(pb[1])};
          p0 = transpose(__byte_perm(wa[0], wa[1], 0x5410u));
          p1 = transpose(__byte_perm(wb[0], wb[1], 0x5410u));
          low0 = transpose(__byte_perm(wa[0], wa[1], 0x7632u));
          low1 = transpose(__byte_perm(wb[0], wb[1], 0x7632u));
        }
  #pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t a[4];
          ldmatrix_trans(vs + (kb >> 2) * kTileBytes + tc::swz_off(v_row, (kb & 3) * 2 + v_chunk), a);
          mma(acc[kb], a, p0, p1);
          if constexpr (kMany) mma(acc[kb], a, low0, low1);
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&empty[slot]);
        if (++slot == stages) slot = 0, phase ^= 1u;
      }
  #pragma unroll
      for (int e = 0; e < kOwn; ++e) {
  #pragma unroll
        for (int s = 4; s < 32; s <<= 1) den[e] += __shfl_xor_sync(0xffffffffu, den[e], s);
        if (lane < (kMany ? 4 : 1)) {
          warp_max[warp][kMany ? 2 * c + e : 0] = m[e];
          warp_den[warp][kMany ? 2 * c + e : 0] = den[e];
        }
      }
      if constexpr (FEW) tc::named_barrier(kBarrier, kThreads);     // all warps have read the ring
      if constexpr (kMany) {
  #pragma unroll
        for (int kb = 0; kb < KB; ++kb)
  #pragma unroll
          for (int e = 0; e < 4; ++e) part[(warp * kTokens + 2 * c + (e & 1)) * D + kb * 16 + r + 4 * (e & 2)] = acc[kb][e];
      } else if (c == 0) {
  #pragma unroll
        for (int kb = 0; kb < KB; ++kb) {                           // both parts of p
          part[warp * kTokens * D + kb * 16 + r] = acc[kb][0] + acc[kb][1];
          part[warp * kTokens * D + kb * 16 + r + 8] = acc[kb][2] + acc[kb][3];
        }
      }
    };
    if constexpr (FEW) {
      if (count > 1) walk(std::true_type{});
      else walk(std::false_type{});                               // (24 rows, two thirds of them of one token: 286 -> 277 us)
    } else {
      walk(std::false_type{});
    }
  }
  __syncthreads();
  // the warps: common maximum, then rescaled sums
  __nv_bfloat16* yrow = y + (int64_t)w.token * heads * D + h * D;
  const int64_t y_token = (int64_t)heads * D;
  const bool whole = w.pieces == 1;
  // sums of a (piece, head), then their maximum and denominator, token after token
  float* prow = partial + ((int64_t)item * heads + h) * partial_tokens * (D + 2);
  for (int i = tid; i < count * D; i += kAllThreads) {
    const int token = i / D, dim = i % D;
    float cta_max = warp_max[0][token];
#pragma unroll
    for (int u = 1; u < kWarps; ++u) cta_max = fmaxf(cta_max, warp_max[u][token]);
    float sum = 0.f, all = 0.f;
#pragma unroll
    for (int u = 0; u < kWarps; ++u) {
      const float f = tc::ex2(warp_max[u][token] - cta_max);
      all = fmaf(warp_den[u][token], f, all);
      sum = fmaf(part[(u * kTokens + token) * D + dim], f, sum);
    }
    if (whole) {
      yrow[token * y_token + dim] = __float2bfloat16_rn(sum / all);
    } else {
      prow[token * (D + 2) + dim] = sum;
      if (dim == 0) {
        prow[token * (D + 2) + D] = cta_max;
        prow[token * (D + 2) + D + 1] = all;
      }
    }
  }
  if (whole && per == 1) return;

  // The last CTA of a (row, head) merges its pieces into y; the last of the heads that share a history vector to finish a piece
  // adds the piece's new selection to it (every reader is done).
  __threadfence();                                                // partials and sel_new visible before the ticket
  __syncthreads();
  unsigned int* row_ticket = tickets + (int64_t)w.first * heads + h;
  unsigned int* range_ticket = tickets + ((int64_t)items_max + item) * heads + g;
  if (tid == 0) {
    ticket_s[0] = whole ? 0u : atomicAdd(row_ticket, 1u);
    ticket_s[1] = per > 1 ? atomicAdd(range_ticket, 1u) : 0u;
  }
  __syncthreads();
  const bool last_of_row = !whole && ticket_s[0] == (unsigned)w.pieces - 1;
  const bool last_of_range = per > 1 && ticket_s[1] == (unsigned)per - 1;
  if (!last_of_row && !last_of_range) return;
  __threadfence();
  if (tid == 0) {                                                 // zero again for the next call
    if (last_of_row) *row_ticket = 0u;
    if (last_of_range) *range_ticket = 0u;
  }
  if (last_of_range) {
    constexpr int kBatch = 8;                                     // independent loads in flight per thread
    for (int base = c0 + tid; base < c1; base += kAllThreads * kBatch) {
      float old_v[kBatch], new_v[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int j = base + u * kAllThreads;
        old_v[u] = (j < c1 && j < a0) ? __ldcg(selb + j) : 0.f;
        new_v[u] = (j < c1) ? __ldcg(selnb + j) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int j = base + u * kAllThreads;
        if (j < c1) selb[j] = old_v[u] + new_v[u];
      }
    }
  }
  if (!last_of_row || warp == kWarps) return;
  // the pieces of the row: their common maximum first, so that the weighted sums have no serial dependence.  A token: warp x folds
  // pieces x, x + 4, .. (lane l owns columns l, l + 32, ..), then the four warps are added; FEW: a warp folds all of a token's.
  // Read past the L1 cache.
  const int64_t next = (int64_t)heads * partial_tokens * (D + 2);
  for (int token = FEW ? warp : 0; token < count; token += FEW ? kWarps : 1) {
    const float* from = partial + ((int64_t)w.first * heads + h) * partial_tokens * (D + 2) + token * (D + 2);
    float top = -FLT_MAX;
    for (int s = lane; s < w.pieces; s += 32) top = fmaxf(top, __ldcg(from + s * next + D));
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    float dsum = 0.f, num[D / 32] = {};
#pragma unroll 4
    for (int s = FEW ? 0 : warp; s < w.pieces; s += FEW ? 1 : kWarps) {
      const float* p = from + s * next;
      const float f = tc::ex2(__ldcg(p + D) - top);
      dsum = fmaf(__ldcg(p + D + 1), f, dsum);
#pragma unroll
      for (int u = 0; u < D / 32; ++u) num[u] = fmaf(__ldcg(p + lane + 32 * u), f, num[u]);
    }
    if constexpr (FEW) {
#pragma unroll
      for (int u = 0; u < D / 32; ++u) yrow[token * y_token + lane + 32 * u] = __float2bfloat16_rn(num[u] / dsum);
    } else {
#pragma unroll
      for (int u = 0; u < D / 32; ++u) part[warp * D + lane + 32 * u] = num[u];
      if (lane == 0) warp_den[warp][0] = dsum;
      tc::named_barrier(kBarrier, kThreads);
      if (tid < D)
        yrow[tid] = __float2bfloat16_rn((part[tid] + part[D + tid] + part[2 * D + tid] + part[3 * D + tid]) /
                                        (warp_den[0][0] + warp_den[1][0] + warp_den[2][0] + warp_den[3][0]));
    }
  }
}

template <int D, bool FEW>
int decode_impl(const Attention& a, bool beside, cudaStream_t s) {
  const StepLayout l = step_layout(a.rows, a.total, a.heads);
  const AttentionScratch w = attention_scratch(a);
  const int page = 1 << a.page_shift, box_rows = min(page, kStageKeys);
  CUtensorMap map_k, map_v;
  int st = tc::make_pool_map(&map_k, a.k_pages, D, page, a.heads, a.num_pages, box_rows);
  if (st != SA_OK) return st;
  st = tc::make_pool_map(&map_v, a.v_pages, D, page, a.heads, a.num_pages, box_rows);
  if (st != SA_OK) return st;
  tc::WaitCtx status;
  st = tc::wait_ctx(&status);
  if (st != SA_OK) return st;
  int* tickets = a.plan_tickets ? a.work + l.tickets : reinterpret_cast<int*>(a.workspace + w.own_tickets);
  if (!a.plan_tickets && !beside) SA_CUDA_CHECK(cudaMemsetAsync(tickets, 0, (size_t)l.tickets_count * 4, s));
  ProfileScope prof(SA_KERNEL_DECODE, s);
  using bf16 = __nv_bfloat16;
  return launch_after(
      decode_pages_kernel<D, FEW>, dim3((unsigned)l.decode_items_max * a.heads + (beside ? 1 : 0)), kAllThreads, smem_bytes<D>(), s,
      map_k, map_v, static_cast<const bf16*>(a.q), Strides{a.q_stride[0], a.q_stride[1]}, static_cast<const bf16*>(a.k),
      Strides{a.k_stride[0], a.k_stride[1]}, static_cast<const bf16*>(a.v), Strides{a.v_stride[0], a.v_stride[1]},
      static_cast<bf16*>(a.k_pages), static_cast<bf16*>(a.v_pages), a.selected, a.sel_stride, a.block_tables, a.max_pages, a.num_pages,
      a.page_shift, box_rows, (const int*)a.work, reinterpret_cast<const DecodeItem*>(a.work + l.decode_items), l.decode_items_max,
      a.workspace + w.partial, min(a.max_count, kFewTokens), a.workspace + w.sel_new, w.key_stride, reinterpret_cast<unsigned*>(tickets),
      a.heads, a.groups, a.exempt, 1.0f / sqrtf((float)D), a.slots, a.total, static_cast<bf16*>(a.y), status, beside);
}

}  // namespace

int decode(const Attention& a, bool beside, cudaStream_t s) {
  const bool few = a.max_count > 1;
  if (a.head_dim == 64) return few ? decode_impl<64, true>(a, beside, s) : decode_impl<64, false>(a, beside, s);
  if (a.head_dim == 128) return few ? decode_impl<128, true>(a, beside, s) : decode_impl<128, false>(a, beside, s);
  return SA_ERR_UNSUPPORTED;
}

}  // namespace paged
}  // namespace sa
