// Selective Attention of a single new token of every row over a paged cache (sm_100a).
//
// What sa_misc.cu's decode step does for one contiguous cache, for rows of any length whose keys and values lie in pages: a row
// has z_j = q.k_j / sqrt(D) - selected[j], y = softmax(z) v, and then selected[j] += relu(q0.k0_j / sqrt(D)) for exempt <= j < t.
//
// The plan of the step has the rows' keys cut into pieces of equal length.  A CTA takes a (piece, head): a warp streams its keys of K
// and V through a ring of stages of 64 keys; a page, or the part of it that fits a stage, is one TMA box, so a page outside the
// pool reads as zeros and not as somebody's memory.  Four warps have 16 keys of a stage each, as rows of a 16 x 16 matrix product
// (mma.sync): logits = K q with q in every column, so that each lane has the logits of two keys; y += V^T [p_hi p_lo], p as two
// bf16 numbers in neighbouring columns, which keeps 16 bits of it.  The warps have softmax sums of their own, merged at the end;
// pieces of a row are merged by the CTA that finishes last, in the order of the pieces.  The piece that ends with the new token
// takes it from k, v and writes it to its page.
//
// Bound by HBM (2 D 2 bytes a key and head).  16 heads of head_dim 64: a row of 131,000 tokens 86.5 us, 96 % of the measured
// copy rate (89 in pages of 16); 64 rows of 1 to 7,000 tokens 142 us, 93 %.  With p in 32 bits on the CUDA cores and a lane
// group a key, which is 28 instructions a key, they took 105 and 190 us.
// Pieces: one wave of CTAs over all heads, or four where the rows alone fill half of one.  131,000 tokens in 1, 1.5, 2, 4 waves:
// 86.5, 91.7, 90.6, 99.7 us; the 64 rows in 1, 2, 4, 8: 159, 159, 139, 140; 16 rows of 1 to 6,000 in 1, 2, 4: 37, 39, 43.
#include <float.h>

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
constexpr int kStages = 3;
constexpr int kBarrier = 1;                     // hardware barrier of the arithmetic warps
template <int D> constexpr size_t smem_bytes() { return (size_t)kStages * 2 * (D / 64) * kTileBytes + 1024; }

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
// p as two bf16 numbers: the rounded one below, what it leaves above
__device__ __forceinline__ uint32_t split(float p) {
  const uint32_t hi = tc::pack_bf16(p, 0.f);
  return (hi & 0xffffu) | (tc::pack_bf16(0.f, p - __uint_as_float(hi << 16)) & 0xffff0000u);
}

template <int D>
__global__ void __launch_bounds__(kAllThreads) decode_pages_kernel(
    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __nv_bfloat16* q,
    Strides q_str, const __nv_bfloat16* k_new, Strides k_str, const __nv_bfloat16* v_new, Strides v_str,
    __nv_bfloat16* k_pages, __nv_bfloat16* v_pages, float* selected, int64_t sel_stride, const int* tables, int max_pages,
    int num_pages, int page_shift, int box_rows, const int* header, const DecodeItem* items, int items_max,
    float* partial, float* sel_new, int64_t new_stride, unsigned int* tickets, int heads, int groups, int exempt,
    float scale, const int64_t* slots, int total, __nv_bfloat16* y, tc::WaitCtx status, bool beside) {
  constexpr int DK = D / 64, KB = D / 16;
  constexpr int kStageBytes = 2 * DK * kTileBytes;                // K, then V
  if (!beside) {
    tc::after_previous_kernel();
  } else {
    // The kernel before is that of the same call's tiles, which this one needs nothing of: it has let this one begin once
    // everything before it was there.  One block more waits for its end, so that what comes after both waits for both.
    asm volatile("griddepcontrol.launch_dependents;");
    if (blockIdx.x == (unsigned)items_max * heads) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      return;
    }
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kStages], empty[kStages];
  __shared__ float part[kWarps][D];
  __shared__ float warp_max[kWarps], warp_den[kWarps];
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
  const int per = heads / groups, g = h / per;
  const bool selector = h - g * per == 0;
  const int t = w.length, c0 = w.c0, c1 = w.c1;
  const int n_stages = (c1 - c0 + kStageKeys - 1) / kStageKeys;
  const bool tail = c1 == t;
  float* selb = selected + ((int64_t)w.row * groups + g) * sel_stride;
  float* selnb = per > 1 ? sel_new + ((int64_t)w.row * groups + g) * new_stride : nullptr;

  if (tid == 0) {
    for (int st = 0; st < kStages; ++st) {
      tc::mbar_init(&full[st], 1);
      tc::mbar_init(&empty[st], kWarps);
    }
    tc::mbar_init_fence();
  }
  __syncthreads();
  if (warp == kWarps) {
    // ---- loads: a lane a box of K or V (64 columns of it); its page of the stage after is fetched meanwhile --------------------
    const int boxes = kStageKeys / box_rows, mine = lane % boxes, tile = lane / boxes;      // tile: K's 64-column tiles, then V's
    const int* table = tables + (int64_t)w.row * max_pages;
    auto page_of = [&](int st) {
      const int j = c0 + st * kStageKeys + mine * box_rows;
      return tile < 2 * DK && j < c1 ? __ldg(table + (j >> page_shift)) : -1;
    };
    int page = page_of(0);
#pragma unroll 1
    for (int st = 0; st < n_stages; ++st) {
      const int slot = st % kStages, j0 = c0 + st * kStageKeys;
      if (st >= kStages) tc::mbar_wait(&empty[slot], ((st / kStages) & 1) ^ 1, status, 611);
      const int used = min(boxes, (c1 - j0 + box_rows - 1) / box_rows);
      if (lane == 0) tc::mbar_expect_tx(&full[slot], (uint32_t)(2 * DK * used * box_rows * 128));
      __syncwarp();
      if (tile < 2 * DK && mine < used)
        tc::tma_load_4d(ring + (size_t)slot * kStageBytes + tile * kTileBytes + mine * box_rows * 128, tile < DK ? &map_k : &map_v, &full[slot],
                        (tile % DK) * 64, (j0 + mine * box_rows) & ((1 << page_shift) - 1), h, page);
      page = page_of(st + 1);
    }
  } else {
    // ---- arithmetic: keys 16 warp .. of every stage; this lane has the logits of keys r and r + 8 of them ----------------------
    const int r = lane >> 2, c = lane & 3;
    uint32_t qb[KB][2];                                           // q in every column
    {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(q + w.token * q_str.token + h * q_str.head);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        qb[kb][0] = src[kb * 8 + c];
        qb[kb][1] = src[kb * 8 + 4 + c];
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
    float m = -FLT_MAX, den = 0.f;                                // (a key whose history is infinite has no weight: -inf - (-inf))
#pragma unroll 1
    for (int st = 0; st < n_stages; ++st) {
      const int slot = st % kStages;
      const int j0 = c0 + st * kStageKeys, ja = j0 + warp * 16 + r, jb = ja + 8;
      // the history sums arrive while the stage is awaited; the new key has none, whatever an earlier row left there
      const float sa = ja < t - 1 && ja < c1 ? selb[ja] : 0.f, sb = jb < t - 1 && jb < c1 ? selb[jb] : 0.f;
      tc::mbar_wait(&full[slot], (st / kStages) & 1, status, 610);
      const uint32_t ks = ring0 + slot * kStageBytes, vs = ks + DK * kTileBytes;
      if (tail && st == n_stages - 1) {
        // the new key and value into their rows of the stage and the pool; values behind them become zeros, whatever stands there
        uint8_t* stage = ring + (size_t)slot * kStageBytes;
        const int64_t token_slot = slots[w.token];
        for (int u = tid; u < 2 * DK * 8; u += kThreads) {
          const int col = u % (DK * 8), row = t - 1 - j0;
          const bool val = u >= DK * 8;
          const uint4 x = val ? reinterpret_cast<const uint4*>(v_new + w.token * v_str.token + h * v_str.head)[col]
                              : reinterpret_cast<const uint4*>(k_new + w.token * k_str.token + h * k_str.head)[col];
          *reinterpret_cast<uint4*>(stage + ((val ? DK : 0) + (col >> 3)) * kTileBytes + tc::swz_off(row, col & 7)) = x;
          if (token_slot >= 0 && token_slot < ((int64_t)num_pages << page_shift)) {
            const int64_t at = (((token_slot >> page_shift) * heads + h) << page_shift) + (token_slot & ((1 << page_shift) - 1));
            reinterpret_cast<uint4*>((val ? v_pages : k_pages) + at * D)[col] = x;
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
      const float raw_a = x[0] * scale, raw_b = x[2] * scale;
      if (selector && c == 0) {
        const float ta = ja >= exempt && ja != t - 1 && raw_a > 0.f ? raw_a : 0.f, tb = jb >= exempt && jb != t - 1 && raw_b > 0.f ? raw_b : 0.f;
        float* to = per > 1 ? selnb : selb;                       // of its own history nobody else reads this key's
        if (ja < c1) to[ja] = per > 1 ? ta : sa + ta;
        if (jb < c1) to[jb] = per > 1 ? tb : sb + tb;
      }
      const float za = ja < c1 ? (raw_a - sa) * kLog2e : -INFINITY, zb = jb < c1 ? (raw_b - sb) * kLog2e : -INFINITY;
      const float mx = fmaxf(za, zb);
      if (__any_sync(0xffffffffu, mx > m)) {                      // the warp's maximum grew: rescale its sums
        float top = fmaxf(mx, m);
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
        const float f = tc::ex2(m - top);
        m = top;
        den *= f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[kb][e] *= f;
      }
      const float pa = tc::ex2(za - m), pb = tc::ex2(zb - m);
      den += pa + pb;
      // keys 2c, 2c + 1 and 2c + 8, 2c + 9, as the product wants them
      const uint32_t wa = split(pa), wb = split(pb);
      const uint32_t a0 = __shfl_sync(0xffffffffu, wa, 8 * c), a1 = __shfl_sync(0xffffffffu, wa, 8 * c + 4);
      const uint32_t b0 = __shfl_sync(0xffffffffu, wb, 8 * c), b1 = __shfl_sync(0xffffffffu, wb, 8 * c + 4);
      const uint32_t p0 = __byte_perm(a0, a1, pick), p1 = __byte_perm(b0, b1, pick);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        uint32_t a[4];
        ldmatrix_trans(vs + (kb >> 2) * kTileBytes + tc::swz_off(v_row, (kb & 3) * 2 + v_chunk), a);
        mma(acc[kb], a, p0, p1);
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty[slot]);
    }
#pragma unroll
    for (int s = 4; s < 32; s <<= 1) den += __shfl_xor_sync(0xffffffffu, den, s);
    if (lane == 0) {
      warp_max[warp] = m;
      warp_den[warp] = den;
    }
    if (c == 0) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {                           // both parts of p
        part[warp][kb * 16 + r] = acc[kb][0] + acc[kb][1];
        part[warp][kb * 16 + r + 8] = acc[kb][2] + acc[kb][3];
      }
    }
  }
  __syncthreads();
  // the warps: common maximum, then rescaled sums
  float cta_max = warp_max[0];
#pragma unroll
  for (int u = 1; u < kWarps; ++u) cta_max = fmaxf(cta_max, warp_max[u]);
  float sum = 0.f, all = 0.f;
#pragma unroll
  for (int u = 0; u < kWarps; ++u) {
    const float f = tc::ex2(warp_max[u] - cta_max);
    all = fmaf(warp_den[u], f, all);
    if (tid < D) sum = fmaf(part[u][tid], f, sum);
  }
  __nv_bfloat16* yrow = y + (int64_t)w.token * heads * D + h * D;
  const bool whole = w.pieces == 1;
  if (whole) {
    if (tid < D) yrow[tid] = __float2bfloat16_rn(sum / all);
    if (per == 1) return;
  } else if (tid < D) {
    float* prow = partial + ((int64_t)item * heads + h) * (D + 2);
    prow[tid] = sum;
    if (tid == 0) {
      prow[D] = cta_max;
      prow[D + 1] = all;
    }
  }

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
        old_v[u] = (j < c1 && j < t - 1) ? __ldcg(selb + j) : 0.f;
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
  // the pieces of the row: their common maximum first, so that the weighted sums have no serial dependence; warp x folds pieces
  // x, x + 4, .. (lane l owns columns l, l + 32, ..), then the four warps are added.  Read past the L1 cache.
  const float* prow = partial + ((int64_t)w.first * heads + h) * (D + 2);
  const int64_t next = (int64_t)heads * (D + 2);
  float top = -FLT_MAX;
  for (int s = lane; s < w.pieces; s += 32) top = fmaxf(top, __ldcg(prow + s * next + D));
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  float dsum = 0.f, num[D / 32] = {};
#pragma unroll 4
  for (int s = warp; s < w.pieces; s += kWarps) {
    const float* p = prow + s * next;
    const float f = tc::ex2(__ldcg(p + D) - top);
    dsum = fmaf(__ldcg(p + D + 1), f, dsum);
#pragma unroll
    for (int u = 0; u < D / 32; ++u) num[u] = fmaf(__ldcg(p + lane + 32 * u), f, num[u]);
  }
#pragma unroll
  for (int u = 0; u < D / 32; ++u) part[warp][lane + 32 * u] = num[u];
  if (lane == 0) warp_den[warp] = dsum;
  tc::named_barrier(kBarrier, kThreads);
  if (tid < D)
    yrow[tid] = __float2bfloat16_rn((part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]) /
                                    (warp_den[0] + warp_den[1] + warp_den[2] + warp_den[3]));
}

template <int D>
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
      decode_pages_kernel<D>, dim3((unsigned)l.decode_items_max * a.heads + (beside ? 1 : 0)), kAllThreads, smem_bytes<D>(), s, map_k, map_v, static_cast<const bf16*>(a.q), Strides{a.q_stride[0], a.q_stride[1]}, static_cast<const bf16*>(a.k),
      Strides{a.k_stride[0], a.k_stride[1]}, static_cast<const bf16*>(a.v), Strides{a.v_stride[0], a.v_stride[1]},
      static_cast<bf16*>(a.k_pages), static_cast<bf16*>(a.v_pages), a.selected, a.sel_stride, a.block_tables, a.max_pages, a.num_pages,
      a.page_shift, box_rows, (const int*)a.work, reinterpret_cast<const DecodeItem*>(a.work + l.decode_items), l.decode_items_max,
      a.workspace + w.partial, a.workspace + w.sel_new, w.key_stride, reinterpret_cast<unsigned*>(tickets), a.heads, a.groups, a.exempt,
      1.0f / sqrtf((float)D), a.slots, a.total, static_cast<bf16*>(a.y), status, beside);
}

}  // namespace

int decode(const Attention& a, bool beside, cudaStream_t s) {
  return a.head_dim == 64 ? decode_impl<64>(a, beside, s) : a.head_dim == 128 ? decode_impl<128>(a, beside, s) : SA_ERR_UNSUPPORTED;
}

}  // namespace paged
}  // namespace sa
