// Selective Attention of a single new token of every row over a paged cache (sm_100a).
//
// What sa_misc.cu's decode step does for one contiguous cache, for rows of any length whose keys and values lie in pages: a row
// has z_j = q.k_j / sqrt(D) - selected[j], y = softmax(z) v, and then selected[j] += relu(q0.k0_j / sqrt(D)) for exempt <= j < t.
//
// The plan of the step has the rows' keys cut into pieces of equal length, about one wave of CTAs (piece, head) where rows
// times heads leave room for it.  A CTA streams its keys of K and V through a ring of 8 KB stages per tensor, two stages ahead
// of the arithmetic; a page, or the part of it that fits a stage, is one TMA box, so a page outside the pool reads as zeros and
// not as somebody's memory.  The piece that ends with the new token takes it from k, v and writes it to its page.  Pieces of a
// row are merged by the CTA that finishes last, in the order of the pieces.
//
// Bound by HBM (2 D 2 bytes a key and head).
#include "sa_paged.cuh"
#include "sa_tc_host.cuh"
#include "sa_tc_ptx.cuh"

namespace sa {
namespace paged {
namespace {

constexpr int kThreads = 128;
constexpr int kStages = 3;
constexpr int kStageBytes = 8192;               // per tensor
constexpr size_t kSmemBytes = (size_t)kStages * 2 * kStageBytes + 128;
constexpr int kWindow = 256;                    // boxes whose pages are held in shared memory

struct Strides { int64_t token, head; };

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __bfloat1622float2(h[e]);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads) decode_pages_kernel(
    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __nv_bfloat16* __restrict__ q,
    Strides q_str, const __nv_bfloat16* __restrict__ k_new, Strides k_str, const __nv_bfloat16* __restrict__ v_new, Strides v_str,
    __nv_bfloat16* k_pages, __nv_bfloat16* v_pages, float* selected, int64_t sel_stride, const int* __restrict__ tables, int max_pages,
    int num_pages, int page_shift, int box_rows, const int* __restrict__ header, const DecodeItem* __restrict__ items, int items_max,
    float* __restrict__ partial, float* __restrict__ sel_new, int64_t new_stride, unsigned int* tickets, int heads, int groups, int exempt,
    float scale, const int64_t* __restrict__ slots, int total, __nv_bfloat16* __restrict__ y, tc::WaitCtx status) {
  constexpr int kLanes = D / 8;                                   // lanes per key
  constexpr int kGroups = kThreads / kLanes;                      // keys the CTA covers per step
  constexpr int kRowBytes = D * 2;
  constexpr int kStageKeys = kStageBytes / kRowBytes;
  constexpr int kPer = kStageKeys / kGroups;                      // keys per group per stage
  static_assert(kPer == 4, "stage layout");
  tc::after_previous_kernel();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  __shared__ uint64_t full[kStages];
  __shared__ float red[kThreads];
  __shared__ float gmax[kGroups];
  __shared__ float accs[kGroups][D];
  __shared__ float part[4][128 + 1];
  __shared__ unsigned int ticket_s[2];
  __shared__ int page_s[kWindow];

  const int tid = threadIdx.x;
  // tokens that no row was given: zeros
  for (int i = blockIdx.x; i < total; i += gridDim.x) {
    if (slots[i] >= 0) continue;
    for (int u = tid; u < heads * D / 8; u += kThreads) reinterpret_cast<uint4*>(y + (int64_t)i * heads * D)[u] = make_uint4(0u, 0u, 0u, 0u);
  }
  const int item = blockIdx.x / (unsigned)heads, h = blockIdx.x - item * heads;
  if (item >= header[kDecodeItems]) return;
  const DecodeItem w = items[item];
  const int per = heads / groups, g = h / per;
  const bool selector = h - g * per == 0;
  const int t = w.length, c0 = w.c0, c1 = w.c1;
  const int n_stages = (c1 - c0 + kStageKeys - 1) / kStageKeys;
  const int grp = tid / kLanes, lane = tid % kLanes;
  const bool tail = c1 == t;
  const int* table = tables + (int64_t)w.row * max_pages;
  const int boxes = kStageKeys / box_rows;                        // of a stage and tensor
  const int window = kWindow / boxes;                             // stages

  auto load_window = [&](int st0) {                               // the pages of stages st0 ..
    for (int i = tid; i < kWindow; i += kThreads) {
      const int j = c0 + st0 * kStageKeys + i * box_rows;
      page_s[i] = j < c1 ? table[j >> page_shift] : -1;
    }
  };
  auto issue = [&](int st) {                                      // warp 0: a lane a box
    const int j0 = c0 + st * kStageKeys;
    uint8_t* dst = ring + (size_t)(st % kStages) * 2 * kStageBytes;
    uint64_t* bar = &full[st % kStages];
    const int used = min(boxes, (c1 - j0 + box_rows - 1) / box_rows);
    if (tid == 0) tc::mbar_expect_tx(bar, 2u * (uint32_t)(used * box_rows * kRowBytes));
    __syncwarp();
    const int u = tid & 15;
    if (u < used) {
      const int page = page_s[(st % window) * boxes + u], at = (j0 + u * box_rows) & ((1 << page_shift) - 1);
      const bool val = tid >= 16;
      tc::tma_load_4d(dst + (val ? kStageBytes : 0) + u * box_rows * kRowBytes, val ? &map_v : &map_k, bar, 0, at, h, page);
    }
  };
  load_window(0);
  if (tid == 0) {
    for (int st = 0; st < kStages; ++st) tc::mbar_init(&full[st], 1);
    tc::mbar_init_fence();
  }
  __syncthreads();
  if (tid < 32)
    for (int st = 0; st < min(kStages - 1, n_stages); ++st) issue(st);

  float qv[8];
  load8(q + w.token * q_str.token + h * q_str.head + lane * 8, qv);
  float* selb = selected + ((int64_t)w.row * groups + g) * sel_stride;
  float* selnb = per > 1 ? sel_new + ((int64_t)w.row * groups + g) * new_stride : nullptr;
  float m = -INFINITY, den = 0.f, acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll 1
  for (int st = 0; st < n_stages; ++st) {
    const int j0 = c0 + st * kStageKeys;
    float sv[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {                              // the history sums arrive while the stage is awaited
      const int j = j0 + u * kGroups + grp;
      sv[u] = (j < c1 && j < t - 1) ? selb[j] : 0.f;              // the new key has none, whatever an earlier row left there
    }
    // the slot that stage st + kStages - 1 uses was read in iteration st - 1; every thread is past it
    const int ahead = st + kStages - 1;
    if (ahead < n_stages) {
      if (ahead % window == 0) {
        load_window(ahead);
        __syncthreads();
      }
      if (tid < 32) issue(ahead);
    }
    tc::mbar_wait(&full[st % kStages], (st / kStages) & 1, status, 610);
    uint8_t* ks = ring + (size_t)(st % kStages) * 2 * kStageBytes;
    uint8_t* vs = ks + kStageBytes;
    if (tail && st == n_stages - 1) {                             // the new key and value: into their rows of the stage and the pool
      constexpr int kChunks = kRowBytes / 16;
      const int64_t slot = slots[w.token];
      if (tid < 2 * kChunks) {
        const bool val = tid >= kChunks;
        const int c = tid - (val ? kChunks : 0);
        const uint4 x = val ? reinterpret_cast<const uint4*>(v_new + w.token * v_str.token + h * v_str.head)[c]
                            : reinterpret_cast<const uint4*>(k_new + w.token * k_str.token + h * k_str.head)[c];
        reinterpret_cast<uint4*>((val ? vs : ks) + (t - 1 - j0) * kRowBytes)[c] = x;
        if (slot >= 0 && slot < ((int64_t)num_pages << page_shift)) {
          const int64_t row = ((slot >> page_shift) * heads + h) * (int64_t)(1 << page_shift) + (slot & ((1 << page_shift) - 1));
          reinterpret_cast<uint4*>((val ? v_pages : k_pages) + row * D)[c] = x;
        }
      }
      __syncthreads();
    }

    float z[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      float kx[8];
      load8(reinterpret_cast<const __nv_bfloat16*>(ks + (u * kGroups + grp) * kRowBytes) + lane * 8, kx);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(qv[e], kx[e], dot);
      z[u] = dot;
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
#pragma unroll
      for (int sft = kLanes / 2; sft > 0; sft >>= 1) z[u] += __shfl_xor_sync(0xffffffffu, z[u], sft);
    }
    float mx = m;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int j = j0 + u * kGroups + grp;
      const float raw = z[u] * scale;
      if (j < c1) {
        if (selector && lane == 0) {
          const float took = (j >= exempt && j != t - 1 && raw > 0.f) ? raw : 0.f;
          if (per > 1) selnb[j] = took;
          else selb[j] = sv[u] + took;                            // nobody else reads this key's history
        }
        z[u] = (raw - sv[u]) * kLog2e;
      } else {
        z[u] = -INFINITY;                                         // behind the row: whatever the page holds there
      }
      mx = fmaxf(mx, z[u]);
    }
    if (mx > m) {                                                 // the group's maximum grew: rescale its sums
      const float c = exp2f(m - mx);                              // m = -inf on the first keys: c = 0
      den *= c;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= c;
      m = mx;
    }
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      if (z[u] != -INFINITY) {
        const float p = exp2f(z[u] - m);
        float vx[8];
        load8(reinterpret_cast<const __nv_bfloat16*>(vs + (u * kGroups + grp) * kRowBytes) + lane * 8, vx);
        den += p;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(p, vx[e], acc[e]);
      }
    }
    __syncthreads();                                              // stage read by everyone: its slot may be refilled
  }

  // merge the groups: common maximum, then rescaled sums
  if (lane == 0) gmax[grp] = m;
  __syncthreads();
  float cta_max = -INFINITY;
#pragma unroll 4
  for (int gg = 0; gg < kGroups; ++gg) cta_max = fmaxf(cta_max, gmax[gg]);
  const float c = (m == -INFINITY) ? 0.f : exp2f(m - cta_max);    // a group that saw no key contributes nothing
#pragma unroll
  for (int e = 0; e < 8; ++e) accs[grp][lane * 8 + e] = acc[e] * c;
  if (lane == 0) red[grp] = den * c;
  __syncthreads();
  float sum = 0.f, all = 0.f;
  if (tid < D) {
#pragma unroll 4
    for (int gg = 0; gg < kGroups; ++gg) {
      sum += accs[gg][tid];
      all += red[gg];
    }
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
    for (int base = c0 + tid; base < c1; base += kThreads * kBatch) {
      float old_v[kBatch], new_v[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int j = base + u * kThreads;
        old_v[u] = (j < c1 && j < t - 1) ? __ldcg(selb + j) : 0.f;
        new_v[u] = (j < c1) ? __ldcg(selnb + j) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int j = base + u * kThreads;
        if (j < c1) selb[j] = old_v[u] + new_v[u];
      }
    }
  }
  if (!last_of_row) return;
  // the pieces of the row: their common maximum first, so that the weighted sums have no serial dependence; warp x folds pieces
  // x, x + 4, .. (lane l owns columns l, l + 32, ..), then the four warps are added.  Read past the L1 cache.
  const float* prow = partial + ((int64_t)w.first * heads + h) * (D + 2);
  const int64_t next = (int64_t)heads * (D + 2);
  const int warp = tid >> 5, ln = tid & 31;
  float top = -INFINITY;
  for (int s = ln; s < w.pieces; s += 32) top = fmaxf(top, __ldcg(prow + s * next + D));
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  float dsum = 0.f, num[D / 32] = {};
#pragma unroll 4
  for (int s = warp; s < w.pieces; s += 4) {
    const float* p = prow + s * next;
    const float f = exp2f(__ldcg(p + D) - top);
    dsum = fmaf(__ldcg(p + D + 1), f, dsum);
#pragma unroll
    for (int u = 0; u < D / 32; ++u) num[u] = fmaf(__ldcg(p + ln + 32 * u), f, num[u]);
  }
#pragma unroll
  for (int u = 0; u < D / 32; ++u) part[warp][ln + 32 * u] = num[u];
  if (ln == 0) part[warp][128] = dsum;
  __syncthreads();
  if (tid < D)
    yrow[tid] = __float2bfloat16_rn((part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid]) /
                                    (part[0][128] + part[1][128] + part[2][128] + part[3][128]));
}

template <int D>
int decode_impl(const Attention& a, cudaStream_t s) {
  const StepLayout l = step_layout(a.rows, a.total, a.heads);
  const AttentionScratch w = attention_scratch(a);
  constexpr int kStageKeys = kStageBytes / (2 * D);
  const int page = 1 << a.page_shift, box_rows = min(page, kStageKeys);
  CUtensorMap map_k, map_v;
  int st = tc::make_pool_map(&map_k, a.k_pages, D, page, a.heads, a.num_pages, D, box_rows, false);
  if (st != SA_OK) return st;
  st = tc::make_pool_map(&map_v, a.v_pages, D, page, a.heads, a.num_pages, D, box_rows, false);
  if (st != SA_OK) return st;
  tc::WaitCtx status;
  st = tc::wait_ctx(&status);
  if (st != SA_OK) return st;
  int* tickets = a.plan_tickets ? a.work + l.tickets : reinterpret_cast<int*>(a.workspace + w.own_tickets);
  if (!a.plan_tickets) SA_CUDA_CHECK(cudaMemsetAsync(tickets, 0, (size_t)l.tickets_count * 4, s));
  auto kernel = decode_pages_kernel<D>;
  SA_CUDA_CHECK(allow_smem(kernel, kSmemBytes));
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3((unsigned)l.decode_items_max * a.heads);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = kSmemBytes;
  config.stream = s;
  config.attrs = &attr;
  config.numAttrs = 1;
  ProfileScope prof(SA_KERNEL_DECODE, s);
  count_launch();
  using bf16 = __nv_bfloat16;
  SA_CUDA_CHECK(cudaLaunchKernelEx(
      &config, kernel, map_k, map_v, static_cast<const bf16*>(a.q), Strides{a.q_stride[0], a.q_stride[1]}, static_cast<const bf16*>(a.k),
      Strides{a.k_stride[0], a.k_stride[1]}, static_cast<const bf16*>(a.v), Strides{a.v_stride[0], a.v_stride[1]},
      static_cast<bf16*>(a.k_pages), static_cast<bf16*>(a.v_pages), a.selected, a.sel_stride, a.block_tables, a.max_pages, a.num_pages,
      a.page_shift, box_rows, (const int*)a.work, reinterpret_cast<const DecodeItem*>(a.work + l.decode_items), l.decode_items_max,
      a.workspace + w.partial, a.workspace + w.sel_new, w.key_stride, reinterpret_cast<unsigned*>(tickets), a.heads, a.groups, a.exempt,
      1.0f / sqrtf((float)D), a.slots, a.total, static_cast<bf16*>(a.y), status));
  return SA_OK;
}

}  // namespace

int decode(const Attention& a, cudaStream_t s) {
  return a.head_dim == 64 ? decode_impl<64>(a, s) : a.head_dim == 128 ? decode_impl<128>(a, s) : SA_ERR_UNSUPPORTED;
}

}  // namespace paged
}  // namespace sa
