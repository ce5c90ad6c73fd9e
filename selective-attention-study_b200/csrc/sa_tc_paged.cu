// Tensor-core engine over a paged cache: rows (requests) of any length, each with the tokens that the step gives it (sm_100a).
//
//   store_kernel          new keys and values into their pages; zeros for tokens that no row was given
//   colsum_pages_kernel   selection pass: column sums of a query tile's relu'd, masked logits, key tile by key tile
//   scan_pages_kernel     their running sum over the tiles of a row, from the row's history on (-> what the tiles start from), and
//                         the history moved on
//   forward_pair_kernel, forward_self_kernel, forward_wide_kernel (PAGED)   sa_tc_fwd_pair.cuh, sa_tc_fwd_self.cuh, sa_tc_fwd_wide.cuh
//
// The plan of the step (sa_paged.cu) says which tiles there are; the host knows bounds, so a grid covers those and CTAs without
// a tile return at once.  A query tile is 128 positions of one row, counted from its token 0, as the key tiles are: the
// triangular running sum needs both to start at the same places.  A key tile is 128 / page_size TMA boxes (or one), which land
// one behind the other as the rows of one swizzled operand tile.
//
// Rows of a tile that are other sequences' queries, and keys behind a row's last token (in its own page, where an earlier row's
// data stands, or in none), must not reach anything: they are left out of the selection and the logits by selection, not by
// multiplication, and the values among them are zeroed in shared memory.
#include "sa_tc_fwd_pair.cuh"
#include "sa_tc_fwd_wide.cuh"

namespace sa {
namespace tc {
namespace {

using paged::Attention;
using paged::TileItem;

// ---- new rows -----------------------------------------------------------------------------------------------------------------
// Bound by memory from some thousand tokens on: 2,048 tokens of 16 heads (17 MB) 6 us, 300 of 12 4 us.
struct TokenRows {
  const uint4* ptr;
  int64_t token, head;               // strides in 16-byte units
};
// A unit is 16 bytes of one token's K or V; heads * units of a token are neighbours.
__global__ void __launch_bounds__(256) store_kernel(TokenRows k, TokenRows v, uint4* k_pages, uint4* v_pages, uint4* y,
                                                    const int64_t* slots, int total, int heads, int row_units, int num_pages,
                                                    int page_shift, unsigned int* tickets, int n_tickets, unsigned int* more_tickets,
                                                    int n_more) {
  after_previous_kernel();
  const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = first; i < n_tickets; i += step) tickets[i] = 0u;
  for (int64_t i = first; i < n_more; i += step) more_tickets[i] = 0u;
  const int per_token = heads * row_units;
  const int64_t n = (int64_t)total * per_token, slots_end = (int64_t)num_pages << page_shift;
  for (int64_t i = first; i < n; i += step) {
    const int token = (int)(i / per_token), u = (int)(i - (int64_t)token * per_token), h = u / row_units, c = u - h * row_units;
    const int64_t slot = slots[token];
    if (slot < 0) y[i] = make_uint4(0u, 0u, 0u, 0u);
    if (slot < 0 || slot >= slots_end) continue;
    const int64_t row = ((((slot >> page_shift) * heads + h) << page_shift) + (slot & ((1 << page_shift) - 1))) * row_units + c;
    k_pages[row] = k.ptr[token * k.token + h * k.head + c];
    v_pages[row] = v.ptr[token * v.token + h * v.head + c];
  }
}

// ---- what the keys have received before each tile ------------------------------------------------------------------------------
// col[t pitch] = what key j has received before tile t of its row, in place of what it receives from it, for tiles [t, n); returns
// the sum after the last.  The loads go past the L1 cache: other CTAs of the same launch may have written them.
__device__ __forceinline__ float scan_key(float* col, int64_t pitch, int t, int n, float run) {
  for (; t + 8 <= n; t += 8) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = __ldcg(col + (t + u) * pitch);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      col[(t + u) * pitch] = run;
      run += x[u];
    }
  }
  for (; t < n; ++t) {
    const float x = __ldcg(col + t * pitch);
    col[t * pitch] = run;
    run += x;
  }
  return run;
}
// The scan of the keys of one row and group (`first`: its first tile): `selected` moved on.  A new key has received nothing before
// the step, whatever an earlier row left there.
struct History {
  float* selected;
  int64_t stride;                    // keys of a row
  unsigned int* tickets;             // colsum_pages_kernel scans: one a row (at its first tile), group and key tile; else null
};
__device__ __forceinline__ void scan_row_key(float* carry, int64_t key_stride, int groups, int t0, int n, int g, int j, const TileItem& w,
                                             const History& history) {
  float* sel = history.selected + ((int64_t)w.row * groups + g) * history.stride + j;
  const float run = j < w.cached ? *sel : 0.f;
  *sel = scan_key(carry + ((int64_t)t0 * groups + g) * key_stride + j, groups * key_stride, max(j / kTile - w.cached / kTile, 0), n, run);
}

// ---- selection column sums --------------------------------------------------------------------------------------------------
// As colsum_kernel (sa_tc_fwd.cu), with the loops the other way round: a CTA keeps one query tile and takes a run of `chunk` key
// tiles, since rows have few query tiles.  128 threads own a key each, a fifth warp loads and issues, one tile ahead.  Bound by latency
// and issue as that one: 17 query tiles x 251 key tiles of head_dim 64 25 us, 16 heads each for itself 17 x 63 64 us.
// With a key tile a CTA, the last of a row's CTAs to finish it also scans it (scan_pages_kernel's work): a launch fewer.
template <int D>
__global__ void __launch_bounds__(160) colsum_pages_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                           float* carry, int exempt, float scale, WaitCtx status, int chunk,
                                                           const TileItem* tiles, const __grid_constant__ PagedWalk paged, History history) {
  constexpr int DK = D / 64;
  after_previous_kernel();
  if ((int)blockIdx.x >= paged.header[paged::kTiles]) return;
  const TileItem w = tiles[blockIdx.x];
  const int nj0 = blockIdx.y * chunk, h = blockIdx.z;
  if (nj0 > w.mi) return;
  const int count = min(chunk, w.mi + 1 - nj0);
  const int i0 = w.mi * kTile;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q0s = smem;                               // DK tiles [128 queries][64]
  uint8_t* k0s = smem + DK * kRowTile;               // 2 stages x DK tiles [128 keys][64]
  __shared__ uint64_t bar_q, bar_zero, bar_k[2], bar_mma[2], bar_read[2];
  __shared__ uint32_t tmem_base_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&bar_q, 1);
    mbar_init(&bar_zero, 4);
    for (int u = 0; u < 2; ++u) {
      mbar_init(&bar_k[u], 1);
      mbar_init(&bar_mma[u], 1);
      mbar_init(&bar_read[u], 4);
    }
    mbar_init_fence();
  }
  if (warp == 0) tmem_alloc(&tmem_base_s, 256);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_base_s;

  if (warp == 4) {
    Waiter wait;
    wait.begin(status);
    auto await = [&](uint64_t* bar, uint32_t parity, int site) { wait.left = wait_call(smem_u32(bar), parity, site, wait.left); };
    const PageBoxes boxes{paged.tables + (int64_t)w.row * paged.max_pages, paged.page_shift, paged.box_rows};
    int page = boxes.page(nj0 * kTile, w.length, lane);
    const uint32_t idesc = instr_desc_bf16(128, 128, false, false);
    const uint32_t k_low = desc_low(smem_u32(k0s), 16), q_low = desc_low(smem_u32(q0s), 16);
    auto load_k = [&](int it) {
      const int j0 = (nj0 + it) * kTile, used = boxes.count(j0, w.length);
      uint64_t* bar = &bar_k[it & 1];
      if (elect_one()) mbar_expect_tx(bar, DK * used * paged.box_rows * 128);
      __syncwarp();
      if (lane < used)
        for (int s = 0; s < DK; ++s)
          tma_load_4d(k0s + ((it & 1) * DK + s) * kRowTile + lane * paged.box_rows * 128, &map_k, bar, s * 64, boxes.at(j0, lane), h, page);
      __syncwarp();
      page = boxes.page(j0 + kTile, w.length, lane);
    };
    if (elect_one()) {
      mbar_expect_tx(&bar_q, DK * kRowTile);
      for (int s = 0; s < DK; ++s) tma_load_4d(q0s + s * kRowTile, &map_q, &bar_q, s * 64, w.token + i0 - w.cached, h, 0);
    }
    __syncwarp();
    load_k(0);
    if (count > 1) load_k(1);
    await(&bar_q, 0, 211);
    await(&bar_zero, 0, 215);
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      const int st = it & 1;
      const uint32_t ph = (uint32_t)((it >> 1) & 1);
      if (it >= 2) await(&bar_read[st], ph ^ 1u, 213);                   // the columns' last tile has been read
      await(&bar_k[st], ph, 210);
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < 4 * DK; ++ks) {
          const uint32_t off = (uint32_t)((ks >> 2) * kRowTile + (ks & 3) * 32) >> 4;
          const uint32_t kl = k_low + (uint32_t)(st * DK * kRowTile >> 4) + off;
          if (ks == 0) mma_ss_low<false>(tmem + st * 128, kl, q_low + off, idesc);
          else mma_ss_low<true>(tmem + st * 128, kl, q_low + off, idesc);
        }
        mma_commit(&bar_mma[st]);
      }
      __syncwarp();
      if (it >= 1 && it + 1 < count) {                                   // the other stage: its MMA has completed
        await(&bar_mma[st ^ 1], (uint32_t)(((it - 1) >> 1) & 1), 214);
        load_k(it + 1);
      }
    }
    if (lane == 0) wait.end(status);
    __syncwarp();
  } else {
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    const int lo = max(w.cached - i0, 0), hi = min(w.length - i0, kTile);  // the tile's queries that are the row's
    float* dst = carry + ((int64_t)blockIdx.x * gridDim.z + h) * paged.key_stride;
    if (lo > 0 || hi < kTile) {                                            // the others select nothing: zeros
      mbar_wait(&bar_q, 0, status, 216);
      if (tid < lo || tid >= hi)
        for (int u = 0; u < 8 * DK; ++u) *reinterpret_cast<uint4*>(q0s + (u >> 3) * kRowTile + tid * 128 + (u & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
      fence_async_smem();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar_zero);
#pragma unroll 1
    for (int it = 0; it < count; ++it) {
      mbar_wait(&bar_mma[it & 1], (uint32_t)((it >> 1) & 1), status, 212);
      tc_fence_after_sync();
      const bool diag = nj0 + it == w.mi;
      const int from = max(lo, tid + 1);                                  // (key and query count from the same position)
      float2 acc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] = make_float2(0.f, 0.f);
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t r[32];
        tmem_ld32(lane_base + (it & 1) * 128 + c0, r);
        tmem_ld_wait();
        if (diag) {                                                        // and where keys behind the row stand
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c0 + e < from || c0 + e >= hi) r[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          acc[(e >> 1) & 3] = __fadd2_rn(acc[(e >> 1) & 3], make_float2(fmaxf(__uint_as_float(r[e]), 0.f),
                                                                        fmaxf(__uint_as_float(r[e + 1]), 0.f)));
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_read[it & 1]);
      const float2 s2 = __fadd2_rn(__fadd2_rn(acc[0], acc[1]), __fadd2_rn(acc[2], acc[3]));
      const int j = (nj0 + it) * kTile + tid;
      if (j < w.length) dst[j] = (j < exempt) ? 0.f : (s2.x + s2.y) * scale;
    }
  }
  tc_fence_before_sync();
  if (history.tickets != nullptr) __threadfence();                         // the sums, before the ticket
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 256);
  if (history.tickets == nullptr) return;
  __shared__ bool last_s;
  const int first = w.cached / kTile, n = (w.length - 1) / kTile + 1 - first, t0 = w.tile - (w.mi - first);      // the row's tiles
  if (tid == 0) {
    const unsigned all = n - max(nj0 - first, 0);                          // of its tiles reach these keys
    last_s = atomicAdd(history.tickets + ((int64_t)t0 * gridDim.z + h) * gridDim.y + blockIdx.y, 1u) == all - 1u;
  }
  __syncthreads();
  if (!last_s || tid >= kTile) return;
  __threadfence();
  const int j = nj0 * kTile + tid;
  if (j < w.length) scan_row_key(carry, paged.key_stride, gridDim.z, t0, n, h, j, w, history);
}

// One thread per key and group of a row that has tiles (8 us for 17 tiles of 32,000 keys).
__global__ void __launch_bounds__(256) scan_pages_kernel(float* carry, int64_t key_stride, const int* tile_start, const TileItem* tiles,
                                                         int groups, History history) {
  after_previous_kernel();
  const int r = blockIdx.z, g = blockIdx.y;
  const int t0 = tile_start[r], n = tile_start[r + 1] - t0;
  if (n == 0) return;
  const TileItem w = tiles[t0];                                 // the row's first tile
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j < w.length) scan_row_key(carry, key_stride, groups, t0, n, g, j, w, history);
}

// The histories of the rows that have tiles as they were before the scan: what their first tile starts from.
__global__ void __launch_bounds__(256) restore_kernel(const float* __restrict__ carry, int64_t key_stride, const int* __restrict__ tile_start,
                                                      const TileItem* __restrict__ tiles, int groups, float* selected, int64_t sel_stride) {
  const int r = blockIdx.z, g = blockIdx.y, t0 = tile_start[r];
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (tile_start[r + 1] == t0 || j >= tiles[t0].cached) return;
  selected[((int64_t)r * groups + g) * sel_stride + j] = carry[((int64_t)t0 * groups + g) * key_stride + j];
}

// Two heads a CTA (10 units of time a step) or one (7)?  Of one row the walks are known: `tiles` of them, up to `longest` key tiles, with
// a set-up of three steps each.  Either kernel takes as long as its longest walk, or as all of them over the SMs; of one head a CTA the walks
// that find no SM at first come after the shortest of the others.  Several rows: by the number of CTAs, as over contiguous caches.
// Two heads and one, in us: 16 heads, a prompt of 1,300 46, 34, of 2,000 57, 48, of 3,000 81, 89, of 8,000 314, 400; 2,000 after 2,000 98,
// 99, after 8,000 207, 239; 8 heads, a prompt of 4,000 97, 73, of 8,000 179, 214; 12 heads, 1,300 after 20,000 402, 283; 32 heads, a
// prompt of 1,300 48, 54, 1,300 after 8,000 327, 328.
bool two_heads(int rows, int tiles, int longest, int heads) {
  if (rows > 1) return (int64_t)tiles * heads > kSms;
  const double steps = tiles * (longest - 0.5 * (tiles - 1) + 3), top = longest + 3, waiting = top - (double)kSms / heads;
  const double two = 10 * max(top, steps * heads / 2 / kSms);
  const double one = 7 * max(max(top, steps * heads / kSms), tiles * heads > kSms ? 2 * waiting : 0.0);
  return two < one;
}

template <int D>
int tiles_impl(const Attention& a, bool* moved, cudaStream_t s) {
  constexpr int DK = D / 64;
  const paged::StepLayout l = paged::step_layout(a.rows, a.total, a.heads);
  const paged::AttentionScratch w = paged::attention_scratch(a);
  const int page = 1 << a.page_shift, box_rows = min(page, kTile);
  const bool self = a.groups == a.heads;
  CUtensorMap map_q, map_k, map_v;
  int st = make_map_16bit(&map_q, a.q, D, a.total, a.heads, 1, a.q_stride[0], a.q_stride[1], 0, kTile);
  if (st != SA_OK) return st;
  st = make_pool_map(&map_k, a.k_pages, D, page, a.heads, a.num_pages, box_rows);
  if (st != SA_OK) return st;
  st = make_pool_map(&map_v, a.v_pages, D, page, a.heads, a.num_pages, box_rows);
  if (st != SA_OK) return st;
  WaitCtx status;
  st = wait_ctx(&status);
  if (st != SA_OK) return st;

  unsigned int* const walk_tickets = reinterpret_cast<unsigned int*>(a.workspace + w.tickets);
  // key tiles per CTA of the selection (the query tile and the set-up are paid per CTA): 32 where that still gives every SM several
  // CTAs, else 8, or 4 where that would be fewer than two an SM (in 2, 4, 8: 1,024 tokens after 8,000 12, 12, 14 us, 2,048 after 30,000
  // 31, 27, 26).  One where all of them are few, and then the scan too.  Calls in 4 with a scan of its own, in one with it, in one
  // without: a prompt of 300 21.5, 20.9, 20.1 us, of 1,000 32.7, 31.2, 30.5, of 2,000 58.8, 58.3, 56.5; 1,024 after 8,000 127.5 in 4, 130 so.
  const int key_tiles = (a.max_length + kTile - 1) / kTile;
  const int64_t products = (int64_t)l.tiles_max * key_tiles * a.groups;
  const int chunk = products >= 32 * 16 * kSms ? 32 : products >= 8 * 2 * kSms ? 8 : products >= 4 * kSms ? 4 : 1;
  const bool scans = chunk == 1;
  // store: also clears the tickets of this call, the walks', the scans' and (where they are not the plan's) the few tokens'
  const int n_walk = l.tiles_max * a.heads, n_scan = scans ? l.tiles_max * a.groups * key_tiles : 0;
  {
    const TokenRows k{static_cast<const uint4*>(a.k), a.k_stride[0] / 8, a.k_stride[1] / 8};
    const TokenRows v{static_cast<const uint4*>(a.v), a.v_stride[0] / 8, a.v_stride[1] / 8};
    const int64_t units = (int64_t)a.total * a.heads * (D / 8);
    const unsigned blocks = (unsigned)max((int64_t)1, min((units + 255) / 256, (int64_t)8 * kSms));
    st = launch_after(store_kernel, dim3(blocks), 256, 0, s, k, v, static_cast<uint4*>(a.k_pages), static_cast<uint4*>(a.v_pages),
                static_cast<uint4*>(a.y), a.slots, a.total, a.heads, D / 8, a.num_pages, a.page_shift, walk_tickets, n_walk + n_scan,
                reinterpret_cast<unsigned int*>(a.workspace + w.own_tickets), a.plan_tickets ? 0 : l.tickets_count);
    if (st != SA_OK) return st;
  }
  PagedWalk walk{};
  walk.header = a.work;
  walk.items = reinterpret_cast<const TileItem*>(a.work + l.tile_items);
  walk.tables = a.block_tables;
  walk.heads = a.heads; walk.max_pages = a.max_pages; walk.page_shift = a.page_shift; walk.box_rows = box_rows;
  walk.key_stride = w.key_stride;
  walk.tickets = walk_tickets;
  walk.part = a.workspace + w.part;
  walk.lse = a.workspace + w.lse;
  const TileItem* tiles = reinterpret_cast<const TileItem*>(a.work + l.tiles);
  float* carry = a.workspace + w.carry;
  const float scale = 1.0f / sqrtf((float)D);
  const History history{a.selected, a.sel_stride, scans ? walk_tickets + n_walk : nullptr};
  {
    ProfileScope prof(SA_KERNEL_TC_COLSUM, s);
    const dim3 grid(l.tiles_max, (key_tiles + chunk - 1) / chunk, a.groups);
    st = launch_after(colsum_pages_kernel<D>, grid, 160, 3 * DK * kRowTile + 1024, s, map_q, map_k, carry, a.exempt, scale, status, chunk,
                      tiles, walk, history);
    if (st != SA_OK) return st;
    *moved = scans;
  }
  if (!scans) {
    ProfileScope prof(SA_KERNEL_TC_SCAN, s);
    st = launch_after(scan_pages_kernel, dim3((a.max_length + 255) / 256, a.groups, a.rows), 256, 0, s, carry, w.key_stride,
                      (const int*)(a.work + l.tile_start), tiles, a.groups, history);
    if (st != SA_OK) return st;
    *moved = true;
  }
  // The plan's numbers are on the device: the host goes by the tiles that there are at least, and by the items that there can be.
  // (A CTA without an item takes an SM for a microsecond.)
  const int items_max = (int)min((int64_t)l.tile_items_max, (int64_t)l.tiles_max * ((key_tiles + paged::kPieceTiles - 1) / paged::kPieceTiles));
  // (Either kernel is right whatever the plan has: one that knows no pieces takes a whole walk for each of them.)  At least: all tokens
  // in full tiles, or one for each row of more than a few, of which none has more than max_count.
  const int tiles_min = max((a.total - (a.rows - 1) + kTile - 1) / kTile, (a.total - paged::kFewTokens * a.rows) / (a.max_count - paged::kFewTokens));
  ProfileScope prof(SA_KERNEL_TC_FORWARD, s);
  __nv_bfloat16* y = static_cast<__nv_bfloat16*>(a.y);
  const RowLayout y_rows{0, D, (int64_t)a.heads * D};
  if constexpr (D == 64) {
    if (!self && a.heads % 2 == 0 && two_heads(a.rows, tiles_min, key_tiles, a.heads))
      return launch_after(forward_pair_kernel<false, true>, dim3((unsigned)items_max * (a.heads / 2)), kThreads, PairSmem::total, s,
                    map_q, map_k, map_v, map_q, map_k, (const float*)carry, (float*)nullptr, (float*)nullptr, a.heads, 0, 0, a.exempt, scale,
                    status, y, y_rows, 0, (const uint8_t*)nullptr, walk);
  }
  if (D == 64 && self && a.heads % 2 == 0 && two_heads(a.rows, tiles_min, key_tiles, a.heads))
    return forward_self_pages(walk, map_q, map_k, map_v, carry, items_max, a.exempt, scale, status, y, y_rows, s);
  auto wide = [&](auto kernel) {
    const dim3 grid((unsigned)items_max * a.heads);
    return launch_after(kernel, grid, kWidePagedThreads, WideSmem<D>::total + 1024, s, map_q, map_k, map_v, map_q, map_k, (const float*)carry,
                  (float*)nullptr, (float*)nullptr, a.heads, 0, 0, a.exempt, scale, status, y, y_rows, 0, (const uint8_t*)nullptr,
                  SplitWalk{}, walk);
  };
  const bool whole = tiles_min >= paged::tile_wave(a.heads);
  if (self) return whole ? wide(forward_wide_kernel<D, true, false, false, true>) : wide(forward_wide_kernel<D, true, false, true, true>);
  return whole ? wide(forward_wide_kernel<D, false, false, false, true>) : wide(forward_wide_kernel<D, false, false, true, true>);
}

}  // namespace
}  // namespace tc

namespace paged {

AttentionScratch attention_scratch(const Attention& a) {
  const StepLayout l = step_layout(a.rows, a.total, a.heads);
  AttentionScratch w{};
  w.key_stride = ((int64_t)a.max_length + 127) / 128 * 128;
  auto take = [&](size_t n) {
    const size_t at = w.floats;
    w.floats += (n + 63) / 64 * 64;
    return at;
  };
  w.own_tickets = take((size_t)l.tickets_count);
  w.partial = take((size_t)l.decode_items_max * a.heads * min(a.max_count, paged::kFewTokens) * (a.head_dim + 2));
  w.sel_new = take(a.groups < a.heads ? (size_t)a.rows * a.groups * w.key_stride : 0);
  if (!few_only(a.total, a.max_count) && l.tiles_max > 0) {
    w.carry = take((size_t)l.tiles_max * a.groups * w.key_stride);
    const size_t cut = (size_t)kTileWaves * tile_wave(a.heads) * a.heads * kTile;      // the plan cuts walks into no more pieces than that
    w.part = take(cut * a.head_dim);
    w.lse = take(cut);
    w.tickets = take((size_t)l.tiles_max * a.heads + (size_t)l.tiles_max * a.groups * (w.key_stride / kTile));      // the walks', the scans'
  }
  return w;
}

int tiles(const Attention& a, bool* moved, cudaStream_t s) {
  return a.head_dim == 64 ? tc::tiles_impl<64>(a, moved, s) : a.head_dim == 128 ? tc::tiles_impl<128>(a, moved, s) : SA_ERR_UNSUPPORTED;
}

int restore_histories(const Attention& a, cudaStream_t s) {
  const StepLayout l = step_layout(a.rows, a.total, a.heads);
  const AttentionScratch w = attention_scratch(a);
  count_launch();
  tc::restore_kernel<<<dim3((a.max_length + 255) / 256, a.groups, a.rows), 256, 0, s>>>(
      a.workspace + w.carry, w.key_stride, a.work + l.tile_start, reinterpret_cast<const TileItem*>(a.work + l.tiles), a.groups, a.selected,
      a.sel_stride);
  SA_CUDA_CHECK(cudaGetLastError());
  return SA_OK;
}

}  // namespace paged
}  // namespace sa
