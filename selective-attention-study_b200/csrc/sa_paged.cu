// Tables of a paged cache (sm_100a): pages handed out to rows, block tables, slots of new tokens, the plan of a step's
// attention; rows that become copies of other rows.  Whole-number work, bound by latency.
//
// State, shared by every layer of a model: block_tables [rows][max_pages] (page of a row's block, -1: none), lengths [rows],
// page_refs [num_pages] (rows that hold a page), and the free pages as a list of which the last free_count are taken from the
// end.  Nothing depends on the order in which threads run.
#include <cooperative_groups.h>

#include "sa_paged.cuh"
#include "sa_tc_ptx.cuh"

namespace sa {
namespace paged {
namespace {

namespace cg = cooperative_groups;

// Exclusive sums of N numbers over the threads of a CTA; `total` receives the sums of all.  `warp_sums`: N x 32 in shared memory.
template <int N>
__device__ __forceinline__ void block_scan(long long (&x)[N], long long (&total)[N], long long (*warp_sums)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  long long own[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    own[n] = x[n];
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x[n], s);
      if (lane >= s) x[n] += y;
    }
    if (lane == 31) warp_sums[n][warp] = x[n];
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      long long v = lane < warps ? warp_sums[n][lane] : 0;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, v, s);
        if (lane >= s) v += y;
      }
      warp_sums[n][lane] = v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    total[n] = warp_sums[n][31];
    x[n] += (warp > 0 ? warp_sums[n][warp - 1] : 0) - own[n];
  }
  __syncthreads();                                              // warp_sums may be written again
}

// The last r in [0, n) with first[r] <= x (first[0] <= x): of rows without anything the one after them is found.
template <typename P>
__device__ __forceinline__ int row_of(P first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int64_t slot_of(const Tables& t, int row, int position) {
  const int page = t.block_tables[(int64_t)row * t.max_pages + (position >> t.page_shift)];
  return ((int64_t)page << t.page_shift) + (position & ((1 << t.page_shift) - 1));
}

struct Append {
  Tables t;
  const int* counts;
  int total, max_length, max_count, least_tokens, wave_tiles, wave_decode, slots_inside;
  int *query_start, *cached;
  int64_t* slots;
  int* work;
  StepLayout layout;
};

// One CTA: PER rows a thread, a handful of prefix sums over the rows (tokens, pages, tiles, pieces), and everything that is
// per page, per tile or per token spread over the threads by a search in those sums.  What it takes is the chain of dependent
// loads, sums and barriers.  Slots of a long step are written by a second kernel
// (slots_kernel): one SM stores about 60 GB/s of them.
template <int PER>
__global__ void __launch_bounds__(1024) append_kernel(const __grid_constant__ Append a) {
  const Tables& t = a.t;
  extern __shared__ int rows_s[];
  __shared__ long long warp_sums[4][32];
  int* start_s = rows_s;                       // rows + 1: first token
  int* page_s = start_s + t.rows + 1;          // rows + 1: pages that the rows before take
  int* tile_s = page_s + t.rows + 1;           // rows + 1: tiles
  int* piece_s = tile_s + t.rows + 1;          // rows + 1: pieces of single tokens
  int* before_s = piece_s + t.rows + 1;        // rows: tokens before the step; -1 where the row is left as it is
  const int tid = threadIdx.x, step = blockDim.x;
  const int r0 = tid * PER;
  const int64_t limit = min((int64_t)t.max_pages << t.page_shift, (int64_t)a.max_length);
  const int page_mask = (1 << t.page_shift) - 1;

  for (int i = tid; i < a.layout.tickets_count; i += step) a.work[a.layout.tickets + i] = 0;
  int count[PER], before[PER];
  long long sum[1] = {0}, total[1];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = r0 + u;
    count[u] = r < t.rows ? max(a.counts[r], 0) : 0;
    before[u] = r < t.rows ? t.lengths[r] : 0;
    sum[0] += count[u];
  }
  block_scan<1>(sum, total, warp_sums);
  // ---- which rows fit, and the pages that they need -----------------------------------------------------------------------
  bool fits[PER];
  int need[PER];
  long long pages[1] = {0}, pages_total[1];
  {
    long long at = sum[0];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = r0 + u;
      if (r < t.rows) start_s[r] = (int)min(at, (long long)a.total);
      at += count[u];
      fits[u] = r < t.rows && at <= a.total && count[u] <= a.max_count && before[u] >= 0 && (int64_t)before[u] + count[u] <= limit;
      need[u] = fits[u] ? ((before[u] + count[u] + page_mask) >> t.page_shift) - ((before[u] + page_mask) >> t.page_shift) : 0;
      pages[0] += need[u];
    }
  }
  const int free_count = min(max(*t.free_count, 0), t.num_pages);
  block_scan<1>(pages, pages_total, warp_sums);
  long long next[4] = {0, 0, 0, 0}, next_total[4];    // tiles, key tiles of their walks, single tokens, their keys
  {
    long long upto = pages[0];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = r0 + u;
      if (r < t.rows) page_s[r] = (int)min(upto, (long long)t.num_pages + 1);
      upto += need[u];
      if (need[u] > 0 && upto > free_count) fits[u] = false;    // and every later row that needs a page
      if (r < t.rows) {
        before_s[r] = fits[u] ? before[u] : -1;
        a.cached[r] = fits[u] ? before[u] : -1;
        if (fits[u] && count[u] > 0) t.lengths[r] = before[u] + count[u];
      }
      if (!fits[u]) count[u] = 0;
      if (count[u] > 0 && count[u] < a.least_tokens) {
        next[2] += 1;
        next[3] += before[u] + 1;
      } else if (count[u] > 0) {
        const long long first = before[u] / kTile, last = (before[u] + count[u] - 1) / kTile;
        next[0] += last - first + 1;
        next[1] += (last - first + 1) * (first + last + 2) / 2;
      }
    }
  }
  if (tid == 0) {
    start_s[t.rows] = (int)min(total[0], (long long)a.total);
    page_s[t.rows] = (int)min(pages_total[0], (long long)t.num_pages + 1);
  }
  block_scan<4>(next, next_total, warp_sums);
  const int n_tiles = (int)next_total[0];
  {
    int at = (int)next[0];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = r0 + u;
      if (r < t.rows) {
        tile_s[r] = at;
        a.work[a.layout.tile_start + r] = at;
      }
      if (count[u] >= a.least_tokens) at += (before[u] + count[u] - 1) / kTile - before[u] / kTile + 1;
    }
    if (tid == 0) {
      tile_s[t.rows] = n_tiles;
      a.work[a.layout.tile_start + t.rows] = n_tiles;
    }
  }
  // ---- pieces of single tokens: about one wave of CTAs over all heads, or several where rows alone are more than that --------
  const int singles = (int)next_total[2];
  int piece_keys = kTile;
  if (singles > 0) {
    const int spread = 2 * singles <= a.wave_decode ? a.wave_decode - singles : kDecodeWaves * a.wave_decode;
    const long long keys = (next_total[3] + spread - 1) / spread;
    piece_keys = (int)max((long long)kTile, (keys + kTile - 1) / kTile * kTile);
  }
  long long pieces[1] = {0}, pieces_total[1] = {0};
  if (singles > 0) {
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (count[u] > 0 && count[u] < a.least_tokens) pieces[0] += before[u] / piece_keys + 1;
    block_scan<1>(pieces, pieces_total, warp_sums);
    int at = (int)pieces[0];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = r0 + u;
      if (r < t.rows) piece_s[r] = at;
      if (count[u] > 0 && count[u] < a.least_tokens) at += before[u] / piece_keys + 1;
    }
    if (tid == 0) piece_s[t.rows] = (int)pieces_total[0];
  }
  for (int i = tid; i <= t.rows; i += step) a.query_start[i] = start_s[i];
  __syncthreads();                                               // the sums, and who is served
  // ---- pages, off the end of the free list -------------------------------------------------------------------------------------
  const int wanted = min(page_s[t.rows], free_count);             // of the rows that are served: those up to the first that is not
  int taken = 0;
  for (int k = tid; k < wanted; k += step) {
    const int r = row_of(page_s, t.rows, k);
    if (before_s[r] < 0) continue;
    const int block = ((before_s[r] + page_mask) >> t.page_shift) + k - page_s[r];
    const int page = t.free_pages[free_count - 1 - k];
    t.block_tables[(int64_t)r * t.max_pages + block] = page;
    if (page >= 0 && page < t.num_pages) atomicAdd(t.page_refs + page, 1);
    ++taken;
  }
  taken = __reduce_add_sync(0xffffffffu, taken);
  if ((tid & 31) == 0 && taken > 0) atomicSub(t.free_count, taken);
  // ---- the plan: tiles (a row's first tile first), walks over their keys (the longest of a row first), pieces ------------------
  TileItem* tiles = reinterpret_cast<TileItem*>(a.work + a.layout.tiles);
  TileItem* items = reinterpret_cast<TileItem*>(a.work + a.layout.tile_items);
  DecodeItem* singles_out = reinterpret_cast<DecodeItem*>(a.work + a.layout.decode_items);
  auto tile_at = [&](int i, TileItem* x) {
    const int r = row_of(tile_s, t.rows, i);
    x->row = r; x->token = start_s[r];
    x->mi = before_s[r] / kTile + i - tile_s[r];
    x->tile = i;
    x->cached = before_s[r];
    x->length = before_s[r] + start_s[r + 1] - start_s[r];
    return r;
  };
  // Few tiles: their walks are cut so that all heads together fill the GPU.  A piece takes at least four key tiles.
  const bool cut = n_tiles > 0 && 2 * n_tiles <= a.wave_tiles;
  int n_items = n_tiles;
  if (cut) {
    const long long per = (next_total[1] + (a.wave_tiles - n_tiles) - 1) / (a.wave_tiles - n_tiles);
    const int piece_tiles = (int)max(4LL, per);
    TileItem x{};
    long long parts[1] = {0}, parts_total[1];
    if (tid < n_tiles) {                                          // at most half a wave of 148
      tile_at(tid, &x);
      tiles[tid] = x;
      x.pieces = (x.mi + piece_tiles) / piece_tiles;
      parts[0] = x.pieces;
    }
    block_scan<1>(parts, parts_total, warp_sums);
    n_items = (int)parts_total[0];
    if (tid < n_tiles)
      for (x.piece = 0; x.piece < x.pieces; ++x.piece) items[parts[0] + x.piece] = x;
  } else {
    for (int i = tid; i < n_tiles; i += step) {
      TileItem x{};
      tile_at(i, &x);
      tiles[i] = x;
      x.pieces = 1;
      items[n_tiles - 1 - i] = x;
    }
  }
  const int n_single = (int)pieces_total[0];
  for (int i = tid; i < n_single; i += step) {
    const int r = row_of(piece_s, t.rows, i);
    DecodeItem x;
    x.row = r; x.token = start_s[r];
    x.first = piece_s[r];
    x.piece = i - x.first;
    x.pieces = piece_s[r + 1] - x.first;
    x.length = before_s[r] + 1;
    x.c0 = x.piece * piece_keys;
    x.c1 = min(x.c0 + piece_keys, x.length);
    singles_out[i] = x;
  }
  if (tid == 0) {
    a.work[kTiles] = n_tiles;
    a.work[kTileItems] = n_items;
    a.work[kDecodeItems] = n_single;
  }
  if (!a.slots_inside) return;
  __syncthreads();                                               // the new pages are in the tables
  for (int i = tid; i < a.total; i += step) {
    const int r = row_of(start_s, t.rows, i);
    const bool in = i < start_s[t.rows] && before_s[r] >= 0;
    a.slots[i] = in ? slot_of(t, r, before_s[r] + i - start_s[r]) : -1;
  }
}

__global__ void __launch_bounds__(256) slots_kernel(Tables t, int total, const int* __restrict__ query_start,
                                                    const int* __restrict__ cached, int64_t* __restrict__ slots) {
  tc::after_previous_kernel();
  extern __shared__ int rows_s[];                                // query_start
  for (int i = threadIdx.x; i <= t.rows; i += blockDim.x) rows_s[i] = query_start[i];
  __syncthreads();
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += gridDim.x * blockDim.x) {
    const int r = row_of(rows_s, t.rows, i);
    const int before = cached[r];
    slots[i] = i < rows_s[t.rows] && before >= 0 ? slot_of(t, r, before + i - rows_s[r]) : -1;
  }
}
constexpr int kSlotsInside = 2048;

// ---- rows that become copies of other rows ------------------------------------------------------------------------------------
// Row r becomes a copy of row parents[r] (outside [0, rows): an empty row).  Full pages are shared.  The page that is being
// filled stays with the lowest child; the others get a page of their own, and `copies` says what has to be copied into it.
//
// One cluster of eight CTAs, in four passes with a cluster barrier between: (1) the new tables into scratch, a reference more
// for each page of a new row (a page that old and new row have at the same place counts for neither); (2) a reference less for
// each page of an old row, marking those that nobody holds; (3) one CTA puts the marked pages on the free list, lowest first,
// and takes the pages for the copies off its end, in row order; (4) the tables.  A row for which there is none becomes empty (its
// full pages are shared with the lowest child, so nothing else is freed).
constexpr int kCluster = 8, kReorderThreads = 512;

// The work of a reordering, int32 words: how many rows change, then (row, parent, tokens, tokens of the page being filled) of
// each | a word a row | a bit a page | the new tables.
struct ReorderWork {
  size_t moved, info, marks, scratch, words;
  ReorderWork(int rows, int max_pages, int num_pages) {
    size_t at = 4;
    moved = 0;
    at += 4 * (size_t)rows;
    info = at;
    at += (rows + 3) / 4 * 4;
    marks = at;
    at += ((size_t)num_pages + 31) / 32 / 4 * 4 + 4;
    scratch = at;
    at += (size_t)rows * max_pages;
    words = at;
  }
};

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kReorderThreads)
    reorder_kernel(Tables t, const int* __restrict__ parents, int* copies, int* moved, int* info, unsigned* marks, int* scratch) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ long long warp_sums[2][32];
  const int tid = threadIdx.x, cta = (int)cluster.block_rank();
  const int all = kCluster * kReorderThreads, me = cta * kReorderThreads + tid;
  const int lane = tid & 31, warp = me >> 5, warps = all >> 5;
  const int page_mask = (1 << t.page_shift) - 1;
  const int words = (t.num_pages + 31) / 32;
  auto length_of = [&](int r) { return min(max(t.lengths[r], 0), t.max_pages << t.page_shift); };
  auto parent_of = [&](int r) {
    const int p = parents[r];
    return p >= 0 && p < t.rows ? p : -1;
  };
  auto real = [&](int page) { return page >= 0 && page < t.num_pages; };

  for (int i = me; i < words; i += all) marks[i] = 0u;
  // (1) a warp a row
  for (int r = warp; r < t.rows; r += warps) {
    const int p = parent_of(r);
    const int len = p >= 0 ? length_of(p) : 0, full = len >> t.page_shift;
    const bool part = (len & page_mask) != 0;
    bool fresh = false;
    if (part) {                                                   // a lower child of the same parent has the page already
      for (int c0 = 0; c0 < r && !fresh; c0 += 32) fresh = __any_sync(0xffffffffu, c0 + lane < r && parents[c0 + lane] == p);
    }
    const int* from = t.block_tables + (int64_t)max(p, 0) * t.max_pages;
    const int* was = t.block_tables + (int64_t)r * t.max_pages;
    const int held = (length_of(r) + page_mask) >> t.page_shift;
    int* to = scratch + (int64_t)r * t.max_pages;
    const int blocks = full + (part ? 1 : 0);
    for (int b = lane; b < t.max_pages; b += 32) {
      const int page = b < blocks ? from[b] : -1;
      to[b] = page;
      const bool counts = b < full || (b < blocks && !fresh);
      if (counts && real(page) && !(b < held && was[b] == page)) atomicAdd(t.page_refs + page, 1);
    }
    if (lane == 0) info[r] = fresh ? 1 : 0;
  }
  __threadfence();
  cluster.sync();
  // (2)
  for (int r = warp; r < t.rows; r += warps) {
    const int held = (length_of(r) + page_mask) >> t.page_shift;
    const int p = parent_of(r), len = p >= 0 ? length_of(p) : 0, full = len >> t.page_shift;
    const int blocks = full + ((len & page_mask) != 0 && __ldcg(info + r) == 0 ? 1 : 0);
    const int* was = t.block_tables + (int64_t)r * t.max_pages;
    const int* now = scratch + (int64_t)r * t.max_pages;
    for (int b = lane; b < held; b += 32) {
      const int page = was[b];
      if (!real(page) || (b < blocks && __ldcg(now + b) == page)) continue;
      if (atomicSub(t.page_refs + page, 1) == 1) atomicOr(marks + (page >> 5), 1u << (page & 31));
    }
  }
  __threadfence();
  cluster.sync();
  // (3)
  if (cta == 0) {
    int count = min(max(*t.free_count, 0), t.num_pages);
    for (int w0 = 0; w0 < words; w0 += kReorderThreads) {
      const int w = w0 + tid;
      unsigned bits = w < words ? __ldcg(marks + w) : 0u;
      long long n[1] = {__popc(bits)}, total[1];
      block_scan<1>(n, total, warp_sums);
      for (int at = count + (int)n[0]; bits != 0u && at < t.num_pages; bits &= bits - 1u, ++at) t.free_pages[at] = w * 32 + __ffs(bits) - 1;
      count = min(count + (int)total[0], t.num_pages);
    }
    __syncthreads();                                              // the list
    int used = 0, n_moved = 0;
    for (int c0 = 0; c0 < t.rows; c0 += kReorderThreads) {
      const int r = c0 + tid;
      const int p = r < t.rows ? parent_of(r) : -1;
      const int len = p >= 0 ? length_of(p) : 0, full = len >> t.page_shift;
      const bool fresh = r < t.rows && __ldcg(info + r) != 0;
      const bool changes = len > 0 && (p != r || fresh);
      long long n[2] = {fresh ? 1 : 0, changes ? 1 : 0}, total[2];
      block_scan<2>(n, total, warp_sums);
      int src = -1, dst = -1;
      bool dropped = false;
      if (fresh) {
        const int k = used + (int)n[0];
        int* to = scratch + (int64_t)r * t.max_pages;
        if (k < count) {
          src = __ldcg(to + full);
          dst = t.free_pages[count - 1 - k];
          to[full] = dst;
          if (real(dst)) atomicAdd(t.page_refs + dst, 1);
        } else {                                                  // out of pages: the row becomes empty
          dropped = true;
          for (int b = 0; b <= full; ++b) {
            const int page = __ldcg(to + b);
            if (b < full && real(page)) atomicSub(t.page_refs + page, 1);
            to[b] = -1;
          }
        }
      }
      if (r < t.rows) {
        copies[2 * r] = src;
        copies[2 * r + 1] = dst;
        info[r] = dropped ? 0 : len;                              // the row's new length
        if (changes)
          reinterpret_cast<int4*>(moved)[1 + n_moved + n[1]] = make_int4(r, p, dropped ? 0 : len, fresh && !dropped ? len & page_mask : 0);
      }
      used += (int)total[0];
      n_moved += (int)total[1];
    }
    if (tid == 0) {
      *t.free_count = count - min(used, count);
      moved[0] = n_moved;
    }
  }
  __threadfence();
  cluster.sync();
  // (4)
  for (int r = me; r < t.rows; r += all) t.lengths[r] = __ldcg(info + r);
  const int64_t n = (int64_t)t.rows * t.max_pages;
  for (int64_t i = me; i < n; i += all) t.block_tables[i] = __ldcg(scratch + i);
}

// The history of the rows of `moved`: a CTA gathers 4 UNITS keys of one group over all rows, through shared memory, since a row
// can be read and written: first everything is read, then everything is written.
template <int UNITS>
__global__ void __launch_bounds__(256) move_history_kernel(const int4* __restrict__ moved, float* selected, int groups, int64_t capacity) {
  tc::after_previous_kernel();
  extern __shared__ float4 keep[];
  const int n = moved[0].x, g = blockIdx.y, unit = threadIdx.x % UNITS;
  const int64_t j = ((int64_t)blockIdx.x * UNITS + unit) * 4;       // capacity is a multiple of 16: whole units
  for (int m = threadIdx.x / UNITS; m < n; m += 256 / UNITS) {
    const int4 x = moved[1 + m];
    if (j < x.z && j < capacity) keep[m * UNITS + unit] = *reinterpret_cast<const float4*>(selected + ((int64_t)x.y * groups + g) * capacity + j);
  }
  __syncthreads();
  for (int m = threadIdx.x / UNITS; m < n; m += 256 / UNITS) {
    const int4 x = moved[1 + m];
    if (j >= x.z || j >= capacity) continue;
    const float4 v = keep[m * UNITS + unit];
    float* to = selected + ((int64_t)x.x * groups + g) * capacity + j;
    if (j + 4 <= x.z) {
      *reinterpret_cast<float4*>(to) = v;
    } else {                                                      // behind the row's last token nothing is written
      to[0] = v.x;
      if (j + 1 < x.z) to[1] = v.y;
      if (j + 2 < x.z) to[2] = v.z;
    }
  }
}

// The tokens of the pages that are being filled, into the pages that their copies got.
__global__ void __launch_bounds__(256) move_pages_kernel(const int4* __restrict__ moved, const int2* __restrict__ copies, uint4* k_pages,
                                                         uint4* v_pages, int heads, int num_pages, int64_t head_units, int row_units) {
  tc::after_previous_kernel();
  const int n = moved[0].x;
  const int64_t page_units = head_units * heads;
  for (int m = blockIdx.x; m < n; m += gridDim.x) {
    const int4 x = moved[1 + m];
    if (x.w == 0) continue;
    const int2 c = copies[x.x];
    if (c.x < 0 || c.x >= num_pages || c.y < 0 || c.y >= num_pages) continue;
    const int units = x.w * row_units;                            // of one head
    uint4* pool = blockIdx.y == 0 ? k_pages : v_pages;
    const uint4* from = pool + c.x * page_units;
    uint4* to = pool + c.y * page_units;
    for (int i = blockIdx.z * blockDim.x + threadIdx.x; i < units * heads; i += gridDim.z * blockDim.x) {
      const int h = i / units, u = i - h * units;
      to[h * head_units + u] = from[h * head_units + u];
    }
  }
}

template <typename... Args>
int launch_after(void (*kernel)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = s;
  config.attrs = &attr;
  config.numAttrs = 1;
  count_launch();
  SA_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, args...));
  return SA_OK;
}

}  // namespace

int append(const Tables& t, const int* counts, int total, int max_length, int max_count, int* query_start, int* cached, int64_t* slots,
           int* work, cudaStream_t s) {
  Append a{};
  a.t = t;
  a.counts = counts;
  a.total = total; a.max_length = max_length; a.max_count = max_count;
  a.least_tokens = tile_tokens(t.rows, total, max_count);
  a.wave_tiles = tile_wave(t.heads);
  a.wave_decode = decode_wave(t.heads);
  a.slots_inside = total <= kSlotsInside;
  a.query_start = query_start; a.cached = cached; a.slots = slots; a.work = work;
  a.layout = step_layout(t.rows, total, t.heads);
  const size_t smem = (5 * (size_t)t.rows + 4) * 4;
  auto launch = [&](auto kernel, int threads) -> int {
    SA_CUDA_CHECK(allow_smem(kernel, smem));
    count_launch();
    kernel<<<1, threads, smem, s>>>(a);
    SA_CUDA_CHECK(cudaGetLastError());
    return SA_OK;
  };
  // 256 threads where they cover rows and tokens: barriers and sums over eight warps are shorter than over thirty-two
  const int st = t.rows <= 256 && total <= 256 ? launch(append_kernel<1>, 256)
                 : t.rows <= 1024              ? launch(append_kernel<1>, 1024)
                                               : launch(append_kernel<kMaxRows / 1024>, 1024);
  if (st != SA_OK || a.slots_inside) return st;
  const unsigned blocks = (unsigned)min((total + 255) / 256, 4 * kSms);
  return launch_after(slots_kernel, dim3(blocks), 256, ((size_t)t.rows + 1) * 4, s, t, total, (const int*)query_start, (const int*)cached, slots);
}

size_t reorder_work_words(int rows, int max_pages, int num_pages) { return ReorderWork(rows, max_pages, num_pages).words; }

int reorder(const Tables& t, const int* parents, int* copies, int* work, cudaStream_t s) {
  const ReorderWork w(t.rows, t.max_pages, t.num_pages);
  count_launch();
  reorder_kernel<<<kCluster, kReorderThreads, 0, s>>>(t, parents, copies, work + w.moved, work + w.info,
                                                      reinterpret_cast<unsigned*>(work + w.marks), work + w.scratch);
  SA_CUDA_CHECK(cudaGetLastError());
  return SA_OK;
}

int move_rows(const Tables& t, const int* copies, const int* work, int groups, int head_dim, int elem_bytes, int64_t capacity, void* k_pages,
              void* v_pages, float* selected, cudaStream_t s) {
  const int4* moved = reinterpret_cast<const int4*>(work);
  // 32 keys a CTA (a line of every row), or 8 where the rows would not fit the shared memory
  auto history = [&](auto kernel, int units) -> int {
    const size_t smem = (size_t)t.rows * units * sizeof(float4);
    SA_CUDA_CHECK(allow_smem(kernel, smem));
    const unsigned chunks = (unsigned)((capacity + 4 * units - 1) / (4 * units));
    return launch_after(kernel, dim3(chunks, groups), 256, smem, s, moved, selected, groups, capacity);
  };
  int st = t.rows <= 1024 ? history(move_history_kernel<8>, 8) : history(move_history_kernel<2>, 2);
  if (st != SA_OK) return st;
  const int row_units = head_dim * elem_bytes / 16;
  return launch_after(move_pages_kernel, dim3(min(t.rows, 512), 2, 2), 256, 0, s, moved, reinterpret_cast<const int2*>(copies),
                      static_cast<uint4*>(k_pages), static_cast<uint4*>(v_pages), t.heads, t.num_pages,
                      (int64_t)row_units << t.page_shift, row_units);
}

}  // namespace paged
}  // namespace sa
