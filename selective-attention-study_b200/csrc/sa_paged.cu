// Tables of a paged cache (sm_100a): pages handed out to rows, block tables, slots of new tokens, the plan of a step's
// attention; rows that become copies of other rows.  Whole-number work, bound by latency.
//
// State, shared by every layer of a model: block_tables [rows][max_pages] (page of a row's block, -1: none), lengths [rows],
// page_refs [num_pages] (rows that hold a page), and the free pages as a list of which the last free_count are taken from the
// end.  Nothing depends on the order in which threads run.
#include <cooperative_groups.h>

#include <type_traits>

#include "sa_paged.cuh"
#include "sa_tc_ptx.cuh"

namespace sa {
namespace paged {
namespace {

namespace cg = cooperative_groups;

// Exclusive sums of N numbers over the threads of a CTA; `total` receives the sums of all.  `warp_sums`: 32 of each in shared
// memory.
template <int N, typename S>
__device__ __forceinline__ void block_scan(S (&x)[N], S (&total)[N], S (*warp_sums)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  S own[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    own[n] = x[n];
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const S y = __shfl_up_sync(0xffffffffu, x[n], s);
      if (lane >= s) x[n] += y;
    }
    if (lane == 31) warp_sums[n][warp] = x[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {                                 // every warp adds up the warps before it
    S v = lane < warps ? warp_sums[n][lane] : 0;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const S y = __shfl_up_sync(0xffffffffu, v, s);
      if (lane >= s) v += y;
    }
    total[n] = __shfl_sync(0xffffffffu, v, 31);
    const S before = __shfl_sync(0xffffffffu, v, max(warp - 1, 0));
    x[n] += (warp > 0 ? before : 0) - own[n];
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

struct Append {
  Tables t;
  const int* counts;
  int total, max_length, max_count, least_tokens, wave_tiles, wave_decode, inside;
  int *query_start, *cached;
  int64_t* slots;
  int* work;
  StepLayout layout;
};
// Sums over the rows before a row (rows + 1 each): tokens, pages that they take, tiles, pieces of rows of few tokens; and the tokens that
// a row has (-1: it is left as it is).
struct RowSums {
  int *start, *page, *tile, *piece, *before;
  __device__ __forceinline__ RowSums(int* at, int rows)
      : start(at), page(at + rows + 1), tile(at + 2 * (rows + 1)), piece(at + 3 * (rows + 1)), before(at + 4 * (rows + 1)) {}
};

// Everything that is per page, per tile or per token, by a search in the sums, and all that changes the tables (a step whose second
// launch fails leaves them as they were): the caller takes every `step`-th from `first` on.
__device__ __forceinline__ void spread(const Append& a, const RowSums& s, const int* header, int first, int step) {
  const Tables& t = a.t;
  const int page_mask = (1 << t.page_shift) - 1;
  const int free_before = header[kFreeBefore], wanted = header[kPagesWanted], n_tiles = header[kTiles], n_single = header[kDecodeItems];
  const int piece_keys = header[kPieceKeys];
  const bool cut = header[kCut] != 0;
  if (first == 0) *t.free_count = header[kFreeAfter];
  for (int r = first; r < t.rows; r += step) {
    const int count = s.start[r + 1] - s.start[r];
    if (s.before[r] >= 0 && count > 0) t.lengths[r] = s.before[r] + count;
  }
  for (int i = first; i < a.layout.tickets_count; i += step) a.work[a.layout.tickets + i] = 0;
  for (int k = first; k < wanted; k += step) {                    // off the end of the free list
    const int r = row_of(s.page, t.rows, k);
    if (s.before[r] < 0) continue;                                // the first row that did not fit
    const int block = ((s.before[r] + page_mask) >> t.page_shift) + k - s.page[r];
    const int page = t.free_pages[free_before - 1 - k];
    t.block_tables[(int64_t)r * t.max_pages + block] = page;
    if (page >= 0 && page < t.num_pages) atomicAdd(t.page_refs + page, 1);
  }
  const int run = a.total > step ? 4 : 1;                          // of tokens: one search, and most often one page (512 rows: 22.5 -> 20.5 us)
  for (int i0 = run * first; i0 < a.total; i0 += run * step) {
    int r = row_of(s.start, t.rows, i0), block_was = -1, page = -1;
    const int i1 = min(i0 + run, a.total);
    for (int i = i0; i < i1; ++i) {
      if (i >= s.start[r + 1]) {
        r = row_of(s.start, t.rows, i);                            // (there may be many empty rows between)
        block_was = -1;
      }
      int64_t slot = -1;
      if (i < s.start[t.rows] && s.before[r] >= 0) {
        const int position = s.before[r] + i - s.start[r], block = position >> t.page_shift;
        if (block != block_was) {
          const int fresh = block - ((s.before[r] + page_mask) >> t.page_shift);  // of the row's new pages
          page = fresh >= 0 ? t.free_pages[free_before - 1 - (s.page[r] + fresh)] : t.block_tables[(int64_t)r * t.max_pages + block];
          block_was = block;
        }
        slot = ((int64_t)page << t.page_shift) + (position & page_mask);
      }
      a.slots[i] = slot;
    }
  }
  // tiles (a row's first tile first), and walks over their keys, the longest of all rows first: a CTA each, taken in this order
  // (a warp a tile: its place is the number of longer walks, and of equal ones of earlier rows)
  for (int i = first >> 5; i < n_tiles && !cut; i += step >> 5) {
    const int r = row_of(s.tile, t.rows, i);
    const int mi = s.before[r] / kTile + i - s.tile[r];
    int at = 0;
    for (int u = first & 31; u < t.rows; u += 32) {
      const int n = s.tile[u + 1] - s.tile[u];
      if (n == 0) continue;
      const int from = s.before[u] / kTile, beyond = from + n - 1 - mi;      // tiles of row u behind tile mi of its own
      at += max(0, min(n, beyond)) + (u < r && from <= mi && beyond >= 0 ? 1 : 0);
    }
    at = __reduce_add_sync(0xffffffffu, at);
    if ((first & 31) != 0) continue;
    const TileItem x{r, s.start[r], mi, i, 0, 1, s.before[r], s.before[r] + s.start[r + 1] - s.start[r]};
    reinterpret_cast<TileItem*>(a.work + a.layout.tiles)[i] = x;
    reinterpret_cast<TileItem*>(a.work + a.layout.tile_items)[at] = x;
  }
  for (int i = first; i < n_single; i += step) {
    const int r = row_of(s.piece, t.rows, i);
    DecodeItem x;
    const int count = s.start[r + 1] - s.start[r];
    x.row = (short)r; x.count = (short)count; x.token = s.start[r];
    x.first = s.piece[r];
    x.piece = i - x.first;
    x.pieces = s.piece[r + 1] - x.first;
    x.length = s.before[r] + count;
    x.c0 = x.piece * piece_keys;
    x.c1 = min(x.c0 + piece_keys, x.length);
    reinterpret_cast<DecodeItem*>(a.work + a.layout.decode_items)[i] = x;
  }
}

// One CTA: PER rows a thread and four prefix sums over the rows; what is per page, tile or token (spread) here too where that is
// little, else in a second kernel of many CTAs (512 rows with 264,000 tokens and 16,800 pages: 6 + 12 us; in one CTA 48).  Bound by
// the chain of dependent loads, sums and barriers: 64 rows of one token 7 us.  S: 32 bits where no sum can pass them.
template <int PER, typename S>
__global__ void __launch_bounds__(1024) append_kernel(const __grid_constant__ Append a) {
  const Tables& t = a.t;
  extern __shared__ int rows_s[];
  __shared__ S warp_sums[4][32];
  __shared__ int header[kHeaderWords];
  __shared__ int mi_s[kSms];                     // tiles whose walks are cut
  const RowSums sums(rows_s, t.rows);
  const int tid = threadIdx.x;
  const int r0 = tid * PER;
  const int64_t limit = min((int64_t)t.max_pages << t.page_shift, (int64_t)a.max_length);
  const int page_mask = (1 << t.page_shift) - 1;

  int count[PER], before[PER];
  S sum[1] = {0}, total[1];
  const int free_count = min(max(*t.free_count, 0), t.num_pages);
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int r = r0 + u;
    count[u] = r < t.rows ? min(max(a.counts[r], 0), a.total + 1) : 0;
    before[u] = r < t.rows ? t.lengths[r] : 0;
    sum[0] += count[u];
  }
  block_scan(sum, total, warp_sums);
  // ---- which rows fit, and the pages that they need -----------------------------------------------------------------------
  bool fits[PER];
  int need[PER];
  S pages[1] = {0}, pages_total[1];
  {
    S at = sum[0];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = r0 + u;
      if (r < t.rows) sums.start[r] = (int)min(at, (S)a.total);
      at += count[u];
      fits[u] = r < t.rows && at <= a.total && count[u] <= a.max_count && before[u] >= 0 && (int64_t)before[u] + count[u] <= limit;
      need[u] = fits[u] ? ((before[u] + count[u] + page_mask) >> t.page_shift) - ((before[u] + page_mask) >> t.page_shift) : 0;
      pages[0] += need[u];
    }
  }
  block_scan(pages, pages_total, warp_sums);
  S next[4] = {0, 0, 0, 0}, next_total[4];       // tiles, rows of few tokens, their keys, pages taken
  {
    S upto = pages[0];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = r0 + u;
      if (r < t.rows) sums.page[r] = (int)min(upto, (S)t.num_pages + 1);
      upto += need[u];
      if (need[u] > 0 && upto > free_count) fits[u] = false;    // and every later row that needs a page
      if (r < t.rows) {
        sums.before[r] = fits[u] ? before[u] : -1;
        a.cached[r] = fits[u] ? before[u] : -1;
      }
      if (!fits[u]) count[u] = 0;
      else next[3] += need[u];
      if (count[u] > 0 && count[u] < a.least_tokens) {
        next[1] += 1;
        next[2] += before[u] + count[u];
      } else if (count[u] > 0) {
        next[0] += (before[u] + count[u] - 1) / kTile - before[u] / kTile + 1;
      }
    }
  }
  block_scan(next, next_total, warp_sums);
  const int n_tiles = (int)next_total[0], singles = (int)next_total[1];
  // pieces of rows of few tokens: about one wave of CTAs over all heads, or several where rows alone are more than that
  int piece_keys = kTile;
  if (singles > 0) {
    const int spread_over = 2 * singles <= a.wave_decode ? a.wave_decode - singles : kDecodeWaves * a.wave_decode;
    const S keys = (next_total[2] + spread_over - 1) / spread_over;
    piece_keys = (int)max((S)kTile, (keys + kTile - 1) / kTile * kTile);
  }
  S pieces[1] = {0}, pieces_total[1] = {0};
  if (singles > 0) {
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (count[u] > 0 && count[u] < a.least_tokens) pieces[0] += (before[u] + count[u] - 1) / piece_keys + 1;
    block_scan(pieces, pieces_total, warp_sums);
  }
  // Few tiles: their walks are cut so that all heads together are one wave of CTAs.
  const bool cut = n_tiles > 0 && n_tiles < a.wave_tiles;
  {
    int tile_at = (int)next[0], piece_at = (int)pieces[0];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int r = r0 + u;
      if (r < t.rows) {
        sums.tile[r] = tile_at;
        sums.piece[r] = piece_at;
        a.work[a.layout.tile_start + r] = tile_at;
        a.query_start[r] = sums.start[r];
      }
      if (count[u] >= a.least_tokens) tile_at += (before[u] + count[u] - 1) / kTile - before[u] / kTile + 1;
      else if (count[u] > 0) piece_at += (before[u] + count[u] - 1) / piece_keys + 1;
    }
    if (tid == 0) {
      sums.start[t.rows] = a.query_start[t.rows] = (int)min(total[0], (S)a.total);
      sums.page[t.rows] = (int)min(pages_total[0], (S)t.num_pages + 1);
      sums.tile[t.rows] = a.work[a.layout.tile_start + t.rows] = n_tiles;
      sums.piece[t.rows] = (int)pieces_total[0];
      header[kTiles] = n_tiles;
      header[kTileItems] = n_tiles;
      header[kDecodeItems] = (int)pieces_total[0];
      header[kPieceKeys] = piece_keys;
      header[kPagesWanted] = min(sums.page[t.rows], free_count);     // of the rows that are served: those up to the first that is not
      header[kFreeBefore] = free_count;
      header[kFreeAfter] = free_count - (int)next_total[3];
      header[kCut] = cut;
    }
  }
  __syncthreads();                                               // the sums, and who is served
  if (cut) {                                                     // a thread a tile, fewer than 148
    TileItem x{};
    if (tid < n_tiles) {
      const int r = row_of(sums.tile, t.rows, tid);
      x = TileItem{r, sums.start[r], sums.before[r] / kTile + tid - sums.tile[r], tid, 0, 1, sums.before[r],
                   sums.before[r] + sums.start[r + 1] - sums.start[r]};
      reinterpret_cast<TileItem*>(a.work + a.layout.tiles)[tid] = x;
      mi_s[tid] = x.mi;
    }
    __syncthreads();
    if (tid < 32) {
      int longest = kPieceTiles;
      for (int u = tid; u < n_tiles; u += 32) longest = max(longest, mi_s[u] + 1);
      longest = __reduce_max_sync(0xffffffffu, longest);
      auto shortest = [&](int most) {                             // pieces, of so many items at most
        int low = kPieceTiles, high = longest;
        while (low < high) {
          const int middle = (low + high) >> 1;
          int n = 0;
          for (int u = tid; u < n_tiles; u += 32) n += (mi_s[u] + middle) / middle;
          if (__reduce_add_sync(0xffffffffu, n) <= most) high = middle;
          else low = middle + 1;
        }
        return low;
      };
      // One wave of CTAs, or two where tiles of one length leave many SMs without a piece.  A CTA's set-up takes as long as three steps.
      const int one = shortest(a.wave_tiles), two = shortest(kTileWaves * a.wave_tiles);
      if (tid == 0) header[kTileItems] = two < one && 2 * (two + 4) < one + 3 ? two : one;
    }
    __syncthreads();
    const int piece_tiles = header[kTileItems];
    S parts[1] = {0}, parts_total[1];
    if (tid < n_tiles) {
      x.pieces = (x.mi + piece_tiles) / piece_tiles;
      parts[0] = x.pieces;
    }
    block_scan(parts, parts_total, warp_sums);
    if (tid < n_tiles)
      for (x.piece = 0; x.piece < x.pieces; ++x.piece) reinterpret_cast<TileItem*>(a.work + a.layout.tile_items)[(int)parts[0] + x.piece] = x;
    if (tid == 0) header[kTileItems] = (int)parts_total[0];
    __syncthreads();
  }
  if (tid < kHeaderWords) a.work[tid] = header[tid];
  if (a.inside) {
    spread(a, sums, header, tid, blockDim.x);
  } else {
    for (int i = tid; i < 5 * (t.rows + 1) - 1; i += blockDim.x) a.work[a.layout.sums + i] = rows_s[i];
  }
}

__global__ void __launch_bounds__(256) spread_kernel(const __grid_constant__ Append a) {
  tc::after_previous_kernel();
  extern __shared__ __align__(16) int rows_s[];
  __shared__ int header[kHeaderWords];
  const int4* sums = reinterpret_cast<const int4*>(a.work + a.layout.sums);      // (in eights of words, as the layout leaves them)
  for (int i = threadIdx.x; i < (5 * (a.t.rows + 1) + 3) / 4; i += blockDim.x) reinterpret_cast<int4*>(rows_s)[i] = __ldcg(sums + i);
  if (threadIdx.x < kHeaderWords) header[threadIdx.x] = __ldcg(a.work + threadIdx.x);
  __syncthreads();
  spread(a, RowSums(rows_s, a.t.rows), header, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
}
constexpr int kInside = 2048;         // tokens of a step that one CTA writes by itself

// ---- rows that become copies of other rows ------------------------------------------------------------------------------------
// Row r becomes a copy of row parents[r] (outside [0, rows): an empty row).  Full pages are shared.  The page that is being
// filled stays with the lowest child; the others get a page of their own, and `copies` says what has to be copied into it.
//
// One cluster of eight CTAs, in passes with a cluster barrier between: (1) the new tables into scratch, a reference more for each
// page of a new row (a page that old and new row have at the same place counts for neither); (2) a reference less for each page
// of an old row, marking those that nobody holds; (3) one CTA puts the marked pages on the free list, lowest first, and takes the
// pages for the copies off its end, in row order, while (4) the others write the tables.  A row for which there is none becomes
// empty (its full pages are shared with the lowest child, so nothing else is freed).  Bound by the latency of the passes: 4 rows of 26
// or of 500 pages 8 to 9 us, 256 rows of 24 11 us; with cold caches 10, 12 and 13 to 14.
constexpr int kCluster = 8, kReorderThreads = 1024;

// The work of a reordering, int32 words: how many rows change, how many were lost for want of a page, then (row, parent, tokens,
// tokens of the page being filled) of each that changes | a word a row | a bit a page | the new tables.
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
    reorder_kernel(Tables t, int part_shift, int span, const int* __restrict__ parents, int* copies, int* moved, int* info, unsigned* marks, int* scratch) {
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ int rows_s[];
  __shared__ int warp_sums[2][32];
  int *parent_s = rows_s, *length_s = rows_s + t.rows;            // -1: none; in tokens
  const int tid = threadIdx.x, cta = (int)cluster.block_rank();
  const int all = kCluster * kReorderThreads, me = cta * kReorderThreads + tid;
  const int lane = tid & 31, warp = me >> 5, warps = all >> 5;
  const int page_mask = (1 << t.page_shift) - 1;
  const int words = (t.num_pages + 31) / 32;
  auto real = [&](int page) { return page >= 0 && page < t.num_pages; };

  for (int r = tid; r < t.rows; r += kReorderThreads) {
    const int p = parents[r];
    parent_s[r] = p >= 0 && p < t.rows ? p : -1;
    length_s[r] = min(max(t.lengths[r], 0), t.max_pages << t.page_shift);
  }
  for (int i = me; i < words; i += all) marks[i] = 0u;
  __syncthreads();
  const int units = t.rows << part_shift;                         // a warp takes a unit: `span` pages of a row
  auto first_page = [&](int unit) { return (unit & ((1 << part_shift) - 1)) * span; };
  // (1)
  for (int i = warp; i < units; i += warps) {
    const int r = i >> part_shift, b0 = first_page(i), b1 = min(b0 + span, t.max_pages);
    const int p = parent_s[r];
    const int len = p >= 0 ? length_s[p] : 0, full = len >> t.page_shift;
    const bool part = (len & page_mask) != 0;
    const int* from = t.block_tables + (int64_t)max(p, 0) * t.max_pages;
    const int* was = t.block_tables + (int64_t)r * t.max_pages;
    const int held = (length_s[r] + page_mask) >> t.page_shift;
    int* to = scratch + (int64_t)r * t.max_pages;
    bool fresh = false;                                           // a lower child of the same parent has the page already
    if (part)
      for (int c0 = 0; c0 < r && !fresh; c0 += 32) fresh = __any_sync(0xffffffffu, c0 + lane < r && parent_s[c0 + lane] == p);
    const int blocks = full + (part ? 1 : 0);
    for (int b = b0 + lane; b < b1; b += 32) {
      const int page = b < blocks ? from[b] : -1;
      to[b] = page;
      const bool counts = b < full || (b < blocks && !fresh);
      if (counts && real(page) && !(b < held && was[b] == page)) atomicAdd(t.page_refs + page, 1);
    }
    if (b0 == 0 && lane == 0) info[r] = fresh ? 1 : 0;
  }
  __threadfence();
  cluster.sync();
  // (2)
  for (int i = warp; i < units; i += warps) {
    const int r = i >> part_shift, b0 = first_page(i);
    const int held = min((length_s[r] + page_mask) >> t.page_shift, b0 + span);
    const int p = parent_s[r], len = p >= 0 ? length_s[p] : 0, full = len >> t.page_shift;
    const int blocks = full + ((len & page_mask) != 0 && __ldcg(info + r) == 0 ? 1 : 0);
    const int* was = t.block_tables + (int64_t)r * t.max_pages;
    const int* now = scratch + (int64_t)r * t.max_pages;
    for (int b = b0 + lane; b < held; b += 32) {
      const int page = was[b];
      if (!real(page) || (b < blocks && __ldcg(now + b) == page)) continue;
      if (atomicSub(t.page_refs + page, 1) == 1) atomicOr(marks + (page >> 5), 1u << (page & 31));
    }
  }
  __threadfence();
  cluster.sync();
  // (3), and (4) by the other CTAs meanwhile: all of the new tables but the pages that (3) takes
  __shared__ int dropped_s;                                       // rows for which there was no page
  if (cta != 0) {
    constexpr int first = kReorderThreads / 32;
    for (int i = warp - first; i < units; i += warps - first) {
      const int r = i >> part_shift, b0 = first_page(i), b1 = min(b0 + span, t.max_pages);
      const int p = parent_s[r], full = p >= 0 ? length_s[p] >> t.page_shift : 0;
      const bool fresh = __ldcg(info + r) != 0;
      int* to = t.block_tables + (int64_t)r * t.max_pages;
      const int* now = scratch + (int64_t)r * t.max_pages;
      for (int b = b0 + lane; b < b1; b += 32)
        if (!(fresh && b == full)) to[b] = __ldcg(now + b);
    }
  } else {
    if (tid == 0) dropped_s = 0;
    int count = min(max(*t.free_count, 0), t.num_pages);
    for (int w0 = 0; w0 < words; w0 += kReorderThreads) {
      const int w = w0 + tid;
      unsigned bits = w < words ? __ldcg(marks + w) : 0u;
      int n[1] = {__popc(bits)}, total[1];
      block_scan(n, total, warp_sums);
      for (int at = count + n[0]; bits != 0u && at < t.num_pages; bits &= bits - 1u, ++at) t.free_pages[at] = w * 32 + __ffs(bits) - 1;
      count = min(count + total[0], t.num_pages);
    }
    __syncthreads();                                              // the list
    int used = 0, n_moved = 0;
    for (int c0 = 0; c0 < t.rows; c0 += kReorderThreads) {
      const int r = c0 + tid;
      const int p = r < t.rows ? parent_s[r] : -1;
      const int len = p >= 0 ? length_s[p] : 0, full = len >> t.page_shift;
      const bool fresh = r < t.rows && __ldcg(info + r) != 0;
      const bool changes = len > 0 && (p != r || fresh);
      int n[2] = {fresh ? 1 : 0, changes ? 1 : 0}, total[2];
      block_scan(n, total, warp_sums);
      int src = -1, dst = -1;
      bool dropped = false;
      if (fresh) {
        const int k = used + n[0];
        const int* now = scratch + (int64_t)r * t.max_pages;
        if (k < count) {
          src = __ldcg(now + full);
          dst = t.free_pages[count - 1 - k];
          t.block_tables[(int64_t)r * t.max_pages + full] = dst;
          if (real(dst)) atomicAdd(t.page_refs + dst, 1);
        } else {                                                  // out of pages: the row becomes empty
          dropped = true;
          atomicAdd(&dropped_s, 1);
          for (int b = 0; b < full; ++b)
            if (real(__ldcg(now + b))) atomicSub(t.page_refs + __ldcg(now + b), 1);
        }
      }
      if (r < t.rows) {
        copies[2 * r] = src;
        copies[2 * r + 1] = dst;
        t.lengths[r] = dropped ? 0 : len;
        if (changes)
          reinterpret_cast<int4*>(moved)[1 + n_moved + n[1]] = make_int4(r, p, dropped ? 0 : len, fresh && !dropped ? len & page_mask : 0);
      }
      used += total[0];
      n_moved += total[1];
    }
    if (tid == 0) {
      *t.free_count = count - min(used, count);
      moved[0] = n_moved;
    }
  }
  cluster.sync();
  if (me == 0) moved[1] = dropped_s;
  if (cta == 0 && dropped_s != 0) {
    for (int r = warp; r < t.rows; r += kReorderThreads / 32) {
      if (__ldcg(info + r) == 0 || copies[2 * r + 1] >= 0) continue;
      for (int b = lane; b < t.max_pages; b += 32) t.block_tables[(int64_t)r * t.max_pages + b] = -1;
    }
  }
}

// The rows of `moved` in one layer.  The first history_ctas CTAs gather the history, 4 UNITS keys of one group over all rows, through shared
// memory, since a row can be read and written: first everything is read, then everything is written.  The others copy the tokens
// of the pages that are being filled into the pages that the copies got: kPagePieces CTAs a row and pool.
// Bound by memory, 65 MB in 20 us for 256 rows of which half get a page of 64 tokens of 16 heads, and two thirds 16 histories of 1,500
// keys: half of the copy rate.  (A row of a warp in flight at a time, in two launches, took 28 us.)
constexpr int kPagePieces = 4;
template <int UNITS>
__global__ void __launch_bounds__(256) move_kernel(const int4* moved, const int2* copies, float* selected, int groups,
                                                   int64_t capacity, int chunks, int history_ctas, uint4* k_pages, uint4* v_pages, int heads,
                                                   int num_pages, int64_t head_units, int row_units) {
  tc::after_previous_kernel();
  extern __shared__ float4 keep[];
  const int n = moved[0].x;
  if ((int)blockIdx.x < history_ctas) {
    const int g = blockIdx.x / chunks, unit = threadIdx.x % UNITS;
    const int64_t j = ((int64_t)(blockIdx.x - g * chunks) * UNITS + unit) * 4;       // capacity is a multiple of 16: whole units
#pragma unroll 4
    for (int m = threadIdx.x / UNITS; m < n; m += 256 / UNITS) {
      const int4 x = moved[1 + m];
      if (j < x.z && j < capacity) keep[m * UNITS + unit] = *reinterpret_cast<const float4*>(selected + ((int64_t)x.y * groups + g) * capacity + j);
    }
    __syncthreads();
#pragma unroll 4
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
    return;
  }
  const int64_t page_units = head_units * heads;
  const int piece = (blockIdx.x - history_ctas) % (2 * kPagePieces), ctas = (gridDim.x - history_ctas) / (2 * kPagePieces);
  uint4* pool = piece < kPagePieces ? k_pages : v_pages;
  for (int m = (blockIdx.x - history_ctas) / (2 * kPagePieces); m < n; m += ctas) {
    const int4 x = moved[1 + m];
    if (x.w == 0) continue;
    const int2 c = copies[x.x];
    if (c.x < 0 || c.x >= num_pages || c.y < 0 || c.y >= num_pages) continue;
    const int units = x.w * row_units;                            // of one head
    const uint4* __restrict__ from = pool + c.x * page_units;
    uint4* __restrict__ to = pool + c.y * page_units;
#pragma unroll 4
    for (int i = piece % kPagePieces * 256 + threadIdx.x; i < units * heads; i += kPagePieces * 256) {
      const int h = i / units, u = i - h * units;
      to[h * head_units + u] = from[h * head_units + u];
    }
  }
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
  a.inside = total <= kInside;
  a.query_start = query_start; a.cached = cached; a.slots = slots; a.work = work;
  a.layout = step_layout(t.rows, total, t.heads);
  const size_t smem = 5 * ((size_t)t.rows + 1) * 4;
  auto launch = [&](auto kernel, int threads) -> int {
    SA_CUDA_CHECK(allow_smem(kernel, smem));
    count_launch();
    kernel<<<1, threads, smem, s>>>(a);
    SA_CUDA_CHECK(cudaGetLastError());
    return SA_OK;
  };
  const int64_t most = (int64_t)t.rows * max(total + 1, min(max_length, t.max_pages << t.page_shift) + 1);
  const bool narrow = most < (1LL << 31);
  auto by_width = [&](auto per, int threads) {
    constexpr int kPer = decltype(per)::value;
    return narrow ? launch(append_kernel<kPer, int>, threads) : launch(append_kernel<kPer, long long>, threads);
  };
  using One = std::integral_constant<int, 1>;
  // 256 threads where they cover rows and tokens: barriers and sums over eight warps are shorter than over thirty-two
  const int st = t.rows <= 256 && total <= 256 ? by_width(One{}, 256)
                 : t.rows <= 1024              ? by_width(One{}, 1024)
                                               : by_width(std::integral_constant<int, kMaxRows / 1024>{}, 1024);
  if (st != SA_OK || a.inside) return st;
  const unsigned blocks = (unsigned)min((total + 255) / 256, 2 * kSms);
  return launch_after(spread_kernel, dim3(blocks), 256, smem + 16, s, a);
}

size_t reorder_work_words(int rows, int max_pages, int num_pages) { return ReorderWork(rows, max_pages, num_pages).words; }

int reorder(const Tables& t, const int* parents, int* copies, int* work, cudaStream_t s) {
  const ReorderWork w(t.rows, t.max_pages, t.num_pages);
  count_launch();
  const size_t smem = 2 * (size_t)t.rows * 4;
  SA_CUDA_CHECK(allow_smem(reorder_kernel, smem));
  // where there are more warps than rows, a row's pages are cut into parts of a warp's width or more, a power of two of them
  // (4 rows of 500 pages: 28.8 us with a warp a row, 8.2 us so; 256 rows of 24 pages: no parts)
  int shift = 0;
  while ((t.rows << (shift + 1)) <= kCluster * kReorderThreads / 32 && (32 << shift) < t.max_pages) ++shift;
  const int span = (t.max_pages + (1 << shift) - 1) >> shift;
  reorder_kernel<<<kCluster, kReorderThreads, smem, s>>>(t, shift, span, parents, copies, work + w.moved, work + w.info,
                                                         reinterpret_cast<unsigned*>(work + w.marks), work + w.scratch);
  SA_CUDA_CHECK(cudaGetLastError());
  return SA_OK;
}

int move_rows(const Tables& t, const int* copies, const int* work, int groups, int head_dim, int elem_bytes, int64_t capacity, void* k_pages,
              void* v_pages, float* selected, cudaStream_t s) {
  const int row_units = head_dim * elem_bytes / 16;
  // 32 keys a CTA (a line of every row), or 8 where the rows would not fit the shared memory
  auto move = [&](auto kernel, int units) -> int {
    const size_t smem = (size_t)t.rows * units * sizeof(float4);
    const int chunks = (int)((capacity + 4 * units - 1) / (4 * units));
    const unsigned history = (unsigned)chunks * groups, pages = (unsigned)min(t.rows, 256) * 2 * kPagePieces;
    return launch_after(kernel, dim3(history + pages), 256, smem, s, reinterpret_cast<const int4*>(work), reinterpret_cast<const int2*>(copies),
                        selected, groups, capacity, chunks, (int)history, static_cast<uint4*>(k_pages), static_cast<uint4*>(v_pages), t.heads,
                        t.num_pages, (int64_t)row_units << t.page_shift, row_units);
  };
  return t.rows <= 1024 ? move(move_kernel<8>, 8) : move(move_kernel<2>, 2);
}

}  // namespace paged
}  // namespace sa
