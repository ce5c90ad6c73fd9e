// Paged caches: what the table kernels (sa_paged.cu), the attention over pages and the C entry points share.
#pragma once

#include "sa_common.cuh"

namespace sa {
namespace paged {

constexpr int kMaxRows = 4096;       // requests of one set of tables (the table kernel keeps five numbers a row in shared memory)
constexpr int kTile = 128;           // query rows and keys of a tile of the tensor-core kernels
constexpr int kDecodeCtas = 4;       // CTAs of the kernel of few tokens that an SM holds

struct Tables {
  int rows, max_pages, num_pages, page_shift, heads;
  int *block_tables, *lengths, *free_pages, *free_count, *page_refs;
};

// ---- the plan of a step: int32 words that sa_page_append writes and the attention over pages reads ------------------------
// header | sums over the rows | first tile of every row | tiles | tile items | decode items | tickets (zero between launches)
enum : int { kTiles = 0, kTileItems = 1, kDecodeItems = 2, kPieceKeys = 3, kPagesWanted = 4, kFreeBefore = 5, kFreeAfter = 6, kCut = 7,
             kHeaderWords = 16 };

// One walk over the keys of a 128-query tile: key tiles from the diagonal back, cut into `pieces` (which stand together).
struct TileItem {
  int row, token;          // the row, and where its new tokens start in q
  int mi, tile;            // query tile inside the row's sequence; number of the tile in the step
  int piece, pieces;
  int cached, length;      // tokens of the row before and after the step
};
// Keys [c0, c1) of a row that gets one token, or a few.
struct DecodeItem {
  short row, count;           // rows are at most kMaxRows; new tokens
  int token;
  int c0, c1;
  int piece, pieces, first;   // `first`: the row's first item
  int length;                 // with the new tokens
};

// Rows of this many new tokens go through the tile kernels, rows of fewer through the kernel of few tokens.  A step of one row
// that may get more takes the tile kernels whatever it gets: the other launch would find nothing, for 2 us.
constexpr int kFewTokens = 8;
inline bool few_only(int total, int max_count) { return min(total, max_count) <= kFewTokens; }
inline int tile_tokens(int rows, int total, int max_count) { return rows == 1 && !few_only(total, max_count) ? 1 : kFewTokens + 1; }

struct StepLayout {
  int tiles_max, tile_items_max, decode_items_max;
  size_t sums, tile_start, tiles, tile_items, decode_items, tickets, words;   // offsets in words
  int tickets_count;
};
inline int decode_wave(int heads) { const int w = kSms * kDecodeCtas / heads; return w > 1 ? w : 1; }
inline int tile_wave(int heads) { const int w = kSms / heads; return w > 1 ? w : 1; }
constexpr int kDecodeWaves = 4;
constexpr int kTileWaves = 2, kPieceTiles = 4;                  // waves of pieces at most; key tiles of a piece at least
inline StepLayout step_layout(int rows, int total, int heads) {
  StepLayout l{};
  const int64_t with_tiles = min(rows, total / (rows == 1 ? 1 : kFewTokens + 1));   // n tokens of one touch (n + 254) / 128 tiles
  l.tiles_max = (int)(((int64_t)total + 254 * with_tiles) / kTile);
  l.tile_items_max = l.tiles_max > 0 ? l.tiles_max + kTileWaves * tile_wave(heads) : 0;
  const int singles = min(rows, total), wave = decode_wave(heads);      // as the plan spreads them (append_kernel)
  l.decode_items_max = 2 * singles <= wave ? wave : singles + kDecodeWaves * wave;
  size_t at = kHeaderWords;
  auto take = [&](size_t n) {
    const size_t x = at;
    at += (n + 7) / 8 * 8;
    return x;
  };
  l.sums = take(5 * ((size_t)rows + 1));
  l.tile_start = take((size_t)rows + 1);
  l.tiles = take(8 * (size_t)l.tiles_max);
  l.tile_items = take(8 * (size_t)l.tile_items_max);
  l.decode_items = take(8 * (size_t)l.decode_items_max);
  l.tickets_count = 2 * l.decode_items_max * heads;           // one a row and head (at the row's first item), one an item and group
  l.tickets = take((size_t)l.tickets_count);
  l.words = at;
  return l;
}

// ---- attention over pages -------------------------------------------------------------------------------------------------
struct Attention {
  int rows, max_pages, num_pages, page_shift, heads, groups, head_dim, exempt;
  int total, max_length, max_count;
  const int* block_tables;
  const int64_t* slots;
  int* work;                          // the step's plan, with its tickets
  bool plan_tickets;                  // the plan's tickets are this call's alone while it runs; false: the call clears its own
  void *k_pages, *v_pages;
  float* selected;
  int64_t sel_stride;                 // keys of a row's history (max_pages pages)
  const void *q, *k, *v;
  int64_t q_stride[2], k_stride[2], v_stride[2];     // token, head
  void* y;                            // (total, heads, head_dim)
  float* workspace;
};
// Floats of scratch: the partial sums of the kernel of few tokens and new selection; the tile kernels' checkpoints and pieces.
struct AttentionScratch {
  size_t own_tickets, partial, sel_new, carry, part, lse, tickets, floats;
  int64_t key_stride;                 // keys of a checkpoint row
};
AttentionScratch attention_scratch(const Attention& a);
// `beside`: launched behind tiles() of the same call, and runs while that still does.
int decode(const Attention& a, bool beside, cudaStream_t s);
// `moved` is set once the histories have been moved on; a call that fails after that puts them back.
int tiles(const Attention& a, bool* moved, cudaStream_t s);
int restore_histories(const Attention& a, cudaStream_t s);

// ---- launches (sa_paged.cu) ---------------------------------------------------------------------------------------------
int append(const Tables& t, const int* counts, int total, int max_length, int max_count, int* query_start, int* cached, int64_t* slots,
           int* work, cudaStream_t s);
size_t reorder_work_words(int rows, int max_pages, int num_pages);
int reorder(const Tables& t, const int* parents, int* copies, int* work, cudaStream_t s);
int move_rows(const Tables& t, const int* copies, const int* work, int groups, int head_dim, int elem_bytes, int64_t capacity, void* k_pages,
              void* v_pages, float* selected, cudaStream_t s);

}  // namespace paged
}  // namespace sa
