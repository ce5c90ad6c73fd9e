// Tensor-core engine, forward: what its translation units share.
#pragma once

#include "sa_paged.cuh"
#include "sa_tc_host.cuh"
#include "sa_tc_ptx.cuh"

namespace sa {
namespace tc {

constexpr int kTile = 128;            // query rows per CTA; also the carry checkpoint spacing
constexpr int kRowTile = 16384;       // bytes of a [128][64] bf16 operand tile
constexpr int kMaxLiveTiles = 1024;   // key tiles of a sequence when dead tiles are left out (sa_tc_skip.cu)

// The PAGED forms of the forward kernels: keys and values in pages, rows of any length (sa_tc_paged.cu).  Maps over (d, token,
// head) of q, and over the pools with boxes of `box_rows` tokens; `carry` has a row of key_stride keys for every tile and group.
struct PagedWalk {
  const int* header;                 // of the step's plan
  const paged::TileItem* items;
  const int* tables;                 // pages of a row
  int heads, max_pages, page_shift, box_rows;
  int64_t key_stride;
  unsigned int* tickets;             // one a tile and head, zero
  float *part, *lse;                 // rows of pieces, by item and head
};
// The boxes of the 128 keys from j0 on that hold a key below `seq`: lane u of a converged warp loads box u (64 columns of it a
// call), from the page that table_entry gave it.
struct PageBoxes {
  const int* row;                    // the row's block table
  int page_shift, box_rows;
  __device__ __forceinline__ int count(int j0, int seq) const { return (min(kTile, seq - j0) + box_rows - 1) / box_rows; }
  __device__ __forceinline__ int page(int j0, int seq, int lane) const {
    const int j = j0 + lane * box_rows;
    return lane * box_rows < kTile && j >= 0 && j < seq ? __ldg(row + (j >> page_shift)) : -1;
  }
  __device__ __forceinline__ int at(int j0, int lane) const { return (j0 + lane * box_rows) & ((1 << page_shift) - 1); }
};

struct ForwardMaps {                  // boxes of 128 rows x 64 columns
  CUtensorMap q, k, v, q0, k0;
};
// Two heads a CTA (sa_tc_fwd_pair.cu): head_dim 64, an even number of heads sharing a selector.
int forward_pair(const Problem& p, const ForwardMaps& m, const float* carry, float* out, float* lse2, const WaitCtx& status,
                 const uint8_t* alive, cudaStream_t s);

// Two rows a CTA (sa_tc_fwd_self.cu): head_dim 64, one head per selector, an even number of rows.
int forward_self(const Problem& p, const ForwardMaps& m, const float* carry, float* out, float* lse2, const WaitCtx& status,
                 const uint8_t* alive, cudaStream_t s);

// The same over pages (sa_tc_paged_self.cu): head_dim 64, every head its own selector, an even number of heads.
int forward_self_pages(const PagedWalk& walk, const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, const float* carry,
                       int items_max, int exempt, float scale, const WaitCtx& status, __nv_bfloat16* y, const RowLayout& y_rows, cudaStream_t s);

}  // namespace tc
}  // namespace sa
