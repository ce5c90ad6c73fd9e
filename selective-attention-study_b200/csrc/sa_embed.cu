// Rows of a table, scaled, and the table's gradient by sorted tokens.
//
// Forward: a copy.  Backward, for vocab rows and N tokens, three launches:
//   order   sorts the tokens by their row, tokens of a row in order.  A CTA owns a range of rows and reads all N indices: its 32
//           warps take a run of tokens each, count theirs by row, and after a prefix sum over the warps every warp writes its own
//           tokens' places without another barrier.  148 CTAs, or one for every 1,600 rows of a larger table, read N indices each
//           out of L2, which costs less than the launches of a radix sort.
//   sum     pieces of 4 to 32 sorted tokens: their gradients are summed row by row in that order; a row inside one piece is finished,
//           the parts of rows that cross pieces are kept.  Rows that no token names are written as zeros beside it.
//   join    sums the parts of each row that crossed pieces.
// So a word that is every tenth token is summed by as many CTAs as it needs, and nothing depends on the order of threads.
#include "sa_layers.cuh"

#include <algorithm>
#include <type_traits>

namespace sa {
namespace embed {
namespace {

constexpr int kOrderThreads = 1024, kOrderWarps = kOrderThreads / 32;
constexpr int kMostRows = 1600;            // of the table, a CTA of `order`: 32 counters and a place each in shared memory
constexpr int kThreads = 256, kJoinThreads = 512;
// Rows of the table that a CTA looks at for the ones without tokens, with `groups` of them side by side.
__host__ __device__ constexpr int zero_rows(int groups) { return groups * 4 > 16 ? groups * 4 : 16; }

template <bool VEC>
__global__ void __launch_bounds__(kThreads) forward_kernel(const sa_embedding p, int chunks) {
  tc::after_previous_kernel();
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (id >= (int64_t)p.tokens * chunks) return;
  const int n = (int)(id / chunks), t = (int)(id - (int64_t)n * chunks);
  const int64_t v = p.idx[n];
  const bool inside = v >= 0 && v < p.vocab;
  // one chunk a thread: with VEC eight neighbours, otherwise values `chunks` apart
  float x[1][8];
  if (VEC) {
    if (inside) load_row<1, 1, true>(x, p.weight, p.weight_dtype, v * p.weight_stride + t * 8, 8, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[0][i] = inside ? x[0][i] * p.scale : NAN;
    store_row<1, 1, true>(x, p.y, p.y_dtype, (int64_t)n * p.width + t * 8, 8, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = i * chunks + t;
      if (col >= p.width) continue;
      float one[1][8];
      if (inside) load_row<1, 1, false>(one, p.weight, p.weight_dtype, v * p.weight_stride + col, 1, 0);
      one[0][0] = inside ? one[0][0] * p.scale : NAN;
      store_row<1, 1, false>(one, p.y, p.y_dtype, (int64_t)n * p.width + col, 1, 0);
    }
  }
}

// sorted: (token, row) by row; starts: where each row's tokens begin, and the number of all behind them.
__global__ void __launch_bounds__(kOrderThreads) order_kernel(const int64_t* idx, int64_t skip, int tokens, int vocab, int rows, int2* sorted,
                                                              int* starts) {
  tc::after_previous_kernel();
  extern __shared__ int counts[];                                  // [rows][warps]
  __shared__ int before_s[kOrderWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lo = blockIdx.x * rows, hi = min(vocab, lo + rows), mine = hi - lo;
  for (int i = threadIdx.x; i < mine * kOrderWarps; i += kOrderThreads) counts[i] = 0;
  __syncthreads();
  const int run = ((tokens + kOrderWarps - 1) / kOrderWarps + 31) / 32 * 32;
  const int from = min(tokens, warp * run), to = min(tokens, from + run);
  int before = 0;                                                  // tokens of earlier rows
  // A run of up to kKept groups of 32 is looked at once: a token's row and its place among its warp's tokens of the row are kept.
  constexpr int kKept = 16;
  const bool kept = run <= 32 * kKept;
  int row[kKept], place[kKept];
  if (kept) {
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
      const int n = from + 32 * k + lane;
      const int64_t v = n < to ? idx[n] : -1;
      before += v >= 0 && v < lo && v != skip;
      row[k] = v >= lo && v < hi && v != skip ? (int)(v - lo) : -1;
    }
#pragma unroll
    for (int k = 0; k < kKept; ++k) {
      place[k] = 0;
      if (__ballot_sync(~0u, row[k] >= 0) == 0u) continue;
      // a warp's counters are its own: of the lanes that have a row's tokens the first moves its counter on
      const unsigned int same = __match_any_sync(~0u, row[k]);
      if (row[k] >= 0) place[k] = counts[row[k] * kOrderWarps + warp] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (row[k] >= 0 && lane == __ffs(same) - 1) counts[row[k] * kOrderWarps + warp] += __popc(same);
      __syncwarp();
    }
  } else {
#pragma unroll 8
    for (int n = from + lane; n < to; n += 32) {
      const int64_t v = idx[n] == skip ? -1 : idx[n];
      if (v >= 0 && v < lo) ++before;
      if (v >= lo && v < hi) atomicAdd(&counts[(int)(v - lo) * kOrderWarps + warp], 1);
    }
  }
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(~0u, before, o);
  if (lane == 0) before_s[warp] = before;
  __syncthreads();
  before = 0;
  for (int i = 0; i < kOrderWarps; ++i) before += before_s[i];
  // Places: rows in order, in each the warps in order.  A warp turns a row's 32 counters into sums of the earlier ones; then the
  // rows' totals are added up, a run of rows a warp.
  int* const totals = counts + rows * kOrderWarps;                 // [rows]
  for (int r = warp; r < mine; r += kOrderWarps) {
    const int own = counts[r * kOrderWarps + lane];
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += other;
    }
    counts[r * kOrderWarps + lane] = upto - own;
    if (lane == 31) totals[r] = upto;
  }
  __syncthreads();
  const int per = (mine + kOrderWarps - 1) / kOrderWarps, r0 = min(mine, warp * per), r1 = min(mine, r0 + per);
  int all = 0;
  for (int r = r0 + lane; r < r1; r += 32) all += totals[r];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(~0u, all, o);
  __syncthreads();                                                 // before_s has been read by all
  if (lane == 0) before_s[warp] = all;
  __syncthreads();
  int upto = before;
  for (int i = 0; i < kOrderWarps; ++i) {
    if (i < warp) upto += before_s[i];
    before += before_s[i];
  }
  for (int r = r0; r < r1; r += 32) {
    const int own = r + lane < r1 ? totals[r + lane] : 0;
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += other;
    }
    if (r + lane < r1) {
      totals[r + lane] = upto + sum - own;
      starts[lo + r + lane] = upto + sum - own;
    }
    upto += __shfl_sync(~0u, sum, 31);
  }
  if (hi == vocab && threadIdx.x == 0) starts[vocab] = before;
  __syncthreads();
  if (kept) {
#pragma unroll
    for (int k = 0; k < kKept; ++k)
      if (row[k] >= 0) sorted[totals[row[k]] + counts[row[k] * kOrderWarps + warp] + place[k]] = make_int2(from + 32 * k + lane, lo + row[k]);
    return;
  }
  constexpr int kAhead = 8;                                        // indices in flight
  for (int n0 = from; n0 < to; n0 += 32 * kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int n = n0 + 32 * k + lane;
      const int64_t v = n < to ? idx[n] : -1;
      row[k] = v >= lo && v < hi && v != skip ? (int)(v - lo) : -1;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = row[k];
      if (__ballot_sync(~0u, r >= 0) == 0u) continue;
      const unsigned int same = __match_any_sync(~0u, r);
      if (r >= 0) {
        const int at = totals[r] + counts[r * kOrderWarps + warp] + __popc(same & ((1u << lane) - 1u));
        sorted[at] = make_int2(n0 + 32 * k + lane, lo + r);
      }
      __syncwarp();
      if (r >= 0 && lane == __ffs(same) - 1) counts[r * kOrderWarps + warp] += __popc(same);
      __syncwarp();
    }
  }
}

struct Sum {
  const int2* sorted;
  const int* starts;
  const void* dy;
  int dtype;                               // of dy
  int64_t dy_stride;
  const float* factor;                     // of its rows, or null
  void* dweight;
  int weight_dtype;
  float scale;
  int vocab, width, chunks, groups;        // chunks of 8 values in a row; rows that a CTA works on side by side
  float* parts;                            // [pieces][2][width]: of a row that began before the piece, of one that goes on behind it
  int pieces, piece;                       // tokens of one
};

// A thread's eight columns of a row: neighbours, or `chunks` apart.
template <bool VEC> __device__ __forceinline__ int column(const Sum& p, int t, int i) { return VEC ? t * 8 + i : i * p.chunks + t; }

template <bool VEC>
__device__ __forceinline__ void read_eight(const Sum& p, const void* base, int dtype, int64_t at, int t, float (&x)[8]) {
  if (VEC) {
    float v[1][8];
    load_row<1, 1, true>(v, base, dtype, at + t * 8, 8, 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[0][i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = column<VEC>(p, t, i);
      x[i] = 0.f;
      if (col < p.width) {
        if (dtype == SA_F32) x[i] = static_cast<const float*>(base)[at + col];
        else if (dtype == SA_BF16) x[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at + col]);
        else x[i] = __half2float(static_cast<const __half*>(base)[at + col]);
      }
    }
  }
}
template <bool VEC>
__device__ __forceinline__ void write_eight(const Sum& p, void* base, int dtype, int64_t at, int t, const float (&x)[8]) {
  if (VEC) {
    float v[1][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[0][i] = x[i];
    store_row<1, 1, true>(v, base, dtype, at + t * 8, 8, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = column<VEC>(p, t, i);
      if (col >= p.width) continue;
      if (dtype == SA_F32) static_cast<float*>(base)[at + col] = x[i];
      else if (dtype == SA_BF16) static_cast<__nv_bfloat16*>(base)[at + col] = __float2bfloat16_rn(x[i]);
      else static_cast<__half*>(base)[at + col] = __float2half_rn(x[i]);
    }
  }
}
// `old`: what stands there, which ADD adds to.
template <bool VEC, bool ADD>
__device__ __forceinline__ void finish_row(const Sum& p, int row, int t, const float (&x)[8], const float (&old)[8]) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = ADD ? fmaf(x[i], p.scale, old[i]) : x[i] * p.scale;
  write_eight<VEC>(p, p.dweight, p.weight_dtype, (int64_t)row * p.width, t, y);
}

// blockIdx.y: columns, kThreads chunks at a time.  The first CTAs take pieces, the others rows without tokens.
template <bool VEC, bool ADD>
__global__ void __launch_bounds__(kThreads) sum_kernel(const Sum p, int piece_blocks) {
  tc::after_previous_kernel();
  const int across = min(p.chunks, kThreads), group = threadIdx.x / across, t = blockIdx.y * kThreads + threadIdx.x - group * across;
  if (group >= (int)blockDim.x / across || t >= p.chunks) return;
  if ((int)blockIdx.x >= piece_blocks) {
    const int groups = (int)blockDim.x / across, v0 = ((int)blockIdx.x - piece_blocks) * zero_rows(groups), v1 = min(p.vocab, v0 + zero_rows(groups));
    const float none[8] = {};
    for (int v = v0 + group; v < v1; v += groups)
      if (p.starts[v] == p.starts[v + 1]) write_eight<VEC>(p, p.dweight, p.weight_dtype, (int64_t)v * p.width, t, none);
    return;
  }
  if (group >= p.groups) return;
  const int piece = blockIdx.x * p.groups + group, all = p.starts[p.vocab];
  const int from = piece * p.piece, to = min(all, from + p.piece);
  if (from >= to) return;
  float sum[8] = {};
  constexpr int kAhead = 4;                                        // rows of dy in flight (8: fewer CTAs an SM, 39 -> 45 us)
  for (int i0 = from; i0 < to; i0 += kAhead) {
    int2 at[kAhead];
    float x[kAhead][8], old[ADD ? kAhead : 1][8];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) at[k] = i0 + k < to ? p.sorted[i0 + k] : make_int2(0, -1);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (at[k].y >= 0) {
        read_eight<VEC>(p, p.dy, p.dtype, at[k].x * p.dy_stride, t, x[k]);
        if (ADD) read_eight<VEC>(p, p.dweight, SA_F32, (int64_t)at[k].y * p.width, t, old[k]);
      }
    const int next = i0 + kAhead < to ? p.sorted[i0 + kAhead].y : -1;
    int begin[kAhead], end[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      begin[k] = at[k].y >= 0 ? p.starts[at[k].y] : 0;
      end[k] = at[k].y >= 0 ? p.starts[at[k].y + 1] : 0;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (at[k].y < 0) continue;
      const float factor = p.factor != nullptr ? p.factor[at[k].x] : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = fmaf(factor, x[k][i], sum[i]);
      if ((k + 1 < kAhead ? at[k + 1 < kAhead ? k + 1 : k].y : next) == at[k].y) continue;
      if (begin[k] >= from && end[k] <= from + p.piece) finish_row<VEC, ADD>(p, at[k].y, t, sum, old[ADD ? k : 0]);
      else write_eight<VEC>(p, p.parts, SA_F32, ((int64_t)piece * 2 + (begin[k] >= from ? 1 : 0)) * p.width, t, sum);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = 0.f;
    }
  }
}

// Rows that cross pieces, by the piece in which they begin: a CTA looks at `some` pieces, a thread at one.  Groups of threads take a row
// of few parts each; the parts of a longer one are dealt to all groups, whose sums are joined in a tree.
constexpr int kJoinPieces = 64, kFewParts = 8;
template <bool VEC, bool ADD>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Sum p, int some) {
  tc::after_previous_kernel();
  __shared__ float by_group[kJoinThreads][9];
  __shared__ int2 found[kJoinPieces];                              // row, its last piece
  __shared__ int first[kJoinPieces];
  __shared__ int count;
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const int all = p.starts[p.vocab];
  if ((int)threadIdx.x < some) {
    const int piece = blockIdx.x * some + threadIdx.x, from = piece * p.piece, to = from + p.piece;
    if (to < all) {
      const int row = p.sorted[to - 1].y;
      // its last row goes on behind it, and did not begin before
      if (p.sorted[to].y == row && p.starts[row] >= from) {
        const int i = atomicAdd(&count, 1);                        // rows in any order
        found[i] = make_int2(row, (p.starts[row + 1] - 1) / p.piece);
        first[i] = piece;
      }
    }
  }
  __syncthreads();
  const int across = min(p.chunks, kJoinThreads), group = threadIdx.x / across, t = blockIdx.y * kJoinThreads + threadIdx.x - group * across;
  int groups = kJoinThreads / across;
  while (groups & (groups - 1)) groups &= groups - 1;              // a power of two
  auto sum_of = [&](int piece, int k0, int k1, float (&sum)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = 0.f;
#pragma unroll 8
    for (int k = k0; k < k1; ++k) {
      float x[8];
      read_eight<VEC>(p, p.parts, SA_F32, ((int64_t)(piece + k) * 2 + (k == 0 ? 1 : 0)) * p.width, t, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += x[i];
    }
  };
  auto finish = [&](int row, const float (&sum)[8]) {
    float old[8] = {};
    if (ADD) read_eight<VEC>(p, p.dweight, SA_F32, (int64_t)row * p.width, t, old);
    finish_row<VEC, ADD>(p, row, t, sum, old);
  };
  float sum[8];
  if (group < groups && t < p.chunks)
    for (int i = group; i < count; i += groups) {
      const int parts = found[i].y - first[i] + 1;
      if (parts > kFewParts) continue;
      sum_of(first[i], 0, parts, sum);
      finish(found[i].x, sum);
    }
  for (int i = 0; i < count; ++i) {
    const int parts = found[i].y - first[i] + 1;
    if (parts <= kFewParts) continue;
    const int per = (parts + groups - 1) / groups, k0 = min(parts, group * per), k1 = min(parts, k0 + per);
    const bool mine = group < groups && t < p.chunks;
    if (mine) sum_of(first[i], k0, k1, sum);
    for (int half = groups >> 1; half > 0; half >>= 1) {
      __syncthreads();
      if (mine && group >= half && group < 2 * half)
#pragma unroll
        for (int e = 0; e < 8; ++e) by_group[threadIdx.x][e] = sum[e];
      __syncthreads();
      if (mine && group < half)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += by_group[threadIdx.x + half * across][e];
    }
    if (mine && group == 0) finish(found[i].x, sum);
  }
}

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
// Sorted tokens that are summed in a row: 32, and fewer where that would leave an SM less than two CTAs of threads with a chunk of a piece each
// (2,048 tokens of 768: 56 us with 32, 10 with 4; but 16,384 of 1,024 with words as often as words are 47 with 32 and 60 with 8, whose
// parts of rows take longer to join).
int piece_of(int tokens, int width) {
  const int64_t chunks = (width + 7) / 8;
  int piece = 32;
  while (piece > 4 && tokens / piece * chunks < 2 * kSms * 128) piece /= 2;
  return piece;
}
int pieces_of(int tokens, int width) { return (tokens + piece_of(tokens, width) - 1) / piece_of(tokens, width); }

}  // namespace

size_t sum_rows_bytes(int tokens, int vocab, int width) {
  return (size_t)(up((int64_t)tokens * 8, 256) + up(((int64_t)vocab + 1) * 4, 256) + (int64_t)pieces_of(tokens, width) * 2 * width * 4);
}
size_t backward_bytes(const sa_embedding& p) { return sum_rows_bytes(p.tokens, p.vocab, p.width); }

int forward(const sa_embedding& p, cudaStream_t s) {
  const int chunks = (p.width + 7) / 8;
  const dim3 grid((unsigned)(((int64_t)p.tokens * chunks + kThreads - 1) / kThreads));
  const bool vec = p.width % 8 == 0 && eights(p.weight, p.weight_dtype, p.weight_stride, p.vocab) && eights(p.y, p.y_dtype, p.width, p.tokens);
  return vec ? launch_after(forward_kernel<true>, grid, kThreads, 0, s, p, chunks) : launch_after(forward_kernel<false>, grid, kThreads, 0, s, p, chunks);
}

int sum_rows(const RowSums& p, cudaStream_t s) {
  char* room = static_cast<char*>(p.workspace);
  int2* sorted = reinterpret_cast<int2*>(room);
  int* starts = reinterpret_cast<int*>(room + up((int64_t)p.tokens * 8, 256));
  float* parts = reinterpret_cast<float*>(reinterpret_cast<char*>(starts) + up(((int64_t)p.vocab + 1) * 4, 256));
  const int rows = std::min((p.vocab + kSms - 1) / kSms, kMostRows);
  const int st = launch_after(order_kernel, dim3((p.vocab + rows - 1) / rows), kOrderThreads, (size_t)rows * (kOrderWarps + 1) * 4, s, p.idx, p.skip, p.tokens,
                        p.vocab, rows, sorted, starts);
  if (st != SA_OK) return st;
  Sum a{sorted, starts, p.dy, p.dtype, p.dy_stride, p.factor, p.out, p.out_dtype, p.scale, p.vocab, p.width, (p.width + 7) / 8, 0, parts, pieces_of(p.tokens, p.width),
        piece_of(p.tokens, p.width)};
  a.groups = a.chunks < kThreads ? std::min(kThreads / a.chunks, std::max(1, a.pieces / (2 * kSms))) : 1;
  const bool vec = p.width % 8 == 0 && eights(p.dy, p.dtype, p.dy_stride, p.tokens) && eights(p.out, p.out_dtype, p.width, p.vocab);
  const int piece_blocks = (a.pieces + a.groups - 1) / a.groups;
  // as many threads as the groups need: a thread takes 80 to 128 registers
  const int across = std::min(a.chunks, kThreads), threads = (int)up(a.groups * across, 32), side = threads / across;
  const dim3 grid(piece_blocks + (p.add ? 0 : (p.vocab + zero_rows(side) - 1) / zero_rows(side)), (a.chunks + kThreads - 1) / kThreads);
  auto launch = [&](auto vec_, auto add) {
    constexpr bool VEC = decltype(vec_)::value, ADD = decltype(add)::value;
    const int status = launch_after(sum_kernel<VEC, ADD>, grid, threads, 0, s, a, piece_blocks);
    if (status != SA_OK || a.pieces < 2) return status;
    const int some = std::min(kJoinPieces, std::max(1, a.pieces / (4 * kSms)));
    return launch_after(join_kernel<VEC, ADD>, dim3((a.pieces - 2) / some + 1, (a.chunks + kJoinThreads - 1) / kJoinThreads), kJoinThreads, 0, s, a, some);
  };
  const std::true_type yes;
  const std::false_type no;
  if (p.add) return vec ? launch(yes, yes) : launch(no, yes);
  return vec ? launch(yes, no) : launch(no, no);
}

int backward(const sa_embedding& p, cudaStream_t s) {
  return sum_rows(RowSums{p.idx, INT64_MIN, p.tokens, p.vocab, p.width, p.dy, p.y_dtype, p.dy_stride, nullptr, p.scale, p.dweight, p.weight_dtype, false, p.workspace}, s);
}

}  // namespace embed
}  // namespace sa
