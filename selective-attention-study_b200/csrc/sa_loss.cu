// Softmax cross entropy over a vocabulary, from the hidden states and the output table, without its logits:
//
//   z = x W^T,  loss_n = log sum_v exp z_nv - z_n,t(n),  dz = (softmax(z) - [v = t]) g_n,  dx = dz W,  dW = dz^T x.
//
// Forward: one product whose epilogue reduces every half tile of logits to its rows' maxima and sums, and a kernel that joins
// them.  Backward: the vocabulary in pieces; a piece's logits are computed again (the same product), turned into dz in 16 bits,
// and read by the two products of the gradients.  Four products of 2 N V d operations in all, one of them for not keeping N V
// logits; the sums of dx over the pieces stay in fp32.
#include "sa_loss.cuh"

#include <algorithm>

#include "sa_product.cuh"

namespace sa {
namespace loss {
namespace {

using namespace product;

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kHalfScale = 16384.f;      // of dz in fp16, whose smallest normal number is 2^-14: probabilities from 2^-28 on keep their bits

// ---- operands of the products: 16 bits, rows at multiples of 16 bytes ------------------------------------------------------------

struct Convert {
  const void* src;
  int dtype;
  int64_t src_stride;
  int rows, width, pitch;
  int64_t part;                            // elements of a part
  int parts, half;
  uint16_t* dst;
  // rows of tokens in a backward: what does not count is nothing, whatever stands there; and every token's factor
  const int64_t* targets;
  int64_t ignore_index;
  int vocab, reduction;
  const float *dloss, *count, *largest;
  float *factor, *scale;
};

__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t at) {
  if (dtype == SA_F32) return static_cast<const float*>(p)[at];
  if (dtype == SA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  return __half2float(static_cast<const __half*>(p)[at]);
}

__global__ void __launch_bounds__(256) convert_kernel(const Convert c) {
  after_previous_kernel();
  const int chunks = c.pitch >> 3;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (int64_t)c.rows * chunks) return;
  const int row = (int)(id / chunks), chunk = (int)(id - (int64_t)row * chunks), col = chunk * 8;
  bool counts = true;
  if (c.targets != nullptr) {
    const int64_t t = c.targets[row];
    counts = t != c.ignore_index;
    if (chunk == 0) {
      float g = c.dloss[c.reduction == SA_REDUCTION_NONE ? row : 0];
      if (c.reduction == SA_REDUCTION_MEAN) g /= *c.count;
      float factor = g;
      if (c.half) {                        // factors of 2^14 at most, and the rest in the results' scale
        const float most = c.reduction == SA_REDUCTION_NONE ? *c.largest : fabsf(g);
        factor = most == 0.f ? 0.f : g / most * kHalfScale;
        if (row == 0) *c.scale = c.reduction == SA_REDUCTION_MEAN && *c.count == 0.f ? 0.f : most / kHalfScale;
      }
      c.factor[row] = !counts ? 0.f : t < 0 || t >= c.vocab ? NAN : factor;
    }
  }
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
  const int64_t at = row * c.src_stride + col;
  const int bytes = c.dtype == SA_F32 ? 4 : 2;
  if (counts) {
    const char* src = static_cast<const char*>(c.src) + at * bytes;
    if (col + 8 <= c.width && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
      if (c.dtype == SA_F32) {
        const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      } else {
        const uint4 a = *reinterpret_cast<const uint4*>(src);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (c.dtype == SA_BF16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
          } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + i < c.width) v[i] = load_as_float(c.src, c.dtype, at + i);
    }
  }
  for (int part = 0; part < c.parts; ++part) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = c.half ? pack_half(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(c.dst + part * c.part + (int64_t)row * c.pitch + col) = make_uint4(w[0], w[1], w[2], w[3]);
    if (part + 1 < c.parts) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16) == INFINITY || __uint_as_float(w[i] << 16) == -INFINITY ? 0.f : v[2 * i] - __uint_as_float(w[i] << 16);
        const float high = __uint_as_float(w[i] & 0xFFFF0000u);
        v[2 * i + 1] = high == INFINITY || high == -INFINITY ? 0.f : v[2 * i + 1] - high;
      }
    }
  }
}

// The largest |dloss| of the tokens that count.
__global__ void __launch_bounds__(1024) largest_kernel(const float* dloss, const int64_t* targets, int64_t ignore_index, int tokens, float* largest) {
  after_previous_kernel();
  __shared__ float warps[32];
  float most = 0.f;
  for (int i = threadIdx.x; i < tokens; i += 1024)
    if (targets[i] != ignore_index) {
      const float g = fabsf(dloss[i]);
      most = g > most || g != g ? g : most;
    }
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(~0u, most, o);
    most = other > most || other != other ? other : most;
  }
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = most;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 32; ++i) most = warps[i] > most || warps[i] != warps[i] ? warps[i] : most;
    *largest = most;
  }
}

// Joins the half tiles of 32 tokens: a lane has a token, the 32 warps take the half tiles in turn, eight loads in flight.  The last CTA
// to end sums all tokens, in order.
constexpr int kJoinThreads = 1024, kJoinWarps = kJoinThreads / 32, kJoinAhead = 8;
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const float2* stats, int slots, const float* at_target, const int64_t* targets,
                                                            int64_t ignore_index, int tokens, int vocab, int reduction, float* lse, float* loss,
                                                            float* count, float2* sums, unsigned int* ticket) {
  after_previous_kernel();
  __shared__ float2 parts[kJoinWarps][32];
  __shared__ bool last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 32 + lane;
  float top = -INFINITY, sum = 0.f;
  auto add = [&](const float2* v, int n) {
    float most = top;
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)
      if (i < n) most = fmaxf(most, v[i].x);
    const float from = most == -INFINITY ? 0.f : most;
    sum *= ex2(top - from);
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)
      if (i < n) sum += v[i].y * ex2(v[i].x - from);
    top = most;
  };
  for (int i = warp; i < slots; i += kJoinWarps * kJoinAhead) {
    float2 v[kJoinAhead];
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k)
      v[k] = i + k * kJoinWarps < slots && row < tokens ? stats[(int64_t)(i + k * kJoinWarps) * tokens + row] : make_float2(-INFINITY, 0.f);
    add(v, kJoinAhead);
  }
  parts[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp == 0) {
    top = -INFINITY;
    sum = 0.f;
    for (int i = 0; i < kJoinWarps; i += kJoinAhead) {
      float2 v[kJoinAhead];
#pragma unroll
      for (int k = 0; k < kJoinAhead; ++k) v[k] = parts[i + k][lane];
      add(v, kJoinAhead);
    }
    float mine = 0.f, counts = 0.f;
    if (row < tokens) {
      const float all = top + log2f(sum);
      lse[row] = all;
      const int64_t t = targets[row];
      if (t != ignore_index) {
        mine = t < 0 || t >= vocab ? NAN : (all - at_target[row]) * kLn2;
        counts = 1.f;
      }
      if (reduction == SA_REDUCTION_NONE) loss[row] = mine;
    }
    if (reduction != SA_REDUCTION_NONE) {
      for (int o = 16; o > 0; o >>= 1) {
        mine += __shfl_xor_sync(~0u, mine, o);
        counts += __shfl_xor_sync(~0u, counts, o);
      }
      if (lane == 0) {
        sums[blockIdx.x] = make_float2(mine, counts);
        __threadfence();
        last = atomicAdd(ticket, 1u) == gridDim.x - 1;
      }
    }
  }
  if (reduction == SA_REDUCTION_NONE) return;
  __syncthreads();
  if (!last || warp > 0) return;
  __threadfence();
  double a = 0.0, b = 0.0;
  for (int i = lane; i < (int)gridDim.x; i += 32) {
    const volatile float2* v = sums + i;
    a += (double)v->x;
    b += (double)v->y;
  }
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(~0u, a, o);
    b += __shfl_xor_sync(~0u, b, o);
  }
  if (lane == 0) {
    *count = (float)b;
    *loss = (float)(reduction == SA_REDUCTION_MEAN ? a / b : a);
  }
}

// Rows of a dealt tile from its slabs, in order: a thread has four columns of a row, four slabs in flight.
constexpr int kFinishThreads = 256;
__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const float* slabs, const Walk w, int tile_rows, const float* scale, void* out,
                                                                int dtype, int64_t out_pitch) {
  after_previous_kernel();
  const int tile = w.whole + blockIdx.x;
  int tm, tn;
  w.place(tile, &tm, &tn);
  const int n = w.slabs_of(tile), columns = min(w.bn, w.n - tn * w.bn), across = w.bn >> 2;
  const int in_tile = blockIdx.y * (kFinishThreads / across) + threadIdx.x / across, c = (threadIdx.x % across) * 4, row = tm * tile_rows + in_tile;
  if (row >= w.m || c >= columns) return;
  const float by = scale != nullptr ? *scale : 1.f;
  const float4* from = reinterpret_cast<const float4*>(slabs + ((int64_t)blockIdx.x * w.slabs * tile_rows + in_tile) * w.bn + c);
  const int64_t stride = (int64_t)tile_rows * w.bn / 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    const float4 x = from[k * stride];
    v.x += x.x;
    v.y += x.y;
    v.z += x.z;
    v.w += x.w;
  }
  const float f[4] = {v.x * by, v.y * by, v.z * by, v.w * by};
  const int64_t at = (int64_t)row * out_pitch + tn * w.bn + c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + i >= columns) break;
    if (dtype == SA_F32) static_cast<float*>(out)[at + i] = f[i];
    else if (dtype == SA_BF16) static_cast<__nv_bfloat16*>(out)[at + i] = __float2bfloat16_rn(f[i]);
    else static_cast<__half*>(out)[at + i] = __float2half_rn(f[i]);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t over(int64_t x, int64_t by) { return (x + by - 1) / by; }

// 3-D map over (inner, row, part) of 16-bit elements; box = (64 elements, box_rows, 1), 128-byte swizzle, zeros outside.
int make_map(CUtensorMap* map, const void* base, int64_t inner, int64_t rows, int parts, int64_t pitch, int64_t part, int box_rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return SA_ERR_CUDA;
  if ((reinterpret_cast<uintptr_t>(base) & 15) != 0 || (pitch & 7) != 0) return SA_ERR_ALIGNMENT;
  if (parts == 1) part = pitch * rows;
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)parts};
  cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)part * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, elem[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_cuda_error(10000 + (int)r);
    return SA_ERR_CUDA;
  }
  return SA_OK;
}

// A matrix of rows as the products read it.
struct Operand {
  const uint16_t* base;
  int64_t rows, width, pitch, part;
  int parts;
  int map(CUtensorMap* m, bool mn_major) const { return make_map(m, base, width, rows, parts, pitch, part, mn_major ? 64 : kRows); }
};

// The walk over an m x n result of contraction `depth`.  `shared`: what is left over of whole rounds is dealt out where it would
// leave clusters idle, which costs slabs; then a row's tiles stand side by side, since their left operand, dz, comes from
// memory and is to be read once.  `ticks`: as in the launch whose slabs this one adds to (0: the first).
Walk walk_of(int m, int n, int64_t depth, int terms, int ctas, bool shared, int segment, int ticks = 0) {
  Walk w{};
  w.m = m;
  w.n = n;
  w.bn = kRows * ctas;
  w.m_tiles = (int)over(m, kRows * ctas);
  w.n_tiles = (int)over(n, w.bn);
  w.depth_blocks = (int)over(depth, kDepth);
  w.blocks = w.depth_blocks * terms;
  w.ticks = ticks > 0 ? ticks : w.blocks;
  w.whole = w.tiles();
  w.slabs = 1;
  const int most = kSms / ctas;
  w.clusters = std::min(w.tiles(), most);
  w.segment = segment > 0 ? std::min(segment, w.blocks) : w.blocks;
  w.group = shared ? 1 : std::min(w.m_tiles, 8);
  const int left = w.tiles() % most;
  if (shared && left * 100 < 88 * most && left > 0) {
    const int64_t stages = (int64_t)left * w.ticks;
    const int c = (int)std::min<int64_t>(most, stages / 8);                                // at least eight stages each
    if (c > left && (c == most || w.tiles() < most)) {
      w.whole -= left;
      w.clusters = c;
      w.slabs = (int)((w.ticks - 1) / (stages / c)) + 2;
    }
  }
  return w;
}
int64_t slab_floats(const Walk& w, int ctas) { return (int64_t)(w.tiles() - w.whole) * w.slabs * kRows * ctas * w.bn; }

template <int CTAS, Kind KIND, bool A_MN, bool B_MN>
int launch(const CUtensorMap& a, const CUtensorMap& b, const Walk& w, Origin at_a, Origin at_b, const Epilogue& e, const WaitCtx& status,
           cudaStream_t s) {
  auto kernel = product_kernel<CTAS, KIND, A_MN, B_MN>;
  SA_CUDA_CHECK(allow_smem(kernel, kSmem));
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = CTAS;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(w.clusters * CTAS);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = kSmem;
  config.stream = s;
  config.attrs = attrs;
  config.numAttrs = 2;
  count_launch();
  SA_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a, b, w, at_a, at_b, e, status));
  return SA_OK;
}
template <Kind KIND, bool A_MN, bool B_MN>
int run(int ctas, const Operand& a, const Operand& b, const Walk& w, Origin at_a, Origin at_b, const Epilogue& e, const WaitCtx& status,
        cudaStream_t s) {
  CUtensorMap map_a, map_b;
  int st = a.map(&map_a, A_MN);
  if (st == SA_OK) st = b.map(&map_b, B_MN);
  if (st != SA_OK) return st;
  return ctas == 2 ? launch<2, KIND, A_MN, B_MN>(map_a, map_b, w, at_a, at_b, e, status, s)
                   : launch<1, KIND, A_MN, B_MN>(map_a, map_b, w, at_a, at_b, e, status, s);
}

// CTAs of a tile: two where there are rows for both.
int ctas_of(int rows) { return rows > kRows ? 2 : 1; }

int parts_of(const Problem& p) { return p.product == SA_F32 ? 3 : 1; }
int terms_of(const Problem& p) { return p.product == SA_F32 ? kTerms : 1; }
size_t bytes_of(int dtype) { return dtype == SA_F32 ? 4 : 2; }
// Sums of fp32 operands leave tensor memory every 2,048 of the contraction: its additions round towards zero.
int segment_of(const Problem& p) { return p.product == SA_F32 ? 32 : 0; }

bool in_place(int dtype, int product, const void* base, int64_t stride, int64_t rows, int64_t width) {
  return product != SA_F32 && dtype == product && (reinterpret_cast<uintptr_t>(base) & 15) == 0 && stride % 8 == 0 && (stride >= width || rows == 1);
}

// Room taken from the workspace; sizes alone when there is none.
struct Room {
  char* base;
  size_t used = 0;
  template <typename T> T* take(int64_t n) {
    T* at = base ? reinterpret_cast<T*>(base + used) : nullptr;
    used += (size_t)up(n * (int64_t)sizeof(T), 256);
    return at;
  }
};

Operand operand_of(const Problem& p, const void* base, int dtype, int64_t stride, int64_t rows, bool copy, Room* room) {
  Operand o{};
  o.rows = rows;
  o.width = p.width;
  o.parts = parts_of(p);
  if (!copy && in_place(dtype, p.product, base, stride, rows, p.width)) {
    o.base = static_cast<const uint16_t*>(base);
    o.pitch = rows == 1 ? up(p.width, 8) : stride;
    return o;
  }
  o.pitch = up(p.width, 8);
  o.part = o.pitch * rows;
  o.base = room->take<uint16_t>(o.part * o.parts);
  return o;
}

Convert convert_of(const Problem& p, const Operand& o, const void* src, int dtype, int64_t stride) {
  Convert c{};
  c.src = src;
  c.dtype = dtype;
  c.src_stride = stride;
  c.rows = (int)o.rows;
  c.width = p.width;
  c.pitch = (int)o.pitch;
  c.part = o.part;
  c.parts = o.parts;
  c.half = p.product == SA_F16;
  c.dst = const_cast<uint16_t*>(o.base);
  return c;
}
int run_convert(const Convert& c, cudaStream_t s) {
  return launch_after(convert_kernel, dim3((unsigned)over((int64_t)c.rows * (c.pitch >> 3), 256)), 256, 0, s, c);
}

struct Forward {
  Room room;
  Operand x, weight;
  int ctas;
  Walk walk;
  float2 *stats, *sums;
  float* at_target;
  unsigned int* ticket;
  Forward(const Problem& p, void* base) : room{static_cast<char*>(base)} {
    x = operand_of(p, p.x, p.x_dtype, p.x_stride, p.tokens, false, &room);
    weight = operand_of(p, p.weight, p.weight_dtype, p.weight_stride, p.vocab, false, &room);
    ctas = ctas_of(p.tokens);
    walk = walk_of(p.tokens, p.vocab, p.width, terms_of(p), ctas, false, 0);
    stats = room.take<float2>((int64_t)2 * walk.n_tiles * p.tokens);
    sums = room.take<float2>(over(p.tokens, 32));
    at_target = room.take<float>(p.tokens);
    ticket = room.take<unsigned int>(1);
  }
};

struct Backward {
  Room room;
  Operand x, weight, dz;
  float *factor, *scale, *largest, *dx_sums = nullptr, *dx_slabs = nullptr, *dw_slabs = nullptr;
  int ctas, piece;
  int64_t pitch;                 // of dx_sums
  Backward(const Problem& p, void* base) : room{static_cast<char*>(base)} {
    ctas = ctas_of(p.tokens);
    x = operand_of(p, p.x, p.x_dtype, p.x_stride, p.tokens, true, &room);
    weight = operand_of(p, p.weight, p.weight_dtype, p.weight_stride, p.vocab, false, &room);
    factor = room.take<float>(p.tokens);
    scale = room.take<float>(1);
    largest = room.take<float>(1);
    piece = piece_of(p);
    dz.rows = p.tokens;
    dz.parts = parts_of(p);
    dz.pitch = up(piece, 64);
    dz.part = dz.pitch * p.tokens;
    dz.base = room.take<uint16_t>(dz.part * dz.parts);
    pitch = up(p.width, 8);
    if (p.dx != nullptr) {
      if (piece < p.vocab) dx_sums = room.take<float>(p.tokens * pitch);
      dx_slabs = room.take<float>(slab_floats(dx_walk(p, piece), ctas));
    }
    if (p.dweight != nullptr) {
      int64_t most = slab_floats(dw_walk(p, piece), ctas_of(piece));
      if (p.vocab % piece != 0) most = std::max(most, slab_floats(dw_walk(p, p.vocab % piece), ctas_of(p.vocab % piece)));
      dw_slabs = room.take<float>(most);
    }
  }
  // Columns of a piece of the vocabulary: its dz takes up to 320 MB (16,384 tokens: 37 tiles of 256 columns, with four tiles across
  // two whole rounds of 74 clusters in dW), or 4,096 columns where that is more; of the sizes down to half of that, the one that
  // leaves the fewest clusters idle in dW.
  static int piece_of(const Problem& p) {
    const int64_t column = (int64_t)p.tokens * 2 * parts_of(p), most = std::max<int64_t>(4096, (320ll << 20) / column / 256 * 256);
    if (p.vocab <= most) return p.vocab;
    const int64_t across = over(p.width, 2 * kRows), clusters = kSms / 2, blocks = most / 256;
    int64_t best = 0, at = blocks;
    for (int64_t b = blocks; 2 * b > blocks; --b) {
      const int64_t tiles = b * across, used = tiles * 1000 / (over(tiles, clusters) * clusters);
      if (used > best) {
        best = used;
        at = b;
      }
    }
    return (int)(at * 256);
  }
  Walk dx_walk(const Problem& p, int columns) const {
    const int terms = terms_of(p);
    return walk_of(p.tokens, p.width, columns, terms, ctas, true, segment_of(p), (int)over(piece, kDepth) * terms);
  }
  Walk dw_walk(const Problem& p, int columns) const {
    return walk_of(columns, p.width, p.tokens, terms_of(p), ctas_of(columns), true, segment_of(p));
  }
};

int finish(const float* slabs, const Walk& w, int ctas, const float* scale, void* out, int dtype, int64_t pitch, cudaStream_t s) {
  if (w.whole == w.tiles()) return SA_OK;
  const int rows = kFinishThreads / (w.bn >> 2);                  // bn: 128 or 256
  return launch_after(finish_kernel, dim3(w.tiles() - w.whole, kRows * ctas / rows), kFinishThreads, 0, s, slabs, w, kRows * ctas, scale, out, dtype, pitch);
}

}  // namespace

size_t forward_bytes(const Problem& p) { return Forward(p, nullptr).room.used; }
size_t backward_bytes(const Problem& p) { return Backward(p, nullptr).room.used; }

int forward(const Problem& p, cudaStream_t s) {
  WaitCtx status;
  int st = wait_ctx(&status);
  if (st != SA_OK) return st;
  const Forward f(p, p.workspace);
  if (f.x.part != 0) st = run_convert(convert_of(p, f.x, p.x, p.x_dtype, p.x_stride), s);
  if (st == SA_OK && f.weight.part != 0) st = run_convert(convert_of(p, f.weight, p.weight, p.weight_dtype, p.weight_stride), s);
  if (st != SA_OK) return st;
  Epilogue e{};
  e.stats = f.stats;
  e.at_target = f.at_target;
  e.targets = p.targets;
  e.zeroed = f.ticket;
  e.half = p.product == SA_F16;
  st = run<kStats, false, false>(f.ctas, f.x, f.weight, f.walk, Origin{0, 0}, Origin{0, 0}, e, status, s);
  if (st != SA_OK) return st;
  return launch_after(join_kernel, dim3((unsigned)over(p.tokens, 32)), kJoinThreads, 0, s, (const float2*)f.stats, 2 * f.walk.n_tiles,
                      (const float*)f.at_target, p.targets, p.ignore_index, p.tokens, p.vocab, p.reduction, p.lse, p.loss, p.count, f.sums, f.ticket);
}

int backward(const Problem& p, cudaStream_t s) {
  WaitCtx status;
  int st = wait_ctx(&status);
  if (st != SA_OK) return st;
  Backward b(p, p.workspace);
  const bool half = p.product == SA_F16;
  if (half && p.reduction == SA_REDUCTION_NONE) {
    st = launch_after(largest_kernel, dim3(1), 1024, 0, s, p.dloss, p.targets, p.ignore_index, p.tokens, b.largest);
    if (st != SA_OK) return st;
  }
  Convert c = convert_of(p, b.x, p.x, p.x_dtype, p.x_stride);
  c.targets = p.targets;
  c.ignore_index = p.ignore_index;
  c.vocab = p.vocab;
  c.reduction = p.reduction;
  c.dloss = p.dloss;
  c.count = p.count;
  c.largest = b.largest;
  c.factor = b.factor;
  c.scale = b.scale;
  st = run_convert(c, s);
  if (st == SA_OK && b.weight.part != 0) st = run_convert(convert_of(p, b.weight, p.weight, p.weight_dtype, p.weight_stride), s);
  const float* scale = half ? b.scale : nullptr;
  for (int v0 = 0; v0 < p.vocab && st == SA_OK; v0 += b.piece) {
    const int columns = std::min(b.piece, p.vocab - v0);
    Epilogue e{};
    e.targets = p.targets;
    e.column0 = v0;
    e.lse = p.lse;
    e.factor = b.factor;
    e.p = const_cast<uint16_t*>(b.dz.base);
    e.p_pitch = b.dz.pitch;
    e.p_part = b.dz.part;
    e.parts = b.dz.parts;
    e.half = half;
    const Walk logits = walk_of(p.tokens, columns, p.width, terms_of(p), b.ctas, false, 0);
    st = run<kProbabilities, false, false>(b.ctas, b.x, b.weight, logits, Origin{0, 0}, Origin{v0, 0}, e, status, s);
    if (st != SA_OK) return st;
    Operand dz = b.dz;
    dz.width = columns;
    const bool first = v0 == 0, last = v0 + columns == p.vocab;
    if (p.dx != nullptr) {
      const Walk w = b.dx_walk(p, columns);
      Epilogue r{};
      r.half = half;
      r.out = last ? p.dx : b.dx_sums;
      r.dtype = last ? p.x_dtype : SA_F32;
      r.out_pitch = last ? p.width : b.pitch;
      r.addend = first ? nullptr : b.dx_sums;
      r.addend_pitch = b.pitch;
      r.scale = last ? scale : nullptr;
      r.slabs = b.dx_slabs;
      r.later = !first;
      st = run<kResult, false, true>(b.ctas, dz, b.weight, w, Origin{0, 0}, Origin{0, v0}, r, status, s);
      if (st == SA_OK && last) st = finish(b.dx_slabs, w, b.ctas, scale, p.dx, p.x_dtype, p.width, s);
      if (st != SA_OK) return st;
    }
    if (p.dweight != nullptr) {
      const int ctas = ctas_of(columns);
      const Walk w = b.dw_walk(p, columns);
      Epilogue r{};
      r.half = half;
      r.out = static_cast<char*>(p.dweight) + (size_t)v0 * p.width * bytes_of(p.weight_dtype);
      r.dtype = p.weight_dtype;
      r.out_pitch = p.width;
      r.scale = scale;
      r.slabs = b.dw_slabs;
      st = run<kResult, true, true>(ctas, dz, b.x, w, Origin{0, 0}, Origin{0, 0}, r, status, s);
      if (st == SA_OK) st = finish(b.dw_slabs, w, ctas, scale, r.out, p.weight_dtype, p.width, s);
    }
  }
  return st;
}

}  // namespace loss
}  // namespace sa
