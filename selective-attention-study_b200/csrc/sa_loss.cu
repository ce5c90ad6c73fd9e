// Softmax cross entropy over a vocabulary, from the hidden states and the output table, without its logits:
//
//   z = x W^T,  loss_n = log sum_v exp z_nv - z_n,t(n),  dz = (softmax(z) - [v = t]) g_n,  dx = dz W,  dW = dz^T x.
//
// Forward alone: one product whose epilogue reduces every half tile of logits to its rows' maxima and sums, and a kernel that joins
// them.
//
// Training with a sum or a mean (bf16 and fp32 products): the cotangent is one number, so the gradients are computed with the loss,
// up to that number, and no logit twice.  Tokens come in runs; of a run, the product's epilogue keeps e = exp(z - ref) in 16 bits
// beside the rows' sums s.  softmax(z) = e / s, so the rest is a scale of rows, of the result in dx = (1 / s) e W and of the
// right operand in dW = e^T (x / s).  e is 0 at the target: its part, c = softmax - 1, is added in fp32, dx_n += c W_t and dW_t +=
// the sum of c x_n over its tokens, sorted as in an embedding's gradient.  ref is the target's logit, a dot product beforehand:
// exp(z - ref) is 1 at the target and at most e^loss elsewhere, which 8 bits of exponent hold with room for 1 / s up to a loss of
// 44.  Rows beyond that are found by the sums and go through the product once more with their maximum for ref.  Three products of
// 2 N V d operations; the sums of dW over the runs stay in fp32.
//
// Otherwise (a cotangent for every token; fp16, whose five bits of exponent do not hold e; problems so small that a product costs
// less than the sums of the gradients, written and read): the backward computes the logits again in pieces of the vocabulary, turns
// a piece's into dz in 16 bits, and reads them with the two products of the gradients; what the rounding takes from dz at the target is
// added to dx in fp32, and one cotangent scales the results.  Four products in all; the sums of dx over the pieces stay in fp32.  Beyond
// 40,960 tokens (fp32: 13,568) they come in runs, so that no more than 320 MB of dz is there; the sums of dW over the runs stay in fp32.
#include "sa_loss.cuh"

#include <algorithm>
#include <type_traits>

#include "sa_layers.cuh"
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
  float *factor, *scale, *less;
};

// Eight values in `parts` parts of 16 bits, each what the ones before it leave.
__device__ __forceinline__ void store_columns(uint16_t* dst, int64_t part_stride, int parts, int half, float (&v)[8]) {
  for (int part = 0; part < parts; ++part) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = half ? pack_half(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(dst + part * part_stride) = make_uint4(w[0], w[1], w[2], w[3]);
    if (part + 1 < parts) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float first = __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
        v[i] = first == INFINITY || first == -INFINITY ? 0.f : v[i] - first;
      }
    }
  }
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
      } else if (c.reduction != SA_REDUCTION_NONE) {      // left to the results: in 8 bits it would move every token's gradient alike
        factor = 1.f;
        if (row == 0) *c.scale = c.reduction == SA_REDUCTION_MEAN && *c.count == 0.f ? 0.f : g;
      }
      c.less[row] = 0.f;
      c.factor[row] = !counts ? 0.f : t < 0 || t >= c.vocab ? NAN : factor;
    }
  }
  float v[8] = {};
  if (counts) load_columns(c.src, c.dtype, row * c.src_stride, col, c.width, v);
  store_columns(c.dst + (int64_t)row * c.pitch + col, c.part, c.parts, c.half, v);
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
                                                            int64_t ignore_index, int tokens, int vocab, int reduction, float2* lse, float* loss,
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
    sum *= ex2(between(top, from));
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i)
      if (i < n) sum += v[i].y * ex2(between(v[i].x, from));
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
      const float rest = log2_above(sum, top);
      lse[row] = make_float2(top, rest);
      const int64_t t = targets[row];
      if (t != ignore_index) {
        mine = t < 0 || t >= vocab ? NAN : (top - at_target[row]) + rest * kLn2;
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

// ---- training: what stands between the products -----------------------------------------------------------------------------------

// What e is relative to: the target's logit; +inf for a token that does not count, NaN for a target outside the vocabulary.  A warp a token.
__global__ void __launch_bounds__(256) reference_kernel(const void* x, int x_dtype, int64_t x_stride, const void* weight, int weight_dtype,
                                                        int64_t weight_stride, const int64_t* targets, int64_t ignore_index, int tokens, int vocab,
                                                        int width, float* ref, int* any, int run) {
  after_previous_kernel();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= tokens) return;
  if (lane == 0 && row % run == 0) any[row / run] = 0;
  const int64_t t = targets[row];
  float sum = 0.f;
  if (t != ignore_index && t >= 0 && t < vocab) {
    for (int col = lane * 8; col < width; col += 256) {
      float a[8], b[8];
      load_columns(x, x_dtype, row * x_stride, col, width, a);
      load_columns(weight, weight_dtype, t * weight_stride, col, width, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(a[i], b[i], sum);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (lane == 0) ref[row] = t == ignore_index ? INFINITY : t < 0 || t >= vocab ? NAN : sum;
}

struct Rows {                              // of a run of tokens
  const float2* stats;                     // (maximum, sum) of every half tile, [slots][tokens]
  int slots;
  const float* at_target;
  const float* e_target;
  const int64_t* targets;
  int64_t ignore_index;
  int tokens, vocab, width;
  float* ref;
  int* far;                                // rows whose sums left the range: the target's logit is far from the largest, or, of logits
                                           // of 10^9, from what the product makes of it
  int* any;                                // whether there is one
  int again;                               // they have been through the product once more
  float* loss;
  float* inverse;                          // 1 / s, 0 for a token that does not count
  float* less;                             // softmax - 1 at the target, in fp32; e is 0 there
  uint16_t* e;
  int64_t e_pitch, e_part;
  const void* x;
  int x_dtype;
  int64_t x_stride;
  uint16_t* scaled;                        // x / s
  int64_t scaled_pitch, scaled_part;
  int parts;
};
constexpr float kFarthest = 18446744073709551616.f;      // 2^64

// Sums of 32 tokens, their losses, and x / s.
__global__ void __launch_bounds__(kJoinThreads) rows_kernel(const Rows r) {
  after_previous_kernel();
  if (r.again && *r.any == 0) return;
  __shared__ float2 parts[kJoinWarps][32];
  __shared__ float inverse_s[32];
  __shared__ int now_s[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row0 = blockIdx.x * 32, row = row0 + lane;
  const bool inside = row < r.tokens;
  float top = -INFINITY, sum = 0.f;
  for (int i = warp; i < r.slots; i += kJoinWarps * kJoinAhead) {
    float2 v[kJoinAhead];
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k)
      v[k] = i + k * kJoinWarps < r.slots && inside ? r.stats[(int64_t)(i + k * kJoinWarps) * r.tokens + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) {
      top = fmaxf(top, v[k].x);
      sum += v[k].y;
    }
  }
  parts[warp][lane] = make_float2(top, sum);
  __syncthreads();
  if (warp == 0) {
    for (int i = 1; i < kJoinWarps; ++i) {
      top = fmaxf(top, parts[i][lane].x);
      sum += parts[i][lane].y;
    }
    const int64_t t = inside ? r.targets[row] : r.ignore_index;
    const bool counts = inside && t != r.ignore_index, good = t >= 0 && t < r.vocab;
    bool now = inside;                                             // finished here
    if (r.again) {
      now = inside && r.far[row] != 0;
    } else if (inside) {
      const bool far = counts && good && !(sum < kFarthest && sum > 1.f / kFarthest);
      r.far[row] = far;
      if (far) {
        r.ref[row] = top;
        *r.any = 1;
        now = false;
      }
    }
    float inverse = 0.f;
    if (now) {
      float loss = 0.f, at_target = 0.f;
      if (counts) {
        const float ref = r.ref[row];
        inverse = good ? 1.f / sum : NAN;
        const float e = r.e_target[row];
        loss = !good ? NAN : e > 1.f / kFarthest ? log2f(sum / e) * kLn2 : (ref - r.at_target[row]) + log2_above(sum, ref) * kLn2;
        at_target = good ? (e - sum) * inverse : NAN;
        if (good)
          for (int part = 0; part < r.parts; ++part) r.e[part * r.e_part + (int64_t)row * r.e_pitch + t] = 0;
      }
      r.loss[row] = loss;
      r.less[row] = at_target;
      r.inverse[row] = inverse;
    }
    inverse_s[lane] = inverse;
    now_s[lane] = now;
  }
  __syncthreads();
  if (r.scaled == nullptr) return;
  const int chunks = (int)(r.scaled_pitch >> 3);
  for (int i = threadIdx.x; i < 32 * chunks; i += kJoinThreads) {
    const int k = i / chunks, col = (i - k * chunks) * 8;
    if (!now_s[k]) continue;
    float v[8] = {};
    if (inverse_s[k] != 0.f) {
      load_columns(r.x, r.x_dtype, (row0 + k) * r.x_stride, col, r.width, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= inverse_s[k];
    }
    store_columns(r.scaled + (int64_t)(row0 + k) * r.scaled_pitch + col, r.scaled_part, r.parts, 0, v);
  }
}

// The loss of all tokens, summed in an order that their number alone decides.
__global__ void __launch_bounds__(1024) total_kernel(const float* losses, const int64_t* targets, int64_t ignore_index, int tokens, int reduction,
                                                     float* loss, float* count) {
  after_previous_kernel();
  __shared__ double2 warps[32];
  double a = 0.0, b = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < tokens; i += 1024) {
    a += (double)losses[i];
    b += targets[i] != ignore_index ? 1.0 : 0.0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(~0u, a, o);
    b += __shfl_xor_sync(~0u, b, o);
  }
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = make_double2(a, b);
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 32; ++i) {
    a += warps[i].x;
    b += warps[i].y;
  }
  *count = (float)b;
  *loss = (float)(reduction == SA_REDUCTION_MEAN ? a / b : a);
}

// Gradients from their sums: times the cotangent, over the tokens that count for a mean.  Eight values a thread.
__global__ void __launch_bounds__(256) scale_kernel(const float* sums, int64_t n, const float* dloss, const float* count, int reduction, void* out,
                                                    int dtype) {
  after_previous_kernel();
  float by = *dloss;
  if (reduction == SA_REDUCTION_MEAN) by = *count == 0.f ? 0.f : by / *count;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= n) return;
  const bool whole = at + 8 <= n && (reinterpret_cast<uintptr_t>(out) & 31) == 0 && (reinterpret_cast<uintptr_t>(sums) & 31) == 0;
  float v[8];
  if (whole) {
    uint32_t r[8];
    load32(sums + at, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]) * by;
    if (dtype == SA_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(v[i]);
      store32(static_cast<float*>(out) + at, r);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = dtype == SA_F16 ? pack_half(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) = make_uint4(r[0], r[1], r[2], r[3]);
    }
    return;
  }
  for (int i = 0; i < 8 && at + i < n; ++i) {
    const float f = sums[at + i] * by;
    if (dtype == SA_F32) static_cast<float*>(out)[at + i] = f;
    else if (dtype == SA_BF16) static_cast<__nv_bfloat16*>(out)[at + i] = __float2bfloat16_rn(f);
    else static_cast<__half*>(out)[at + i] = __float2half_rn(f);
  }
}

// Rows of a cut tile from its slabs, in order: a thread has four columns of a row, four slabs in flight.
constexpr int kFinishThreads = 256;
__global__ void __launch_bounds__(kFinishThreads) finish_kernel(const Epilogue e, const Walk w, int tile_rows) {
  after_previous_kernel();
  int tm, tn;
  w.place(w.whole + blockIdx.x, &tm, &tn);
  const int columns = min(w.bn, w.n - tn * w.bn), across = w.bn >> 2;
  const int in_tile = blockIdx.y * (kFinishThreads / across) + threadIdx.x / across, c = (threadIdx.x % across) * 4, row = tm * tile_rows + in_tile;
  if (row >= w.m || c >= columns) return;
  const float by = e.scale != nullptr ? e.scale[e.scale_rows ? row : 0] : 1.f;
  const float4* from = reinterpret_cast<const float4*>(e.slabs + ((int64_t)blockIdx.x * w.slabs * tile_rows + in_tile) * w.bn + c);
  const int64_t stride = (int64_t)tile_rows * w.bn / 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < w.slabs; ++k) {
    const float4 x = from[k * stride];
    v.x += x.x;
    v.y += x.y;
    v.z += x.z;
    v.w += x.w;
  }
  const int col = tn * w.bn + c;
  float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (e.cut_addend && c + i < columns) f[i] += e.addend[(int64_t)row * e.addend_pitch + col + i];
    f[i] *= by;
  }
  if (e.table != nullptr && e.table_factor[row] != 0.f) {
    const int64_t t = e.targets[row];
    if (t >= 0 && t < e.vocab) {
      float x[8];
      load_columns(e.table, e.table_dtype, t * e.table_stride, col, w.n, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = fmaf(e.table_factor[row], x[i], f[i]);
    }
  }
  const int64_t at = (int64_t)row * e.out_pitch + col;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + i >= columns) break;
    if (e.dtype == SA_F32) static_cast<float*>(e.out)[at + i] = f[i];
    else if (e.dtype == SA_BF16) static_cast<__nv_bfloat16*>(e.out)[at + i] = __float2bfloat16_rn(f[i]);
    else static_cast<__half*>(e.out)[at + i] = __float2half_rn(f[i]);
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
  const uint16_t* base = nullptr;
  int64_t rows = 0, width = 0, pitch = 0, part = 0;
  int parts = 0;
  int map(CUtensorMap* m, bool mn_major, int box) const { return make_map(m, base, width, rows, parts, pitch, part, mn_major ? 64 : box); }
};

// The walk over an m x n result of contraction `depth`.  `result`: a product of dz, which comes from memory: a row's tiles stand side by
// side, so that it is read once, and what is left of whole rounds may be cut, in parts of at least eight stages of `longest`, the
// longest contraction of the launches that add to the same slabs.  (Dealing all stages out evenly, without regard to depth,
// kept 72 clusters busy where 40 whole tiles keep 40, and took 237 us instead of 215: every tile read dz for itself.)
Walk walk_of(int m, int n, int64_t depth, int terms, int ctas, bool result, int64_t longest = 0) {
  Walk w{};
  w.m = m;
  w.n = n;
  w.bn = kRows * ctas;
  w.m_tiles = (int)over(m, kRows * ctas);
  w.n_tiles = (int)over(n, w.bn);
  w.depth_blocks = (int)over(depth, kDepth);
  w.blocks = w.depth_blocks * terms;
  w.whole = w.tiles();
  w.slabs = 1;
  const int most = kSms / ctas;
  w.clusters = std::min(w.tiles(), most);
  const bool three = terms == kTerms;      // parts of an fp32 operand
  const bool cut = three ? result || w.depth_blocks > kSegment : w.blocks > (result ? kSegmentResult : kUncutLogits);
  w.segment = !cut ? w.blocks : three ? kSegment : result ? kSegmentResult : kSegmentLogits;
  w.group = result ? 1 : std::min(w.m_tiles, 32);
  const int left = w.tiles() % most;
  if (result && left > 0) {
    const int parts = (int)std::min<int64_t>(most / left, over(longest, kDepth) * terms / 8);
    if (parts > 1) {
      w.whole -= left;
      w.slabs = parts;
      w.clusters = std::max(w.clusters, std::min(most, left * parts));
    }
  }
  return w;
}
int64_t slab_floats(const Walk& w, int ctas) { return (int64_t)(w.tiles() - w.whole) * w.slabs * kRows * ctas * w.bn; }

template <int CTAS, Kind KIND, bool A_MN, bool B_MN, bool SEGMENTS>
int launch(const CUtensorMap& a, const CUtensorMap& b, const Walk& w, Origin at_a, Origin at_b, int a_bytes, const Epilogue& e, const WaitCtx& status,
           cudaStream_t s) {
  auto kernel = product_kernel<CTAS, KIND, A_MN, B_MN, SEGMENTS>;
  constexpr size_t kBytes = KIND == kResult ? kSmemResult : kSmem;
  SA_CUDA_CHECK(allow_smem(kernel, kBytes));
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
  config.dynamicSmemBytes = kBytes;
  config.stream = s;
  config.attrs = attrs;
  config.numAttrs = 2;
  count_launch();
  SA_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, a, b, w, at_a, at_b, a_bytes, e, status));
  return SA_OK;
}
template <Kind KIND, bool A_MN, bool B_MN>
int run(int ctas, const Operand& a, const Operand& b, const Walk& w, Origin at_a, Origin at_b, const Epilogue& e, const WaitCtx& status,
        cudaStream_t s) {
  CUtensorMap map_a, map_b;
  // few tokens: a copy takes as long for a row outside the tensor as for one inside (16 tokens of 50,304 words: 33 us with 128 rows)
  const int box = ctas == 1 ? std::min(kRows, (int)up(w.m, 8)) : kRows;
  int st = a.map(&map_a, A_MN, box);
  if (st == SA_OK) st = b.map(&map_b, B_MN, kRows);
  if (st != SA_OK) return st;
  const int a_bytes = A_MN ? kOperand : box * kDepth * 2;
  auto go = [&](auto segments) {
    constexpr bool SEGMENTS = decltype(segments)::value;
    return ctas == 2 ? launch<2, KIND, A_MN, B_MN, SEGMENTS>(map_a, map_b, w, at_a, at_b, a_bytes, e, status, s)
                     : launch<1, KIND, A_MN, B_MN, SEGMENTS>(map_a, map_b, w, at_a, at_b, a_bytes, e, status, s);
  };
  return w.segment < w.blocks ? go(std::true_type()) : go(std::false_type());
}

// CTAs of a tile: two where there are rows for both.
int ctas_of(int rows) { return rows > kRows ? 2 : 1; }

int parts_of(const Problem& p) { return p.product == SA_F32 ? 3 : 1; }
int terms_of(const Problem& p) { return p.product == SA_F32 ? kTerms : 1; }
size_t bytes_of(int dtype) { return dtype == SA_F32 ? 4 : 2; }

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
// The same values as one matrix of a plain type: as the products have them, or, of three parts, as they were given.
struct Matrix {
  const void* base;
  int dtype;
  int64_t stride;
};
Matrix matrix_of(const Problem& p, const Operand& o, const void* given, int dtype, int64_t stride) {
  return o.parts == 1 ? Matrix{o.base, p.product, o.pitch} : Matrix{given, dtype, stride};
}
int run_convert(const Convert& c, cudaStream_t s) {
  return launch_after(convert_kernel, dim3((unsigned)over((int64_t)c.rows * (c.pitch >> 3), 256)), 256, 0, s, c);
}

constexpr int64_t kMost = 320ll << 20;     // bytes of what stands for logits at a time, where the rest of a call does not ask for more

struct Forward {
  Room room;
  Operand x, weight;
  int ctas, run;
  float2 *stats, *sums;
  float *at_target, *losses = nullptr;       // losses: of several runs
  unsigned int* ticket;
  Forward(const Problem& p, void* base) : room{static_cast<char*>(base)} {
    x = operand_of(p, p.x, p.x_dtype, p.x_stride, p.tokens, false, &room);
    weight = operand_of(p, p.weight, p.weight_dtype, p.weight_stride, p.vocab, false, &room);
    ctas = ctas_of(p.tokens);
    run = run_of(p);
    stats = room.take<float2>((int64_t)2 * walk_of(run, p.vocab, p.width, terms_of(p), ctas, false).n_tiles * run);
    sums = room.take<float2>(over(run, 32));
    at_target = room.take<float>(run);
    if (run < p.tokens && p.reduction != SA_REDUCTION_NONE) losses = room.take<float>(p.tokens);
    ticket = room.take<unsigned int>(1);
  }
  // Tokens whose half tiles are kept at a time: up to 65,536 (200 MB of 50,304 words), of many words fewer.
  static int run_of(const Problem& p) {
    const int64_t token = over(p.vocab, kRows * ctas_of(p.tokens)) * 2 * sizeof(float2);
    return (int)std::min<int64_t>(p.tokens, std::max<int64_t>(256, std::min<int64_t>(65536, kMost / token / 256 * 256)));
  }
};

struct Backward {
  Room room;
  Operand x, weight, dz;
  float *factor, *scale, *largest, *less, *dx_sums = nullptr, *dx_slabs = nullptr, *dw_sums = nullptr, *dw_slabs = nullptr;
  int ctas, run, piece;
  int64_t pitch;                 // of dx_sums and dw_sums
  Backward(const Problem& p, void* base) : room{static_cast<char*>(base)} {
    run = run_of(p);
    ctas = ctas_of(run);
    x = operand_of(p, p.x, p.x_dtype, p.x_stride, p.tokens, true, &room);
    weight = operand_of(p, p.weight, p.weight_dtype, p.weight_stride, p.vocab, false, &room);
    factor = room.take<float>(p.tokens);
    scale = room.take<float>(1);
    largest = room.take<float>(1);
    less = room.take<float>(p.tokens);
    piece = piece_of(p, run);
    dz.parts = dz_parts(p);
    dz.pitch = up(piece, 64);
    dz.part = dz.pitch * run;
    dz.base = room.take<uint16_t>(dz.part * dz.parts);
    pitch = up(p.width, 8);
    int64_t dx = 0, dw = 0;      // slabs of the largest of the products
    for (int tokens : {run, p.tokens % run})
      if (tokens > 0) {
        dx = std::max(dx, slab_floats(dx_walk(p, tokens, piece), ctas));
        for (int columns : {piece, p.vocab % piece})
          if (columns > 0) dw = std::max(dw, slab_floats(dw_walk(p, columns, tokens), ctas_of(columns)));
      }
    if (p.dx != nullptr) {
      if (piece < p.vocab) dx_sums = room.take<float>(run * pitch);
      dx_slabs = room.take<float>(dx);
    }
    if (p.dweight != nullptr) {
      if (run < p.tokens) dw_sums = room.take<float>(p.vocab * pitch);
      dw_slabs = room.take<float>(dw);
    }
  }
  // Of few tokens dz is kept in two parts for dW, whose product is bound by what it writes up to here (128 tokens of 50,304 words of 768
  // 107 us a call, with one part 105): the bits of one would make most of its error (2.3e-3 to 2.9e-3 against 64 bits, 1.7e-3 with
  // two; fp16 2.6e-4 to 4e-4 and 2.1e-4).  dx has the first part.
  static int dz_parts(const Problem& p) { return p.product != SA_F32 && p.tokens <= kRows ? 2 : parts_of(p); }
  // Tokens of a run: as many as leave a piece of the vocabulary 4,096 columns, or all that there are.  The sums of dW over the runs are kept
  // in fp32; fewer columns instead would have those of dx read and written more often (131,072 tokens of 50,304 words of 1,024: 42.8 ms in
  // four runs, 43.2 with 4,096 columns of all tokens in 1.2 GB more).
  static int run_of(const Problem& p) {
    const int64_t row = up(std::min(p.vocab, 4096), 64) * 2 * dz_parts(p), most = kMost / row / 256 * 256;
    return p.tokens <= most ? p.tokens : (int)up(over(p.tokens, over(p.tokens, most)), 256);
  }
  // Columns of a piece of the vocabulary: its dz takes up to 320 MB (16,384 tokens: 37 tiles of 256 columns, with four tiles across
  // two whole rounds of 74 clusters in dW); of the sizes down to half of that, the one that leaves the fewest clusters idle in dW.
  static int piece_of(const Problem& p, int run) {
    const int64_t column = (int64_t)run * 2 * dz_parts(p), most = kMost / column / 256 * 256;
    if (up(p.vocab, 64) * column <= kMost) return p.vocab;
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
  Walk dx_walk(const Problem& p, int tokens, int columns) const { return walk_of(tokens, p.width, columns, terms_of(p), ctas, true, piece); }
  Walk dw_walk(const Problem& p, int columns, int tokens) const {
    return walk_of(columns, p.width, tokens, p.product == SA_F32 ? kTerms : dz_parts(p), ctas_of(columns), true, tokens);
  }
};

int finish(const Epilogue& e, const Walk& w, int ctas, cudaStream_t s) {
  if (w.whole == w.tiles()) return SA_OK;
  const int rows = kFinishThreads / (w.bn >> 2);                  // bn: 128 or 256
  return launch_after(finish_kernel, dim3(w.tiles() - w.whole, kRows * ctas / rows), kFinishThreads, 0, s, (const Epilogue)e, (const Walk)w, kRows * ctas);
}

// A product into a result.
template <bool A_MN, bool B_MN>
int run_result(int ctas, const Operand& a, const Operand& b, const Walk& w, Origin at_a, Origin at_b, Epilogue e,
               const WaitCtx& status, cudaStream_t s) {
  e.aligned = ((reinterpret_cast<uintptr_t>(e.out) | (uintptr_t)e.out_pitch * bytes_of(e.dtype)) & (e.dtype == SA_F32 ? 31 : 15)) == 0;
  e.addend_first = ((reinterpret_cast<uintptr_t>(e.addend) | (uintptr_t)e.addend_pitch * 4) & 31) == 0;
  return run<kResult, A_MN, B_MN>(ctas, a, b, w, at_a, at_b, e, status, s);
}

struct Train {
  Room room;
  Operand x, weight, e, scaled;
  int run;                       // tokens of a run
  float *ref, *losses, *less, *e_target, *inverse, *dx_slabs = nullptr, *dw_slabs = nullptr;
  int *far, *any;                // of tokens, of runs
  void* sorted = nullptr;        // of the targets
  float2* stats;
  float* at_target;
  Train(const Problem& p, void* base) : room{static_cast<char*>(base)} {
    x = operand_of(p, p.x, p.x_dtype, p.x_stride, p.tokens, false, &room);
    weight = operand_of(p, p.weight, p.weight_dtype, p.weight_stride, p.vocab, false, &room);
    run = run_of(p);
    ref = room.take<float>(p.tokens);
    losses = room.take<float>(p.tokens);
    less = room.take<float>(p.tokens);
    far = room.take<int>(p.tokens);
    any = room.take<int>(over(p.tokens, run));
    at_target = room.take<float>(run);
    e_target = room.take<float>(run);
    inverse = room.take<float>(run);
    stats = room.take<float2>((int64_t)2 * logits_walk(p, run).n_tiles * run);
    e.parts = scaled.parts = parts_of(p);
    e.rows = scaled.rows = run;
    e.width = p.vocab;
    e.pitch = up(p.vocab, 64);
    e.part = e.pitch * run;
    e.base = room.take<uint16_t>(e.part * e.parts);
    scaled.width = p.width;
    scaled.pitch = up(p.width, 8);
    scaled.part = scaled.pitch * run;
    if (p.dweight_sums != nullptr) {
      scaled.base = room.take<uint16_t>(scaled.part * scaled.parts);
      dw_slabs = room.take<float>(slab_floats(dw_walk(p, run), ctas_of(p.vocab)));
      sorted = room.take<char>((int64_t)embed::sum_rows_bytes(p.tokens, p.vocab, p.width));
    }
    if (p.dx_sums != nullptr) {
      int64_t most = slab_floats(dx_walk(p, run), ctas_of(run));
      if (p.tokens % run != 0) most = std::max(most, slab_floats(dx_walk(p, p.tokens % run), ctas_of(p.tokens % run)));
      dx_slabs = room.take<float>(most);
    }
  }
  // Tokens of a run: e takes up to 512 MB, or 256 tokens' where that is more (see prefers_train); of the sizes down to half of that, the one whose dx takes
  // the fewest rounds of the clusters (16,384 tokens of 50,304 words, four tiles across: three runs of 20 tiles of tokens and one of
  // 4 take 3.5 rounds, four runs of 16 take 4).
  static constexpr int64_t kMost = 512ll << 20;
  static int run_of(const Problem& p) {
    const int64_t row = up(p.vocab, 64) * 2 * parts_of(p), most = std::max<int64_t>(256, kMost / row / 256 * 256) / 256;
    if (p.tokens <= most * 256) return p.tokens;
    const int64_t across = over(p.width, 2 * kRows), clusters = kSms / 2, all = over(p.tokens, 256);
    auto rounds = [&](int64_t blocks) {                          // in thousandths, as walk_of cuts what is left of whole ones
      const int64_t tiles = blocks * across, left = tiles % clusters;
      return tiles / clusters * 1000 + (left > 0 ? 1000 / (clusters / left) : 0) + (blocks > 0 ? 50 : 0);
    };
    int64_t best = INT64_MAX, at = most;
    for (int64_t b = most; 2 * b > most; --b) {
      const int64_t cost = all / b * rounds(b) + rounds(all % b);
      if (cost < best) {
        best = cost;
        at = b;
      }
    }
    return (int)(at * 256);
  }
  Walk logits_walk(const Problem& p, int tokens) const { return walk_of(tokens, p.vocab, p.width, terms_of(p), ctas_of(run), false); }
  Walk dx_walk(const Problem& p, int tokens) const { return walk_of(tokens, p.width, p.vocab, terms_of(p), ctas_of(tokens), true, p.vocab); }
  Walk dw_walk(const Problem& p, int tokens) const { return walk_of(p.vocab, p.width, tokens, terms_of(p), ctas_of(p.vocab), true, run); }
};

}  // namespace

size_t forward_bytes(const Problem& p) { return Forward(p, nullptr).room.used; }
size_t backward_bytes(const Problem& p) { return Backward(p, nullptr).room.used; }
size_t train_bytes(const Problem& p) { return Train(p, nullptr).room.used; }

int forward(const Problem& p, cudaStream_t s) {
  WaitCtx status;
  int st = wait_ctx(&status);
  if (st != SA_OK) return st;
  const Forward f(p, p.workspace);
  if (f.x.part != 0) st = run_convert(convert_of(p, f.x, p.x, p.x_dtype, p.x_stride), s);
  if (st == SA_OK && f.weight.part != 0) st = run_convert(convert_of(p, f.weight, p.weight, p.weight_dtype, p.weight_stride), s);
  if (st != SA_OK) return st;
  for (int n0 = 0; n0 < p.tokens && st == SA_OK; n0 += f.run) {
    const int tokens = std::min(f.run, p.tokens - n0);
    const Walk walk = walk_of(tokens, p.vocab, p.width, terms_of(p), f.ctas, false);
    Epilogue e{};
    e.stats = f.stats;
    e.at_target = f.at_target;
    e.targets = p.targets + n0;
    e.zeroed = f.ticket;
    e.half = p.product == SA_F16;
    st = run<kStats, false, false>(f.ctas, f.x, f.weight, walk, Origin{n0, 0}, Origin{0, 0}, e, status, s);
    if (st != SA_OK) return st;
    const bool each = f.losses != nullptr || p.reduction == SA_REDUCTION_NONE;
    st = launch_after(join_kernel, dim3((unsigned)over(tokens, 32)), kJoinThreads, 0, s, (const float2*)f.stats, 2 * walk.n_tiles, (const float*)f.at_target,
                      e.targets, p.ignore_index, tokens, p.vocab, each ? (int)SA_REDUCTION_NONE : p.reduction, reinterpret_cast<float2*>(p.lse) + n0,
                      each ? (f.losses != nullptr ? f.losses : p.loss) + n0 : p.loss, p.count, f.sums, f.ticket);
  }
  if (st != SA_OK || f.losses == nullptr) return st;
  return launch_after(total_kernel, dim3(1), 1024, 0, s, (const float*)f.losses, p.targets, p.ignore_index, p.tokens, p.reduction, p.loss, p.count);
}

// A product (and a copy of the table in the products' parts) saved against the fp32 sums of the gradients, of the table's in every run of
// tokens, and eight more launches: the smaller of both estimates, in us at 1.4 PFLOP/s (fp32: 0.75) and 6.4 TB/s.  Near the border it
// leans to the second way, whose dW is the more exact one.  Measured, the logits computed again and the gradients with the loss, bf16: 64
// tokens of 50,304 words of 1,024 132 and 203 us, 1,024 of 50,304 of 768 252 and 264, 2,048 462 and 481 (it takes 481), 4,096 1,181 and
// 1,007, 16,384 of 1,024 4,480 and 4,200, 4,096 of 262,144 of 256 (four runs) 2,484 and 2,481, of 500,000 4,829 and 6,089; fp32: 1,024 of 8,000 of 512 198 and 189, 512 of
// 32,000 of 768 559 and 472, 2,048 of 200,000 of 128 3,446 and 3,671 (it takes 3,671).
bool prefers_train(const Problem& p) {
  if (p.reduction == SA_REDUCTION_NONE || p.product == SA_F16) return false;
  const double values = (double)p.vocab * p.width, tokens = (double)up(p.tokens, kRows);
  double saved = 2.0 * tokens * values * terms_of(p) / (p.product == SA_F32 ? 0.75e9 : 1.4e9);
  if (!in_place(p.weight_dtype, p.product, p.weight, p.weight_stride, p.vocab, p.width)) saved += values * (bytes_of(p.weight_dtype) + 2 * parts_of(p)) / 6.4e6;
  const int64_t run = Train::run_of(p);
  if (run * up(p.vocab, 64) * 2 * parts_of(p) > Train::kMost) return false;
  return saved > 8.0 * (values * (double)over(p.tokens, run) + tokens * p.width) / 6.4e6 + 50.0;
}

int train(const Problem& p, cudaStream_t s) {
  WaitCtx status;
  int st = wait_ctx(&status);
  if (st != SA_OK) return st;
  const Train t(p, p.workspace);
  if (t.x.part != 0) st = run_convert(convert_of(p, t.x, p.x, p.x_dtype, p.x_stride), s);
  if (st == SA_OK && t.weight.part != 0) st = run_convert(convert_of(p, t.weight, p.weight, p.weight_dtype, p.weight_stride), s);
  const Matrix x = matrix_of(p, t.x, p.x, p.x_dtype, p.x_stride), weight = matrix_of(p, t.weight, p.weight, p.weight_dtype, p.weight_stride);
  if (st == SA_OK)
    st = launch_after(reference_kernel, dim3((unsigned)over(p.tokens, 8)), 256, 0, s, x.base, x.dtype, x.stride, weight.base, weight.dtype, weight.stride,
                      p.targets, p.ignore_index, p.tokens, p.vocab, p.width, t.ref, t.any, t.run);
  for (int n0 = 0; n0 < p.tokens && st == SA_OK; n0 += t.run) {
    const int tokens = std::min(t.run, p.tokens - n0);
    const bool first = n0 == 0, last = n0 + tokens == p.tokens;
    const Walk logits = t.logits_walk(p, tokens);
    Epilogue e{};
    e.stats = t.stats;
    e.at_target = t.at_target;
    e.e_target = t.e_target;
    e.targets = p.targets + n0;
    e.ref = t.ref + n0;
    e.p = const_cast<uint16_t*>(t.e.base);
    e.p_pitch = t.e.pitch;
    e.p_part = t.e.part;
    e.parts = t.e.parts;
    Rows r{};
    r.stats = t.stats;
    r.slots = 2 * logits.n_tiles;
    r.at_target = t.at_target;
    r.e_target = t.e_target;
    r.targets = e.targets;
    r.ignore_index = p.ignore_index;
    r.tokens = tokens;
    r.vocab = p.vocab;
    r.width = p.width;
    r.ref = t.ref + n0;
    r.far = t.far + n0;
    r.any = t.any + n0 / t.run;
    r.loss = t.losses + n0;
    r.inverse = t.inverse;
    r.less = t.less + n0;
    r.e = e.p;
    r.e_pitch = e.p_pitch;
    r.e_part = e.p_part;
    r.x = static_cast<const char*>(x.base) + (size_t)n0 * x.stride * bytes_of(x.dtype);
    r.x_dtype = x.dtype;
    r.x_stride = x.stride;
    r.scaled = const_cast<uint16_t*>(t.scaled.base);
    r.scaled_pitch = t.scaled.pitch;
    r.scaled_part = t.scaled.part;
    r.parts = e.parts;
    for (int again = 0; again < 2 && st == SA_OK; ++again) {       // the second time for rows that are far, where there are any
      e.only = again ? r.far : nullptr;
      e.any = again ? r.any : nullptr;
      r.again = again;
      st = run<kBoth, false, false>(ctas_of(t.run), t.x, t.weight, logits, Origin{n0, 0}, Origin{0, 0}, e, status, s);
      if (st == SA_OK) st = launch_after(rows_kernel, dim3((unsigned)over(tokens, 32)), kJoinThreads, 0, s, (const Rows)r);
    }
    Operand left = t.e, right = t.scaled;
    left.rows = right.rows = tokens;
    if (p.dx_sums != nullptr && st == SA_OK) {
      const int ctas = ctas_of(tokens);
      const Walk w = t.dx_walk(p, tokens);
      Epilogue o{};
      o.out = p.dx_sums + (int64_t)n0 * p.width;
      o.dtype = SA_F32;
      o.out_pitch = p.width;
      o.scale = t.inverse;
      o.scale_rows = 1;
      o.slabs = t.dx_slabs;
      o.table = weight.base;
      o.table_dtype = weight.dtype;
      o.table_stride = weight.stride;
      o.table_factor = t.less + n0;
      o.targets = e.targets;
      o.vocab = p.vocab;
      st = run_result<false, true>(ctas, left, t.weight, w, Origin{0, 0}, Origin{0, 0}, o, status, s);
      if (st == SA_OK) st = finish(o, w, ctas, s);
    }
    if (p.dweight_sums != nullptr && st == SA_OK) {
      const int ctas = ctas_of(p.vocab);
      const Walk w = t.dw_walk(p, tokens);
      Epilogue o{};
      o.out = p.dweight_sums;
      o.dtype = SA_F32;
      o.out_pitch = p.width;
      o.addend = first ? nullptr : p.dweight_sums;
      o.addend_pitch = p.width;
      o.slabs = t.dw_slabs;
      o.later = !first;
      st = run_result<true, true>(ctas, left, right, w, Origin{0, 0}, Origin{0, 0}, o, status, s);
      if (st == SA_OK && last) st = finish(o, w, ctas, s);
    }
  }
  if (p.dweight_sums != nullptr && st == SA_OK) {
    embed::RowSums o{};
    o.idx = p.targets;
    o.skip = p.ignore_index;
    o.tokens = p.tokens;
    o.vocab = p.vocab;
    o.width = p.width;
    o.dy = x.base;
    o.dtype = x.dtype;
    o.dy_stride = x.stride;
    o.factor = t.less;
    o.scale = 1.f;
    o.out = p.dweight_sums;
    o.out_dtype = SA_F32;
    o.add = true;
    o.workspace = t.sorted;
    st = embed::sum_rows(o, s);
  }
  if (st != SA_OK) return st;
  return launch_after(total_kernel, dim3(1), 1024, 0, s, (const float*)t.losses, p.targets, p.ignore_index, p.tokens, p.reduction, p.loss, p.count);
}

int scale(const Problem& p, cudaStream_t s) {
  int st = SA_OK;
  const int64_t n[2] = {(int64_t)p.tokens * p.width, (int64_t)p.vocab * p.width};
  const float* const from[2] = {p.dx_sums, p.dweight_sums};
  void* const to[2] = {p.dx, p.dweight};
  const int types[2] = {p.x_dtype, p.weight_dtype};
  for (int i = 0; i < 2 && st == SA_OK; ++i)
    if (to[i] != nullptr)
      st = launch_after(scale_kernel, dim3((unsigned)over(over(n[i], 8), 256)), 256, 0, s, from[i], n[i], p.dloss, (const float*)p.count, p.reduction,
                        to[i], types[i]);
  return st;
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
  c.less = b.less;
  st = run_convert(c, s);
  if (st == SA_OK && b.weight.part != 0) st = run_convert(convert_of(p, b.weight, p.weight, p.weight_dtype, p.weight_stride), s);
  const float* scale = half || p.reduction != SA_REDUCTION_NONE ? b.scale : nullptr;
  const Matrix weight = matrix_of(p, b.weight, p.weight, p.weight_dtype, p.weight_stride);
  for (int n0 = 0; n0 < p.tokens && st == SA_OK; n0 += b.run) {
    const int tokens = std::min(b.run, p.tokens - n0);
    for (int v0 = 0; v0 < p.vocab && st == SA_OK; v0 += b.piece) {
      const int columns = std::min(b.piece, p.vocab - v0);
      Epilogue e{};
      e.targets = p.targets + n0;
      e.column0 = v0;
      e.lse = reinterpret_cast<const float2*>(p.lse) + n0;
      e.factor = b.factor + n0;
      e.p = const_cast<uint16_t*>(b.dz.base);
      e.p_pitch = b.dz.pitch;
      e.p_part = b.dz.part;
      e.parts = b.dz.parts;
      e.half = half;
      e.scale = scale;
      e.less = b.less + n0;
      const Walk logits = walk_of(tokens, columns, p.width, terms_of(p), b.ctas, false);
      st = run<kProbabilities, false, false>(b.ctas, b.x, b.weight, logits, Origin{n0, 0}, Origin{v0, 0}, e, status, s);
      if (st != SA_OK) return st;
      Operand dz = b.dz;
      dz.rows = tokens;
      dz.width = columns;
      if (p.dx != nullptr) {
        const bool first = v0 == 0, last = v0 + columns == p.vocab;
        const Walk w = b.dx_walk(p, tokens, columns);
        Epilogue r{};
        r.half = half;
        r.out = last ? static_cast<char*>(p.dx) + (size_t)n0 * p.width * bytes_of(p.x_dtype) : static_cast<void*>(b.dx_sums);
        r.dtype = last ? p.x_dtype : SA_F32;
        r.out_pitch = last ? p.width : b.pitch;
        r.addend = first ? nullptr : b.dx_sums;
        r.addend_pitch = b.pitch;
        r.scale = last ? scale : nullptr;
        r.table = last && b.dz.parts < 3 ? weight.base : nullptr;
        r.table_dtype = weight.dtype;
        r.table_stride = weight.stride;
        r.table_factor = b.less + n0;
        r.targets = e.targets;
        r.vocab = p.vocab;
        r.slabs = b.dx_slabs;
        r.later = !first;
        st = run_result<false, true>(b.ctas, dz, b.weight, w, Origin{0, 0}, Origin{0, v0}, r, status, s);
        if (st == SA_OK && last) st = finish(r, w, b.ctas, s);
        if (st != SA_OK) return st;
      }
      if (p.dweight != nullptr) {
        const bool first = n0 == 0, last = n0 + tokens == p.tokens;
        const int ctas = ctas_of(columns);
        const Walk w = b.dw_walk(p, columns, tokens);
        Epilogue r{};
        r.half = half;
        r.out = last ? static_cast<char*>(p.dweight) + (size_t)v0 * p.width * bytes_of(p.weight_dtype) : static_cast<void*>(b.dw_sums + v0 * b.pitch);
        r.dtype = last ? p.weight_dtype : SA_F32;
        r.out_pitch = last ? p.width : b.pitch;
        r.addend = first ? nullptr : b.dw_sums + v0 * b.pitch;
        r.addend_pitch = b.pitch;
        r.cut_addend = !first;
        r.scale = last ? scale : nullptr;
        r.slabs = b.dw_slabs;
        st = run_result<true, true>(ctas, dz, b.x, w, Origin{0, 0}, Origin{0, n0}, r, status, s);
        if (st == SA_OK) st = finish(r, w, ctas, s);
      }
    }
  }
  return st;
}

}  // namespace loss
}  // namespace sa
