// Layer norm, after a residual sum or alone, and its gradient.  s = x + branch, h = (s - mean) / sqrt(var + eps), y = h w + b;
//   ds = r (g - mean(g) - h mean(g h)) + ds_out,  g = dy w;   dw = sum over rows of dy h,   db = sum over rows of dy.
//
// Both directions are bound by memory: a row stays in the registers of one warp (up to 512 values) or of one CTA between its only
// load and its only store; mean and variance are two sums over the registers, the second about the mean.  The backward's CTAs walk
// over rows and keep their columns' sums for dw and db in registers; a second kernel joins the CTAs' sums in their order.
#include "sa_layers.cuh"

#include <algorithm>

namespace sa {
namespace norm {
namespace {

// Sums of two values over the T threads of a row: a warp, or the CTA.  `buffer` is one of two that rows take in turn, so one barrier
// a sum is enough.
template <int T>
__device__ __forceinline__ float2 row_sum(float2 v, float2 (*buffer)[32], int& turn) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(~0u, v.x, o);
    v.y += __shfl_xor_sync(~0u, v.y, o);
  }
  if constexpr (T > 32) {
    float2* b = buffer[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
    __syncthreads();
    v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
      v.x += b[i].x;
      v.y += b[i].y;
    }
  }
  return v;
}

template <int T> constexpr int kBlock = T < 128 ? 128 : T;
template <int T> constexpr int kRowsOf = kBlock<T> / T;

template <int T, int NV, bool VEC>
__global__ void __launch_bounds__(kBlock<T>) forward_kernel(const sa_norm p) {
  tc::after_previous_kernel();
  __shared__ float2 buffer[2][32];
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * kRowsOf<T> + threadIdx.x / T;
  if (row >= p.rows) return;                                     // a whole warp, or the whole CTA
  int turn = 0;
  float s[NV][8];
  load_row<NV, T, VEC>(s, p.x, p.x_dtype, row * p.x_stride, p.width, t);
  if (p.branch != nullptr) {
    float b[NV][8];
    load_row<NV, T, VEC>(b, p.branch, p.branch_dtype, row * p.branch_stride, p.width, t);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[c][i] = rounded_to(s[c][i] + b[c][i], p.x_dtype);
    store_row<NV, T, VEC>(s, p.sum, p.x_dtype, row * p.width, p.width, t);
  }
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (column_of<T, VEC>(c, i, t) < p.width) sum.x += s[c][i];
  const float mean = row_sum<T>(sum, buffer, turn).x / (float)p.width;
  sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[c][i] -= mean;
      if (column_of<T, VEC>(c, i, t) < p.width) sum.x += s[c][i] * s[c][i];
    }
  const float r = 1.f / sqrtf(row_sum<T>(sum, buffer, turn).x / (float)p.width + p.eps);
  if (t == 0 && p.stats != nullptr) {
    p.stats[2 * row] = mean;
    p.stats[2 * row + 1] = r;
  }
  if (p.weight != nullptr) {
    float w[NV][8];
    load_row<NV, T, VEC>(w, p.weight, p.weight_dtype, 0, p.width, t);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[c][i] = s[c][i] * r * w[c][i];
  } else {
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[c][i] *= r;
  }
  if (p.bias != nullptr) {
    float b[NV][8];
    load_row<NV, T, VEC>(b, p.bias, p.weight_dtype, 0, p.width, t);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[c][i] += b[c][i];
  }
  store_row<NV, T, VEC>(s, p.y, p.y_dtype, row * p.width, p.width, t);
}

// `sums`: (CTAs, 2, width), the parts of dw and db; null when neither is asked for.
template <int T, int NV, bool VEC, bool BIAS>
__global__ void __launch_bounds__(kBlock<T>) backward_kernel(const sa_norm p, float* sums) {
  tc::after_previous_kernel();
  __shared__ float2 buffer[2][32];
  const int t = threadIdx.x % T, lane_row = threadIdx.x / T;
  int turn = 0;
  float dw[NV][8], db[BIAS ? NV : 1][8];
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[c][i] = 0.f;
      if (BIAS) db[c][i] = 0.f;
    }
  for (int64_t row = (int64_t)blockIdx.x * kRowsOf<T> + lane_row; row < p.rows; row += (int64_t)gridDim.x * kRowsOf<T>) {
    float h[NV][8], g[NV][8];
    load_row<NV, T, VEC>(h, p.x, p.x_dtype, row * p.x_stride, p.width, t);
    load_row<NV, T, VEC>(g, p.dy, p.y_dtype, row * p.dy_stride, p.width, t);
    const float2 stats = make_float2(p.stats[2 * row], p.stats[2 * row + 1]);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[c][i] = (h[c][i] - stats.x) * stats.y;
        dw[c][i] += g[c][i] * h[c][i];
        if (BIAS) db[c][i] += g[c][i];
      }
    if (p.weight != nullptr) {
      float w[NV][8];
      load_row<NV, T, VEC>(w, p.weight, p.weight_dtype, 0, p.width, t);
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) g[c][i] *= w[c][i];
    }
    float2 m = make_float2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (column_of<T, VEC>(c, i, t) < p.width) {
          m.x += g[c][i];
          m.y += g[c][i] * h[c][i];
        }
    m = row_sum<T>(m, buffer, turn);
    m.x /= (float)p.width;
    m.y /= (float)p.width;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) g[c][i] = stats.y * (g[c][i] - m.x - h[c][i] * m.y);
    if (p.dsum != nullptr) {
      load_row<NV, T, VEC>(h, p.dsum, p.x_dtype, row * p.dsum_stride, p.width, t);
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) g[c][i] += h[c][i];
    }
    store_row<NV, T, VEC>(g, p.dx, p.x_dtype, row * p.width, p.width, t);
    if (p.dbranch != nullptr) store_row<NV, T, VEC>(g, p.dbranch, p.branch_dtype, row * p.width, p.width, t);
  }
  if (sums == nullptr) return;
  if constexpr (kRowsOf<T> > 1) {                                // the CTA's warps, in their order
    __shared__ float part[kRowsOf<T> - 1][T * NV * 8 * (BIAS ? 2 : 1)];
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (lane_row > 0) {
          part[lane_row - 1][(c * 8 + i) * T + t] = dw[c][i];
          if (BIAS) part[lane_row - 1][((NV + c) * 8 + i) * T + t] = db[c][i];
        }
    __syncthreads();
    if (lane_row > 0) return;
    for (int k = 0; k < kRowsOf<T> - 1; ++k)
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dw[c][i] += part[k][(c * 8 + i) * T + t];
          if (BIAS) db[c][i] += part[k][((NV + c) * 8 + i) * T + t];
        }
  }
  float* mine = sums + (int64_t)blockIdx.x * (BIAS ? 2 : 1) * p.width;
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int col = column_of<T, VEC>(c, i, t);
      if (col >= p.width) continue;
      mine[col] = dw[c][i];
      if (BIAS) mine[p.width + col] = db[c][i];
    }
}

// Columns of the parameters' gradients: 32 a CTA, whose 16 warps take the parts in turn.
__global__ void __launch_bounds__(512) parameters_kernel(const float* sums, int parts, int width, int columns, int dtype, void* dweight, void* dbias) {
  tc::after_previous_kernel();
  __shared__ float by_warp[16][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (col < columns) {
#pragma unroll 8
    for (int i = warp; i < parts; i += 16) v += sums[(int64_t)i * columns + col];
  }
  by_warp[warp][lane] = v;
  __syncthreads();
  if (warp != 0 || col >= columns) return;
  for (int i = 1; i < 16; ++i) v += by_warp[i][lane];
  void* out = col < width ? dweight : dbias;
  if (out == nullptr) return;
  const int at = col < width ? col : col - width;
  if (dtype == SA_F32) static_cast<float*>(out)[at] = v;
  else if (dtype == SA_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else static_cast<__half*>(out)[at] = __float2half_rn(v);
}

bool vectors(const sa_norm& p, bool backward) {
  const int64_t w = p.width;
  bool ok = w % 8 == 0 && eights(p.x, p.x_dtype, p.x_stride, p.rows) && eights(p.weight, p.weight_dtype, 0, 1);
  if (!backward)
    return ok && eights(p.branch, p.branch_dtype, p.branch_stride, p.rows) && eights(p.bias, p.weight_dtype, 0, 1) && eights(p.sum, p.x_dtype, w, 1) &&
           eights(p.y, p.y_dtype, w, 1);
  return ok && eights(p.dy, p.y_dtype, p.dy_stride, p.rows) && eights(p.dsum, p.x_dtype, p.dsum_stride, p.rows) && eights(p.dx, p.x_dtype, w, 1) &&
         eights(p.dbranch, p.branch_dtype, w, 1);
}

// Threads and values of a row by its width: f(threads, chunks of 8 a thread).
template <typename F>
int by_width(int width, F f) {
  using std::integral_constant;
#define SA_NORM_CASE(most, threads, chunks) \
  if (width <= most) return f(integral_constant<int, threads>(), integral_constant<int, chunks>())
  SA_NORM_CASE(256, 32, 1);
  SA_NORM_CASE(512, 32, 2);
  SA_NORM_CASE(1024, 128, 1);
  SA_NORM_CASE(2048, 128, 2);
  SA_NORM_CASE(4096, 256, 2);
  SA_NORM_CASE(8192, 512, 2);
  SA_NORM_CASE(16384, 1024, 2);
#undef SA_NORM_CASE
  return SA_ERR_UNSUPPORTED;
}

int threads_of(int width) { return width <= 512 ? 32 : width <= 2048 ? 128 : width <= 4096 ? 256 : width <= 8192 ? 512 : 1024; }
// CTAs of the backward: about 1,024 threads an SM.
int blocks_of(const sa_norm& p) {
  const int t = threads_of(p.width), block = std::max(t, 128), rows = block / t;
  return (int)std::min<int64_t>((p.rows + rows - 1) / rows, (int64_t)kSms * (1024 / block));
}
int columns_of(const sa_norm& p) { return p.width * (p.dbias != nullptr ? 2 : 1); }

}  // namespace

size_t backward_bytes(const sa_norm& p) {
  return p.dweight == nullptr && p.dbias == nullptr ? 0 : (size_t)blocks_of(p) * columns_of(p) * sizeof(float);
}

int forward(const sa_norm& p, cudaStream_t s) {
  return by_width(p.width, [&](auto threads, auto chunks) {
    constexpr int T = decltype(threads)::value, NV = decltype(chunks)::value;
    const dim3 grid((unsigned)((p.rows + kRowsOf<T> - 1) / kRowsOf<T>));
    return vectors(p, false) ? launch_after(forward_kernel<T, NV, true>, grid, kBlock<T>, 0, s, p)
                             : launch_after(forward_kernel<T, NV, false>, grid, kBlock<T>, 0, s, p);
  });
}

int backward(const sa_norm& p, cudaStream_t s) {
  const int blocks = blocks_of(p);
  float* sums = p.dweight == nullptr && p.dbias == nullptr ? nullptr : static_cast<float*>(p.workspace);
  int st = by_width(p.width, [&](auto threads, auto chunks) {
    constexpr int T = decltype(threads)::value, NV = decltype(chunks)::value;
    const dim3 grid(blocks);
    if (p.dbias != nullptr)
      return vectors(p, true) ? launch_after(backward_kernel<T, NV, true, true>, grid, kBlock<T>, 0, s, p, sums)
                              : launch_after(backward_kernel<T, NV, false, true>, grid, kBlock<T>, 0, s, p, sums);
    return vectors(p, true) ? launch_after(backward_kernel<T, NV, true, false>, grid, kBlock<T>, 0, s, p, sums)
                            : launch_after(backward_kernel<T, NV, false, false>, grid, kBlock<T>, 0, s, p, sums);
  });
  if (st != SA_OK || sums == nullptr) return st;
  return launch_after(parameters_kernel, dim3((columns_of(p) + 31) / 32), 512, 0, s, (const float*)sums, blocks, p.width, columns_of(p), p.weight_dtype,
                      p.dweight, p.dbias);
}

}  // namespace norm
}  // namespace sa
