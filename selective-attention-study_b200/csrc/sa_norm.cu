// Layer norm, after a residual sum or alone, and its gradient.  s = x + branch, h = (s - mean) / sqrt(var + eps), y = h w + b;
//   ds = r (g - mean(g) - h mean(g h)) + ds_out,  g = dy w;   dw = sum over rows of dy h,   db = sum over rows of dy.
//
// Both directions are bound by memory: a row stays in the registers of a warp or a part of one (up to 512 values) or of one CTA between
// its only load and its only store; mean and variance are two sums over the registers, the second about the mean.  The backward's CTAs
// walk over rows and keep their columns' sums for dw and db, in registers up to 8,192 columns; a second kernel joins the CTAs' sums in
// their order.
#include "sa_layers.cuh"

#include <algorithm>

namespace sa {
namespace norm {
namespace {

// Sums of N values over the T threads of a row: part of a warp, a warp, or the CTA.  `buffer` is one of two that rows take in turn, so
// one barrier a sum is enough.
template <int T, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float2 (*buffer)[32], int& turn) {
#pragma unroll
  for (int o = T < 32 ? T / 2 : 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(~0u, v[k], o);
  if constexpr (T > 32) {
    float2* b = buffer[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = make_float2(v[0], N > 1 ? v[N - 1] : 0.f);
    __syncthreads();
    float2 all = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
      all.x += b[i].x;
      all.y += b[i].y;
    }
    v[0] = all.x;
    if (N > 1) v[N - 1] = all.y;
  }
}

template <int T> constexpr int kBlock = T < 128 ? 128 : T;
template <int T> constexpr int kRowsOf = kBlock<T> / T;

// Rows of which a team has the loads in flight together: narrow ones are too short to keep memory busy by themselves.
template <int T, int NV> constexpr int kTogether = T <= 32 && NV == 1 ? 2 : 1;

template <int T, int NV, bool VEC>
__global__ void __launch_bounds__(kBlock<T>, T == 512 ? 2 : 1) forward_kernel(const sa_norm p) {
  tc::after_previous_kernel();
  constexpr int R = kTogether<T, NV>;
  __shared__ float2 buffer[2][32];
  const int t = threadIdx.x % T;
  int turn = 0;
  float s[R][NV][8];
  int64_t row[R];
  int width[R];                                                  // threads of a warp that have no row go through the sums with the others
#pragma unroll
  for (int q = 0; q < R; ++q) {
    row[q] = ((int64_t)blockIdx.x * R + q) * kRowsOf<T> + threadIdx.x / T;
    width[q] = row[q] < p.rows ? p.width : 0;
    load_row<NV, T, VEC>(s[q], p.x, p.x_dtype, row[q] * p.x_stride, width[q], t);
  }
  if (p.branch != nullptr) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      float b[NV][8];
      load_row<NV, T, VEC>(b, p.branch, p.branch_dtype, row[q] * p.branch_stride, width[q], t);
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[q][c][i] = rounded_to(s[q][c][i] + b[c][i], p.x_dtype);
      store_row<NV, T, VEC>(s[q], p.sum, p.x_dtype, row[q] * p.width, width[q], t);
    }
  }
  const float over = 1.f / (float)p.width;
#pragma unroll
  for (int q = 0; q < R; ++q) {
    float sum[1] = {0.f};
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (in_row<T, VEC>(c, i, t, width[q])) sum[0] += s[q][c][i];
    row_sum<T>(sum, buffer, turn);
    const float mean = sum[0] * over;
    sum[0] = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[q][c][i] -= mean;
        if (in_row<T, VEC>(c, i, t, width[q])) sum[0] += s[q][c][i] * s[q][c][i];
      }
    row_sum<T>(sum, buffer, turn);
    const float r = rsqrtf(sum[0] * over + p.eps);
    if (t == 0 && width[q] > 0 && p.stats != nullptr) {
      p.stats[2 * row[q]] = mean;
      p.stats[2 * row[q] + 1] = r;
    }
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[q][c][i] *= r;
  }
  if (p.weight != nullptr) {
    float w[NV][8];
    load_row<NV, T, VEC>(w, p.weight, p.weight_dtype, 0, p.width, t);
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[q][c][i] *= w[c][i];
  }
  if (p.bias != nullptr) {
    float b[NV][8];
    load_row<NV, T, VEC>(b, p.bias, p.weight_dtype, 0, p.width, t);
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[q][c][i] += b[c][i];
  }
#pragma unroll
  for (int q = 0; q < R; ++q) store_row<NV, T, VEC>(s[q], p.y, p.y_dtype, row[q] * p.width, width[q], t);
}

// ---- backward -------------------------------------------------------------------------------------------------------------------

// Rows of more than 8,192 values leave no registers for their columns' sums: those are in shared memory, a thread's apart by the threads
// (4,000 rows of 12,288 in bf16 with a bias: 340 us with the sums in registers, most of them spilled, 230 this way, where a thread still spills
// 380 to 640 bytes; rows of 4,096 and 8,192, which spill 80 to 150 bytes, gain nothing from it).
template <int T, int NV> constexpr bool kSumsShared = T * NV * 8 > 8192;

// A thread's part of the gradient: of rows, h and g = dy in and dx out, and its columns' sums for dw and db.
template <int T, int NV, bool VEC, bool BIAS>
struct Gradient {
  static constexpr bool kShared = kSumsShared<T, NV>;
  float dw[kShared ? 1 : NV][8], db[BIAS && !kShared ? NV : 1][8];
  float* const mine;                       // in shared memory: dw, then db
  __device__ __forceinline__ Gradient(uint8_t* smem, int t) : mine(reinterpret_cast<float*>(smem) + t) {
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) add(c, i, 0.f, 0.f, true);
  }
  __device__ __forceinline__ void add(int c, int i, float w, float b, bool first = false) {
    if constexpr (kShared) {
      float* const at = mine + (c * 8 + i) * T;
      *at = first ? w : *at + w;
      if (BIAS) at[NV * 8 * T] = first ? b : at[NV * 8 * T] + b;
    } else {
      dw[c][i] = first ? w : dw[c][i] + w;
      if (BIAS) db[c][i] = first ? b : db[c][i] + b;
    }
  }
  // `width` is 0 in threads that have no row but go through the sums with the others.
  __device__ __forceinline__ void row(const sa_norm& p, float (&h)[NV][8], float (&g)[NV][8], float2 stats, int width, int t, float2 (*buffer)[32],
                                      int& turn) {
    const float over = 1.f / (float)p.width;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool inside = in_row<T, VEC>(c, i, t, width);
        h[c][i] = inside ? (h[c][i] - stats.x) * stats.y : 0.f;
        g[c][i] = inside ? g[c][i] : 0.f;
        add(c, i, g[c][i] * h[c][i], g[c][i]);
      }
    if (p.weight != nullptr) {
      float w[NV][8];
      load_row<NV, T, VEC>(w, p.weight, p.weight_dtype, 0, p.width, t);
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (in_row<T, VEC>(c, i, t, p.width)) g[c][i] *= w[c][i];
    }
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m[0] += g[c][i];
        m[1] += g[c][i] * h[c][i];
      }
    row_sum<T>(m, buffer, turn);
    const float mean_g = m[0] * over, mean_gh = m[1] * over;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) g[c][i] = stats.y * (g[c][i] - mean_g - h[c][i] * mean_gh);
  }
  // The CTA's sums into its part, its teams in their order.
  __device__ __forceinline__ void finish(const sa_norm& p, float* sums, float* shared, int t, int team) {
    if constexpr (kRowsOf<T> > 1) {
      constexpr int kTeam = T * NV * 8 * (BIAS ? 2 : 1);
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (team > 0) {
            shared[(team - 1) * kTeam + (c * 8 + i) * T + t] = dw[c][i];
            if (BIAS) shared[(team - 1) * kTeam + ((NV + c) * 8 + i) * T + t] = db[c][i];
          }
      __syncthreads();
      if (team > 0) return;
      for (int k = 0; k < kRowsOf<T> - 1; ++k)
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dw[c][i] += shared[k * kTeam + (c * 8 + i) * T + t];
            if (BIAS) db[c][i] += shared[k * kTeam + ((NV + c) * 8 + i) * T + t];
          }
    }
    float* out = sums + (int64_t)blockIdx.x * (BIAS ? 2 : 1) * p.width;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int col = column_of<T, VEC>(c, i, t);
        if (col >= p.width) continue;
        out[col] = kShared ? mine[(c * 8 + i) * T] : dw[kShared ? 0 : c][i];
        if (BIAS) out[p.width + col] = kShared ? mine[(NV * 8 + c * 8 + i) * T] : db[kShared ? 0 : c][i];
      }
  }
};
template <int T, int NV, bool BIAS>
constexpr size_t kTeamBytes = (kSumsShared<T, NV> ? 1 : kRowsOf<T> - 1) * (size_t)T * NV * 8 * (BIAS ? 2 : 1) * 4;

// Rows as they lie, by plain loads: strides and addresses that the copies below do not take, or rows too long for them.
// `sums`: (CTAs, 1 or 2, width), the parts of dw and db; null when neither is asked for.
template <int T, int NV, bool VEC, bool BIAS>
__global__ void __launch_bounds__(kBlock<T>) backward_kernel(const sa_norm p, float* sums) {
  tc::after_previous_kernel();
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 buffer[2][32];
  const int t = threadIdx.x % T, team = threadIdx.x / T;
  int turn = 0;
  Gradient<T, NV, VEC, BIAS> gradient(smem, t);
  const int64_t rounds = (p.rows + kRowsOf<T> - 1) / kRowsOf<T>;
  for (int64_t i0 = blockIdx.x; i0 < rounds; i0 += gridDim.x) {
    const int64_t row = i0 * kRowsOf<T> + team;
    const int width = row < p.rows ? p.width : 0;
    float h[NV][8], g[NV][8];
    load_row<NV, T, VEC>(h, p.x, p.x_dtype, row * p.x_stride, width, t);
    load_row<NV, T, VEC>(g, p.dy, p.y_dtype, row * p.dy_stride, width, t);
    const float2 stats = width > 0 ? make_float2(p.stats[2 * row], p.stats[2 * row + 1]) : make_float2(0.f, 0.f);
    gradient.row(p, h, g, stats, width, t, buffer, turn);
    if (p.dsum != nullptr) {
      load_row<NV, T, VEC>(h, p.dsum, p.x_dtype, row * p.dsum_stride, width, t);
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) g[c][i] += h[c][i];
    }
    store_row<NV, T, VEC>(g, p.dx, p.x_dtype, row * p.width, width, t);
    if (p.dbranch != nullptr) store_row<NV, T, VEC>(g, p.dbranch, p.branch_dtype, row * p.width, width, t);
  }
  if (sums != nullptr) gradient.finish(p, sums, reinterpret_cast<float*>(smem), t, team);
}

// Rows copied ahead into shared memory by bulk copies: what is in flight takes no registers, so the few CTAs that a thread's 60
// to 100 registers allow keep memory busy.  A stage has `rows` rows of x, dy and dsum with their statistics; contiguous rows of any
// width come in one copy a tensor (a multiple of 8 rows begins on 16 bytes), others row by row.
constexpr int kRing = 3;
struct Copies {
  int rows;                                // of a stage, even and a multiple of the rows that a CTA works on at a time
  int bytes[3];                            // of a row of x, dy, dsum (0: none)
  int at[4];                               // of x, dy, dsum and the statistics in a stage
  int stage;                               // bytes
  int64_t stride[3];                       // of rows, in bytes
  bool together[3];                        // contiguous
};
template <int T, int NV> constexpr int kResident = NV == 1 && T <= 32 ? 6 : 1;    // 85 registers a thread
template <int T, int NV, bool VEC, bool BIAS>
__global__ void __launch_bounds__(kBlock<T>, kResident<T, NV>) backward_copied_kernel(const sa_norm p, float* sums, const Copies c, const tc::WaitCtx status) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 buffer[2][32];
  __shared__ uint64_t full[kRing];
  const int t = threadIdx.x % T, team = threadIdx.x / T;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) tc::mbar_init(&full[i], 1);
    tc::mbar_init_fence();
  }
  __syncthreads();
  tc::after_previous_kernel();
  tc::Waiter wait;
  wait.begin(status);
  const int64_t stages = (p.rows + c.rows - 1) / c.rows;
  const char* const from[3] = {static_cast<const char*>(p.x), static_cast<const char*>(p.dy), static_cast<const char*>(p.dsum)};
  auto load = [&](int64_t i, int slot) {                          // by one thread
    const int64_t row = i * c.rows;
    const int n = (int)min((int64_t)c.rows, p.rows - row);
    uint8_t* to = smem + slot * c.stage;
    const uint32_t stats = (uint32_t)(n * 8) & ~15u;
    uint32_t all = stats;
#pragma unroll
    for (int k = 0; k < 3; ++k) all += (uint32_t)(n * c.bytes[k]) & ~15u;
    tc::mbar_expect_tx(&full[slot], all);
    if (stats > 0) tc::bulk_load(to + c.at[3], p.stats + 2 * row, stats, &full[slot]);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      if (c.bytes[k] == 0) continue;
      const char* src = from[k] + row * c.stride[k];
      if (c.together[k]) {
        const uint32_t size = (uint32_t)(n * c.bytes[k]) & ~15u;
        if (size > 0) tc::bulk_load(to + c.at[k], src, size, &full[slot]);
      } else {
        for (int r = 0; r < n; ++r) tc::bulk_load(to + c.at[k] + r * c.bytes[k], src + r * c.stride[k], (uint32_t)c.bytes[k], &full[slot]);
      }
    }
  };
  if (threadIdx.x == 0)
    for (int k = 0; k < kRing; ++k)
      if (blockIdx.x + (int64_t)k * gridDim.x < stages) load(blockIdx.x + (int64_t)k * gridDim.x, k);
  int turn = 0, slot = 0, round = 0;
  Gradient<T, NV, VEC, BIAS> gradient(smem, t);
  for (int64_t i = blockIdx.x; i < stages; i += gridDim.x) {
    const int64_t row0 = i * c.rows;
    const int n = (int)min((int64_t)c.rows, p.rows - row0);
    uint8_t* const at = smem + slot * c.stage;
    wait(tc::smem_u32(&full[slot]), round & 1, 1100);
    if (n < c.rows) {                                             // the last stage: what is left of 16 bytes
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const int done = (n * c.bytes[k]) & ~15, rest = n * c.bytes[k] - done;
        if ((int)threadIdx.x < rest / 2)
          reinterpret_cast<uint16_t*>(at + c.at[k] + done)[threadIdx.x] =
              reinterpret_cast<const uint16_t*>(from[k] + row0 * c.stride[k] + done)[threadIdx.x];
      }
      if (threadIdx.x < 2 && n % 2 != 0) reinterpret_cast<float*>(at + c.at[3])[2 * (n - 1) + threadIdx.x] = p.stats[2 * (row0 + n - 1) + threadIdx.x];
      __syncthreads();
    }
    auto rows = [&](int r0) {
      const int r = r0 + team;
      const int width = r < n ? p.width : 0;
      float h[NV][8], g[NV][8];
      load_row<NV, T, VEC, true>(h, at + c.at[0] + r * c.bytes[0], p.x_dtype, 0, width, t);
      load_row<NV, T, VEC, true>(g, at + c.at[1] + r * c.bytes[1], p.y_dtype, 0, width, t);
      const float2 stats = reinterpret_cast<const float2*>(at + c.at[3])[r];
      gradient.row(p, h, g, stats, width, t, buffer, turn);
      if (c.bytes[2] != 0) {
        load_row<NV, T, VEC, true>(h, at + c.at[2] + r * c.bytes[2], p.x_dtype, 0, width, t);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) g[k][e] += h[k][e];
      }
      store_row<NV, T, VEC>(g, p.dx, p.x_dtype, (row0 + r) * p.width, width, t);
      if (p.dbranch != nullptr) store_row<NV, T, VEC>(g, p.dbranch, p.branch_dtype, (row0 + r) * p.width, width, t);
    };
    if constexpr (T <= 32) {                                      // several rows in a turn of the loop would take too many registers
#pragma unroll 1
      for (int r0 = 0; r0 < n; r0 += kRowsOf<T>) rows(r0);
    } else {
      for (int r0 = 0; r0 < n; r0 += kRowsOf<T>) rows(r0);
    }
    __syncthreads();                                              // the stage has been read
    if (threadIdx.x == 0 && i + (int64_t)kRing * gridDim.x < stages) load(i + (int64_t)kRing * gridDim.x, slot);
    if (++slot == kRing) {
      slot = 0;
      ++round;
    }
  }
  wait.end(status);
  if (sums != nullptr) gradient.finish(p, sums, reinterpret_cast<float*>(smem), t, team);
}

// Columns of the parameters' gradients: 8 a CTA (a sector of each part), whose 64 groups of 8 threads take the parts in turn.
__global__ void __launch_bounds__(512) parameters_kernel(const float* sums, int parts, int width, int columns, int dtype, void* dweight, void* dbias) {
  tc::after_previous_kernel();
  __shared__ float by_group[64][9];
  const int c = threadIdx.x & 7, group = threadIdx.x >> 3, col = blockIdx.x * 8 + c;
  float v = 0.f;
  if (col < columns) {
#pragma unroll 8
    for (int i = group; i < parts; i += 64) v += sums[(int64_t)i * columns + col];
  }
  by_group[group][c] = v;
  __syncthreads();
  if (group >= 8) return;
  for (int i = group + 8; i < 64; i += 8) v += by_group[i][c];
  __syncwarp();
  by_group[group][c] = v;
  asm volatile("bar.sync 1, 64;" ::: "memory");
  if (group != 0 || col >= columns) return;
  for (int i = 1; i < 8; ++i) v += by_group[i][c];
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

// Threads and values of a row by its width: f(threads, chunks of 8 a thread).  Of narrow rows, as few threads as hold them: with eight,
// 5,333,333 rows of 3 bf16 values took 335 us forward and 936 with the gradients, with one 41 and 139; 500,000 of 32 25 and 80, with four
// 14 and 76.
template <bool FORWARD, typename F>
int by_width(int width, F f) {
  using std::integral_constant;
#define SA_NORM_CASE(most, threads, chunks) \
  if (width <= most) return f(integral_constant<int, threads>(), integral_constant<int, chunks>())
  SA_NORM_CASE(8, 1, 1);
  SA_NORM_CASE(16, 2, 1);
  SA_NORM_CASE(32, 4, 1);
  SA_NORM_CASE(64, 8, 1);
  SA_NORM_CASE(128, 16, 1);
  SA_NORM_CASE(256, 32, 1);
  SA_NORM_CASE(512, 32, 2);
  SA_NORM_CASE(1024, 128, 1);
  // wide ones: the forward has many CTAs an SM of few threads, each with 32 values (8,000 rows of 8,192 in bf16: 61 us, with 1,024
  // threads of 8 values 119; 8,000 of 2,048: 14 and 19); the backward's sums of columns leave room for 8 values
  if constexpr (FORWARD) {
    SA_NORM_CASE(2048, 128, 2);
    SA_NORM_CASE(4096, 128, 4);
    SA_NORM_CASE(8192, 256, 4);
  } else {
    SA_NORM_CASE(2048, 256, 1);
    SA_NORM_CASE(4096, 512, 1);
    SA_NORM_CASE(8192, 1024, 1);
  }
  SA_NORM_CASE(16384, 512, 4);
#undef SA_NORM_CASE
  return SA_ERR_UNSUPPORTED;
}

// What the backward's copies look like; false where rows do not take them.
bool copies_of(const sa_norm& p, int threads, int rows_at_a_time, Copies* c) {
  const void* const from[3] = {p.x, p.dy, p.dsum};
  const int types[3] = {p.x_dtype, p.y_dtype, p.x_dtype};
  const int64_t strides[3] = {p.x_stride, p.dy_stride, p.dsum_stride};
  bool odd = false;                        // rows that are no multiple of 16 bytes
  int row = 8;
  for (int k = 0; k < 3; ++k) {
    const int size = types[k] == SA_F32 ? 4 : 2;
    c->bytes[k] = from[k] != nullptr ? p.width * size : 0;
    c->stride[k] = strides[k] * size;
    c->together[k] = p.rows == 1 || strides[k] == p.width;
    if (from[k] == nullptr) continue;
    if (reinterpret_cast<uintptr_t>(from[k]) % 16 != 0) return false;
    if (!c->together[k] && (c->bytes[k] % 16 != 0 || c->stride[k] % 16 != 0)) return false;
    odd = odd || c->bytes[k] % 16 != 0;
    row += c->bytes[k];
  }
  if (reinterpret_cast<uintptr_t>(p.stats) % 16 != 0) return false;
  // stages of about 8 KB, of whole rounds of the CTA's teams
  const int step = std::max(rows_at_a_time, odd ? 8 : 2);
  c->rows = std::max(step, 8192 / row / step * step);
  int at = 0;
  for (int k = 0; k < 3; ++k) {
    c->at[k] = at;
    at += (c->rows * c->bytes[k] + 15) / 16 * 16;
  }
  c->at[3] = at;
  c->stage = (at + c->rows * 8 + 127) / 128 * 128;
  return c->stage * kRing <= (threads < 1024 ? 104 : 212) * 1024;        // two CTAs an SM, or the one that has all registers
}

// CTAs of the backward: at most 768 threads an SM, one CTA at least (of 1,024 threads for rows of 4,097 to 8,192 values), or as many as
// their stages leave room for.
int blocks_of(const sa_norm& p) {
  int blocks = 0;
  by_width<false>(p.width, [&](auto threads, auto chunks) {
    constexpr int T = decltype(threads)::value;
    Copies c;
    const bool copied = copies_of(p, kBlock<T>, kRowsOf<T>, &c);
    const int64_t rows = copied ? c.rows : kRowsOf<T>;
    const int here = copied ? std::min(768 / kBlock<T>, 200 * 1024 / (c.stage * kRing + 2048)) : 512 / kBlock<T>;
    blocks = (int)std::min<int64_t>((p.rows + rows - 1) / rows, (int64_t)kSms * std::max(1, here));
    return SA_OK;
  });
  return blocks;
}
int columns_of(const sa_norm& p) { return p.width * (p.dbias != nullptr ? 2 : 1); }

template <int T, int NV, bool VEC, bool BIAS>
int launch_backward(const sa_norm& p, int blocks, float* sums, cudaStream_t s) {
  if constexpr (!kSumsShared<T, NV>) {     // whose stages would be too large
    Copies c;
    if (copies_of(p, kBlock<T>, kRowsOf<T>, &c)) {
      tc::WaitCtx status;
      const int st = tc::wait_ctx(&status);
      if (st != SA_OK) return st;
      const size_t smem = std::max((size_t)c.stage * kRing, kTeamBytes<T, NV, BIAS>);
      return launch_after(backward_copied_kernel<T, NV, VEC, BIAS>, dim3(blocks), kBlock<T>, smem, s, p, sums, (const Copies)c,
                          (const tc::WaitCtx)status);
    }
  }
  return launch_after(backward_kernel<T, NV, VEC, BIAS>, dim3(blocks), kBlock<T>, kTeamBytes<T, NV, BIAS>, s, p, sums);
}

}  // namespace

size_t backward_bytes(const sa_norm& p) {
  return p.dweight == nullptr && p.dbias == nullptr ? 0 : (size_t)blocks_of(p) * columns_of(p) * sizeof(float);
}

int forward(const sa_norm& p, cudaStream_t s) {
  return by_width<true>(p.width, [&](auto threads, auto chunks) {
    constexpr int T = decltype(threads)::value, NV = decltype(chunks)::value;
    constexpr int kRows = kRowsOf<T> * kTogether<T, NV>;
    const dim3 grid((unsigned)((p.rows + kRows - 1) / kRows));
    return vectors(p, false) ? launch_after(forward_kernel<T, NV, true>, grid, kBlock<T>, 0, s, p)
                             : launch_after(forward_kernel<T, NV, false>, grid, kBlock<T>, 0, s, p);
  });
}

int backward(const sa_norm& p, cudaStream_t s) {
  const int blocks = blocks_of(p);
  float* sums = p.dweight == nullptr && p.dbias == nullptr ? nullptr : static_cast<float*>(p.workspace);
  const int st = by_width<false>(p.width, [&](auto threads, auto chunks) {
    constexpr int T = decltype(threads)::value, NV = decltype(chunks)::value;
    const bool vec = vectors(p, true);
    if (p.dbias != nullptr) return vec ? launch_backward<T, NV, true, true>(p, blocks, sums, s) : launch_backward<T, NV, false, true>(p, blocks, sums, s);
    return vec ? launch_backward<T, NV, true, false>(p, blocks, sums, s) : launch_backward<T, NV, false, false>(p, blocks, sums, s);
  });
  if (st != SA_OK || sums == nullptr) return st;
  return launch_after(parameters_kernel, dim3((columns_of(p) + 7) / 8), 512, 0, s, (const float*)sums, blocks, p.width, columns_of(p), p.weight_dtype,
                      p.dweight, p.dbias);
}

}  // namespace norm
}  // namespace sa
