// The best continuations over beams and vocabulary (sm_100a).
//
//   score[k][v] = scores[k] + logits[k][v] - log sum_u exp(logits[k][u]);   the WIDTH largest over (k, v) of a group, in order,
//   equal ones by the lowest k V + v.
//
// Two launches.  candidates_kernel reads the logits once: a CTA keeps a chunk of one beam's vocabulary in registers, and leaves
// the chunk's maximum, its sum of exponentials and its WIDTH largest logits.  choose_kernel (a CTA a group) makes the beams'
// log-sum-exp of those and takes the best of all candidates, in 64 bits: two beams' scores can be as near to one another as
// the rounding of a 32-bit sum, and which one comes first is a whole number.
// Bound by memory where there are many beams, else by the latency of the two launches.
//
// The largest of a set, without sorting it: every thread's own maximum is ranked among those of the CTA; the WIDTH-th of them
// bounds the WIDTH-th of the set from below, and the few elements that reach it are ranked among themselves.  Where more than
// kList reach it (equal or masked logits) they are taken one by one.
#include "sa_common.cuh"
#include "sa_beam.cuh"
#include "sa_tc_ptx.cuh"

namespace sa {
namespace beam {
namespace {

constexpr int kThreads = 256;
constexpr int kList = 256;

template <typename V>
struct Entry {
  V value;
  long long index;           // below 0: none
};
// a comes before b
template <typename V>
__device__ __forceinline__ bool before(const V a, const long long ia, const V b, const long long ib) {
  return a > b || (a == b && ia < ib);
}

template <typename V>
struct Shared {
  V top[kThreads];
  Entry<V> list[kList];
  V threshold;
  int count;
  Entry<V> warp_best[kThreads / 32];
};

// Calls emit(rank, value, index) for the `width` first of the CTA's elements.  each(f) calls f(value, index) for every element
// of the calling thread (no value a NaN); the same ones each time.  All threads call this; emit is called by any.
template <typename V, typename Each, typename Emit>
__device__ __forceinline__ void largest(Shared<V>& sh, int width, const Each& each, const Emit& emit) {
  const int tid = threadIdx.x;
  constexpr V kNone = -INFINITY;
  V mine = kNone;
  bool any = false;
  each([&](V x, long long) {
    mine = any ? (x > mine ? x : mine) : x;
    any = true;
  });
  sh.top[tid] = mine;                                       // a thread without elements: -inf bounds as well
  if (tid == 0) sh.count = 0;
  __syncthreads();
  int rank = 0;
  for (int u = 0; u < kThreads; ++u) rank += before(sh.top[u], (long long)u, mine, (long long)tid) ? 1 : 0;
  if (rank == width - 1) sh.threshold = mine;
  __syncthreads();
  const V bound = sh.threshold;
  each([&](V x, long long i) {
    if (x >= bound) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = Entry<V>{x, i};
    }
  });
  __syncthreads();
  const int n = sh.count;
  if (n <= kList) {
    if (tid < n) {
      const Entry<V> e = sh.list[tid];
      int at = 0;
      for (int u = 0; u < n; ++u) at += before(sh.list[u].value, sh.list[u].index, e.value, e.index) ? 1 : 0;
      if (at < width) emit(at, e.value, e.index);
    }
    for (int u = n + tid; u < width; u += kThreads) emit(u, kNone, -1LL);     // fewer elements than that
    return;
  }
  Entry<V> last{INFINITY, -1};                               // one by one
  for (int w = 0; w < width; ++w) {
    Entry<V> best{kNone, -1};
    each([&](V x, long long i) {
      const bool left = w == 0 || before(last.value, last.index, x, i);
      if (left && (best.index < 0 || before(x, i, best.value, best.index))) best = Entry<V>{x, i};
    });
    auto better = [&](const Entry<V>& o) {
      if (o.index >= 0 && (best.index < 0 || before(o.value, o.index, best.value, best.index))) best = o;
    };
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      Entry<V> o;
      o.value = __shfl_xor_sync(0xffffffffu, best.value, s);
      o.index = __shfl_xor_sync(0xffffffffu, best.index, s);
      better(o);
    }
    if ((tid & 31) == 0) sh.warp_best[tid >> 5] = best;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kThreads / 32; ++u) better(sh.warp_best[u]);
    __syncthreads();
    last = best;
    if (tid == 0) emit(w, best.value, best.index);
  }
}

// Elements are taken in units of 16 bytes from a 16-byte boundary on: a row that begins elsewhere has `lead` elements fewer in
// its first unit.  Ends of a row are read element by element.
template <typename T, int UNITS>
__global__ void __launch_bounds__(kThreads) candidates_kernel(const T* __restrict__ logits, int64_t group_stride, int64_t beam_stride,
                                                              int beams, int vocab, int width, int chunks, float2* __restrict__ sums,
                                                              float* __restrict__ values, int* __restrict__ tokens) {
  constexpr int kPer = 16 / (int)sizeof(T);
  __shared__ Shared<float> sh;
  __shared__ float red[2][kThreads / 32];
  const int n = blockIdx.x / chunks, chunk = blockIdx.x - n * chunks;      // n: beam over all groups
  const int g = n / beams;
  const T* row = logits + g * group_stride + (int64_t)(n - g * beams) * beam_stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int tid = threadIdx.x;
  float x[UNITS * kPer];
  int first[UNITS];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int64_t v64 = ((int64_t)chunk * UNITS + u) * kThreads * kPer + (int64_t)tid * kPer - lead;
    const int v = (int)min(v64, (int64_t)vocab);
    first[u] = v;
    if (v >= 0 && v64 + kPer <= vocab) {
      const uint4 raw = *reinterpret_cast<const uint4*>(row + v);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[u * kPer + i] = to_float<T>(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[u * kPer + i] = v + i >= 0 && v64 + i < vocab ? to_float<T>(row[v + i]) : -INFINITY;
    }
  }
  // the chunk's maximum (NaNs aside) and its sum of exponentials (with them)
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < UNITS * kPer; ++i) top = fmaxf(top, x[i]);
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  if ((tid & 31) == 0) red[0][tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kThreads / 32; ++u) top = fmaxf(top, red[0][u]);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < UNITS * kPer; ++i) {
    sum += x[i] == -INFINITY ? 0.f : exp2f((x[i] - top) * kLog2e);         // +inf: inf - inf, the beam has no finite sum
    if (isnan(x[i])) x[i] = -INFINITY;
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
  if ((tid & 31) == 0) red[1][tid >> 5] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int u = 1; u < kThreads / 32; ++u) sum += red[1][u];
    sums[blockIdx.x] = make_float2(top, sum);
  }
  auto each = [&](auto f) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (first[u] + i >= 0 && first[u] + i < vocab) f(x[u * kPer + i], (long long)(first[u] + i));
  };
  float* out_v = values + (int64_t)blockIdx.x * width;
  int* out_t = tokens + (int64_t)blockIdx.x * width;
  largest(sh, width, each, [&](int at, float v, long long i) {
    out_v[at] = v;
    out_t[at] = (int)i;
  });
}

__global__ void __launch_bounds__(kThreads) choose_kernel(const float* __restrict__ scores, int beams, int vocab, int width, int chunks,
                                                          const float2* __restrict__ sums, const float* __restrict__ values,
                                                          const int* __restrict__ tokens, float* __restrict__ out_scores,
                                                          int* __restrict__ out_rows, long long* __restrict__ out_tokens) {
  tc::after_previous_kernel();
  __shared__ Shared<double> sh;
  __shared__ double base[kMaxBeams];                         // score - log-sum-exp of a beam; NaN: all of its scores are -inf
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  for (int k = tid >> 5; k < beams; k += kThreads / 32) {
    const float2* part = sums + ((int64_t)g * beams + k) * chunks;
    float top = -INFINITY;
    for (int c = lane; c < chunks; c += 32) top = fmaxf(top, part[c].x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    double sum = 0.0;
    for (int c = lane; c < chunks; c += 32) {
      const float2 p = part[c];
      if (p.y != 0.f) sum += (double)p.y * exp((double)p.x - (double)top);      // 0: nothing but -inf; a NaN stays
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (lane == 0) {
      const double b = (double)scores[(int64_t)g * beams + k] - ((double)top + log(sum));
      base[k] = isfinite(b) ? b : nan("");
    }
  }
  __syncthreads();
  const int per_beam = chunks * width;
  const int64_t first = (int64_t)g * beams * per_beam;
  auto each = [&](auto f) {
    for (int i = tid; i < beams * per_beam; i += kThreads) {
      const int k = i / per_beam;
      if (isnan(base[k])) {                                   // equal ones: the lowest tokens stand for all
        const int v = i - k * per_beam;
        if (v < width && v < vocab) f(-(double)INFINITY, (long long)k * vocab + v);
        continue;
      }
      const int v = tokens[first + i];
      if (v >= 0) f(base[k] + (double)values[first + i], (long long)k * vocab + v);
    }
  };
  largest(sh, width, each, [&](int at, double v, long long i) {
    const int64_t o = (int64_t)g * width + at;
    const int k = (int)(i / vocab);
    out_scores[o] = (float)v;
    out_rows[o] = g * beams + k;
    out_tokens[o] = i - (long long)k * vocab;
  });
}

template <typename T>
int units_of(int rows, int vocab) {
  // 8,192 logits a CTA where that still gives every SM several, else 2,048 (of 32 bits half as many)
  constexpr int kPer = 16 / (int)sizeof(T);
  const int64_t large = (int64_t)rows * ((vocab + 4 * kThreads * kPer - 1) / (4 * kThreads * kPer));
  return large >= 4 * kSms ? 4 : 1;
}
int units_for(int dtype, int rows, int vocab) {
  return dtype == SA_F32 ? units_of<float>(rows, vocab) : units_of<__half>(rows, vocab);
}
int chunks_for(int dtype, int rows, int vocab) {
  const int per = dtype == SA_F32 ? 4 : 8, chunk = units_for(dtype, rows, vocab) * kThreads * per;
  return (int)(((int64_t)vocab + per - 1 + chunk - 1) / chunk);             // a row may begin up to per - 1 elements into a unit
}

}  // namespace

size_t workspace_bytes(int dtype, int groups, int beams, int vocab, int width) {
  return (size_t)groups * beams * chunks_for(dtype, groups * beams, vocab) * (8 + 8 * (size_t)width);
}

int select(const Select& p, cudaStream_t s) {
  const int rows = p.groups * p.beams, chunks = chunks_for(p.dtype, rows, p.vocab);
  float2* sums = static_cast<float2*>(p.workspace);
  float* values = reinterpret_cast<float*>(sums + (size_t)rows * chunks);
  int* tokens = reinterpret_cast<int*>(values + (size_t)rows * chunks * p.width);
  auto launch = [&](auto kernel, auto ptr) {
    count_launch();
    kernel<<<(unsigned)rows * chunks, kThreads, 0, s>>>(ptr, p.group_stride, p.beam_stride, p.beams, p.vocab, p.width, chunks, sums, values,
                                                        tokens);
  };
  const bool four = units_for(p.dtype, rows, p.vocab) == 4;
  switch (p.dtype) {
    case SA_F32: {
      const float* x = static_cast<const float*>(p.logits);
      four ? launch(candidates_kernel<float, 4>, x) : launch(candidates_kernel<float, 1>, x);
      break;
    }
    case SA_BF16: {
      const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.logits);
      four ? launch(candidates_kernel<__nv_bfloat16, 4>, x) : launch(candidates_kernel<__nv_bfloat16, 1>, x);
      break;
    }
    case SA_F16: {
      const __half* x = static_cast<const __half*>(p.logits);
      four ? launch(candidates_kernel<__half, 4>, x) : launch(candidates_kernel<__half, 1>, x);
      break;
    }
    default: return SA_ERR_BAD_ARGUMENT;
  }
  SA_CUDA_CHECK(cudaGetLastError());
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(p.groups);
  config.blockDim = dim3(kThreads);
  config.stream = s;
  config.attrs = &attr;
  config.numAttrs = 1;
  count_launch();
  SA_CUDA_CHECK(cudaLaunchKernelEx(&config, choose_kernel, p.scores, p.beams, p.vocab, p.width, chunks, (const float2*)sums,
                                   (const float*)values, (const int*)tokens, p.out_scores, p.out_rows, p.out_tokens));
  return SA_OK;
}

}  // namespace beam
}  // namespace sa
