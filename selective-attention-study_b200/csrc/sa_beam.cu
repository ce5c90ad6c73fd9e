// The best continuations over beams and vocabulary (sm_100a).
//
//   score[k][v] = scores[k] + logits[k][v] - log sum_u exp(logits[k][u]);   the WIDTH largest over (k, v) of a group, in order,
//   equal ones by the lowest k V + v.
//
// Two launches.  candidates_kernel: a CTA takes a run of one beam's vocabulary into shared memory and leaves the run's maximum, its
// sum of exponentials and its WIDTH largest logits.  choose_kernel (a CTA a group) makes the
// beams' log-sum-exp of those and takes the best of all candidates, in 64 bits: two beams' scores can be as near to one another as
// the rounding of a 32-bit sum, and which one comes first is a whole number.
// 256 beams of 50,304 bf16 logits (25.7 MB): 16.2 us both, each alone with cold caches 14.6 and 6.2.  Where the first goes, in cycles
// of a CTA that ends last: 1,500 until its loads are issued, 12,000 until its first part is there (behind the three other CTAs of its
// SM), 19,000 until it has looked at the run, 24,000 with the ranking.  From L2 the first part takes 4,600 and the rest as long, so the
// exponentials (8 cycles of a warp each) and the loads share the blame.  4 beams: 7.6 us both, alone 6 to 7 and 5 to 6: latency.
//
// The largest of a set, without sorting it: each warp that has elements gives the largest of its lanes' own maxima, about two times
// WIDTH of them in all.  WIDTH elements at least reach the WIDTH-th of those, and not many more do.  They are ranked among
// themselves.  Where more than kList reach it (one beam far above the others, most often), the WIDTH-th of the first kList of them is a
// better bound; where that does not help because many are equal to it (masked logits, most often), those above it are ranked and the
// first of the equal ones are found in order; where that is not so either, they are taken one by one.
#include <type_traits>

#include "sa_common.cuh"
#include "sa_beam.cuh"
#include "sa_tc_ptx.cuh"

namespace sa {
namespace beam {
namespace {

constexpr int kThreads = 256;
constexpr int kList = kThreads;
constexpr int kTops = 64;              // maxima that make the first bound: a lane of every warp ranks two
constexpr bool tops_are_enough(int warps) { return warps == 0 || (kTops / warps >= (kMaxWidth + warps - 1) / warps && tops_are_enough(warps - 1)); }
static_assert(tops_are_enough(kThreads / 32), "the maxima of any number of warps are as many as the widest selection");

template <typename V, typename I>
struct Entry {
  V value;
  I index;                   // below 0: none
};
// a comes before b
template <typename V, typename I>
__device__ __forceinline__ bool before(const Entry<V, I>& a, const Entry<V, I>& b) {
  return a.value > b.value || (a.value == b.value && a.index < b.index);
}

template <typename V, typename I>
struct Shared {
  V tops[kTops];
  V bound;
  Entry<V, I> list[kList];
  int count;
  Entry<V, I> warp_best[kThreads / 32];
};

__device__ __forceinline__ float warp_max(float x) {
  float top;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(x));
  return top;
}
// (no NaN) by the bits, as a whole number whose order is the values': its upper half, then the lower one of those that have that
__device__ __forceinline__ double warp_max(double x) {
  const long long bits = __double_as_longlong(x), key = bits ^ ((bits >> 63) & 0x7fffffffffffffffLL);
  const int high = (int)(key >> 32), top = __reduce_max_sync(0xffffffffu, high);
  const unsigned low = __reduce_max_sync(0xffffffffu, high == top ? (unsigned)key : 0u);
  const long long best = ((long long)top << 32) | low;
  return __longlong_as_double(best ^ ((best >> 63) & 0x7fffffffffffffffLL));
}

// Calls emit(rank, value, index) for the `width` first of the CTA's elements, which the first `warps` warps have.  `mine` is the
// largest value of the calling thread's (-inf: none).  reach(bound, above, f) calls f(value, index) for the CTA's elements that are
// not below `bound` (`above`: that are above it), until that says no, one(f) for the calling thread's (no value a NaN), of a list in
// order up to the first that f says yes to at least.
// equal(x, n, f) calls f(k, index) for the first n of the elements that are x, or returns false.  All threads call this; emit is
// called by any.
template <typename V, typename I, typename Reach, typename One, typename Equal, typename Emit>
__device__ __forceinline__ void largest(Shared<V, I>& sh, int width, int warps, V mine, const Reach& reach, const One& one, const Equal& equal,
                                        const Emit& emit) {
  const int tid = threadIdx.x, lane = tid & 31;
  constexpr V kNone = -INFINITY;
  // of w warps all but the last have 32 lanes' elements (or every lane of all has one): 2 ceil(width / w) of each are enough, and
  // so is what kTops has room for (where w does not divide the width twice as many would be up to 72)
  const int each = min(32, min(2 * ((width + warps - 1) / warps), kTops / warps)), given = each * warps;
  for (int u = 0; u < each && (tid >> 5) < warps; ++u) {
    const V top = warp_max(mine);
    const unsigned at = __ballot_sync(0xffffffffu, mine == top);
    if (lane == __ffs(at) - 1) mine = kNone;                // one of them is done with
    if (lane == 0) sh.tops[u * warps + (tid >> 5)] = top;
  }
  if (tid == 0) sh.count = 0;
  __syncthreads();
  V bound;                                                  // the `width`-th of them: every warp finds it for itself
  {
    const V own[2] = {lane < given ? sh.tops[lane] : kNone, lane + 32 < given ? sh.tops[lane + 32] : kNone};
    int rank[2] = {0, 0};
#pragma unroll 8
    for (int u = 0; u < given; ++u) {
      const V other = sh.tops[u];
      rank[0] += other > own[0] || (other == own[0] && u < lane) ? 1 : 0;
      if (given > 32) rank[1] += other > own[1] || (other == own[1] && u < lane + 32) ? 1 : 0;
    }
    const unsigned first = __ballot_sync(0xffffffffu, lane < given && rank[0] == width - 1);
    const unsigned second = __ballot_sync(0xffffffffu, lane + 32 < given && rank[1] == width - 1);
    bound = first != 0u ? __shfl_sync(0xffffffffu, own[0], __ffs(first) - 1) : __shfl_sync(0xffffffffu, own[1], __ffs(second) - 1);
  }
  reach(bound, false, [&](V x, I i) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kList) sh.list[at] = Entry<V, I>{x, i};
    return at <= kList;
  });
  __syncthreads();
  int n = sh.count;
  while (n > kList) {                                        // of those that are on the list the `width`-th is a better bound
    const V own = sh.list[tid].value;
    int rank = 0;
#pragma unroll 8
    for (int u = 0; u < kList; ++u) rank += sh.list[u].value > own || (sh.list[u].value == own && u < tid) ? 1 : 0;
    if (rank == width - 1) sh.bound = own;
    __syncthreads();
    const V better = sh.bound;
    if (!(better > bound)) break;
    bound = better;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    reach(bound, false, [&](V x, I i) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = Entry<V, I>{x, i};
      return at <= kList;
    });
    __syncthreads();
    n = sh.count;
  }
  int ties = 0;                                              // of the first `width`, those that are equal to the bound
  if (n > kList) {
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
    reach(bound, true, [&](V x, I i) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = Entry<V, I>{x, i};
      return at <= kList;
    });
    __syncthreads();
    n = sh.count;
    if (n < width) {
      ties = width - n;
      if (!equal(bound, ties, [&](int k, I i) { emit(n + k, bound, i); })) n = kList + 1;
    }
  }
  if (n <= kList) {
    if (tid < n) {
      const Entry<V, I> e = sh.list[tid];
      int at = 0;
#pragma unroll 4
      for (int u = 0; u < n; ++u) at += before(sh.list[u], e) ? 1 : 0;
      if (at < width) emit(at, e.value, e.index);
    }
    for (int u = n + ties + tid; u < width; u += kThreads) emit(u, kNone, (I)-1);     // fewer elements than that
    return;
  }
  Entry<V, I> last{INFINITY, -1};                            // one by one
  for (int w = 0; w < width; ++w) {
    Entry<V, I> best{kNone, -1};
    auto better = [&](const Entry<V, I>& o) {
      if (o.index >= 0 && (best.index < 0 || before(o, best))) best = o;
    };
    one([&](V x, I i) {
      const Entry<V, I> e{x, i};
      const bool left = w == 0 || before(last, e);
      if (left) better(e);
      return left;
    });
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      Entry<V, I> o;
      o.value = __shfl_xor_sync(0xffffffffu, best.value, s);
      o.index = __shfl_xor_sync(0xffffffffu, best.index, s);
      better(o);
    }
    if (lane == 0) sh.warp_best[tid >> 5] = best;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kThreads / 32; ++u) better(sh.warp_best[u]);
    __syncthreads();
    last = best;
    if (tid == 0) emit(w, best.value, best.index);
  }
}

// Two logits of a 32-bit word, or one.
template <typename T> struct Word;
template <> struct Word<float> {
  static constexpr int kPer = 1;
  static __device__ __forceinline__ float at(uint32_t w, int) { return __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t none() { return 0xff800000u; }
};
template <> struct Word<__nv_bfloat16> {
  static constexpr int kPer = 2;
  static __device__ __forceinline__ float at(uint32_t w, int e) { return __uint_as_float(e ? w & 0xffff0000u : w << 16); }
  static __device__ __forceinline__ uint32_t none() { return 0xff80u; }
};
template <> struct Word<__half> {
  static constexpr int kPer = 2;
  static __device__ __forceinline__ float at(uint32_t w, int e) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return e ? __high2float(h) : __low2float(h);
  }
  static __device__ __forceinline__ uint32_t none() { return 0xfc00u; }
};

// Elements are taken in units of 16 bytes from a 16-byte boundary on: a row that begins elsewhere has `lead` elements fewer in
// its first unit.  A unit that sticks out of the row is put together element by element; the others come by bulk copies in
// kParts parts, so that the first is worked on while the last is on its way (in 1, 2, 3, 4, 12: 14.0, 13.4, 12.7, 13.6, 16.3 us for 256
// beams of 50,304: every wait costs some 250 cycles).
constexpr int kParts = 3;
constexpr int kMostUnits = 3328;     // of a CTA: 52 KB, four CTAs an SM

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) candidates_kernel(const T* __restrict__ logits, int64_t group_stride, int64_t beam_stride,
                                                                 int beams, int vocab, int width, int chunks, int units,
                                                                 float2* __restrict__ sums, float* __restrict__ values,
                                                                 int* __restrict__ tokens, tc::WaitCtx status) {
  using W = Word<T>;
  constexpr int kPer = 16 / (int)sizeof(T);
  asm volatile("griddepcontrol.launch_dependents;");
  extern __shared__ __align__(128) uint4 run[];
  __shared__ uint64_t arrived[kParts];
  __shared__ Shared<float, int> sh;
  __shared__ float2 red[kThreads / 32];
  __shared__ int sums_s[kThreads / 32];
  const int n = blockIdx.x / chunks, chunk = blockIdx.x - n * chunks;      // n: beam over all groups
  const int g = n / beams;
  const T* row = logits + g * group_stride + (int64_t)(n - g * beams) * beam_stride;
  const int lead = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int tid = threadIdx.x;
  // this CTA's units: [unit0, unit0 + count) of the row's, of which [whole0, whole1) lie inside the row
  const int total = (int)(((int64_t)vocab + lead + kPer - 1) / kPer);
  const int unit0 = chunk * units, count = max(0, min(units, total - unit0));
  const int whole0 = unit0 == 0 && lead > 0 ? 1 : 0, whole1 = max(whole0, min(count, (int)(((int64_t)vocab + lead) / kPer) - unit0));
  const int part_units = (whole1 - whole0 + kParts - 1) / kParts;
  if (tid == 0) {
    for (int p = 0; p < kParts; ++p) tc::mbar_init(&arrived[p], 1);
    tc::mbar_init_fence();
    for (int p = 0; p < kParts; ++p) {
      const int u0 = whole0 + p * part_units, u1 = min(u0 + part_units, whole1);
      tc::mbar_expect_tx(&arrived[p], u1 > u0 ? (uint32_t)(u1 - u0) * 16u : 0u);
      if (u1 > u0) tc::bulk_load(run + u0, row + (int64_t)(unit0 + u0) * kPer - lead, (uint32_t)(u1 - u0) * 16u, &arrived[p]);
    }
  }
  for (int u = tid; u < whole0 + count - whole1; u += kThreads) {          // at most two
    const int at = u < whole0 ? u : whole1 + u - whole0;
    const int64_t v = (int64_t)(unit0 + at) * kPer - lead;
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = 0;
#pragma unroll
      for (int e = 0; e < W::kPer; ++e) {
        const int64_t j = v + i * W::kPer + e;
        uint32_t one = W::none();
        if (j >= 0 && j < vocab) {
          if constexpr (sizeof(T) == 4) one = __float_as_uint(row[j]);
          else one = *reinterpret_cast<const uint16_t*>(row + j);
        }
        x[i] |= one << (16 * e);
      }
    }
    run[at] = make_uint4(x[0], x[1], x[2], x[3]);
  }
  __syncthreads();
  // The run's maximum (NaNs aside) and its sum of exponentials (with them), by thread with a maximum of its own.
  // +inf: inf - inf, a NaN as a NaN among the logits: the beam has no finite sum.
  float mine = -INFINITY, sum = 0.f;
  auto take = [&](int u, auto n_units) {                       // n_units of them, kThreads apart
    constexpr int kUnits = decltype(n_units)::value;
    float x[kUnits][kPer], top = mine;
#pragma unroll
    for (int o = 0; o < kUnits; ++o) {
      const uint4 raw = run[u + o * kThreads];
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < kPer; ++i) x[o][i] = W::at(w[i / W::kPer], i % W::kPer);
    }
#pragma unroll
    for (int o = 0; o < kUnits; ++o)
#pragma unroll
      for (int i = 0; i < kPer; i += 2) top = fmaxf(top, fmaxf(x[o][i], x[o][i + 1]));
    const float from = top == -INFINITY ? 0.f : top;
    if (top > mine) sum *= tc::ex2((mine - from) * kLog2e);
    mine = top;
    const float2 shift = make_float2(-from, -from), scale = make_float2(kLog2e, kLog2e);
#pragma unroll
    for (int o = 0; o < kUnits; ++o) {
      float2 part = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kPer; i += 2) {
        const float2 d = __fmul2_rn(__fadd2_rn(make_float2(x[o][i], x[o][i + 1]), shift), scale);
        part = __fadd2_rn(part, make_float2(tc::ex2(d.x), tc::ex2(d.y)));
      }
      sum += part.x + part.y;
    }
  };
  int here = whole0, part = 0;                              // units below `here` have arrived
  auto arrive = [&](int u) {
    for (; u >= here && part < kParts; here = min(here + part_units, whole1)) tc::mbar_wait(&arrived[part++], 0, status, 700);
  };
  int u = tid;
  for (; u + kThreads < count; u += 2 * kThreads) {
    arrive(u + kThreads);
    take(u, std::integral_constant<int, 2>{});
  }
  if (u < count) {
    arrive(u);
    take(u, std::integral_constant<int, 1>{});
  }
  for (; part < kParts; ++part) tc::mbar_wait(&arrived[part], 0, status, 700);
  {
    const float top = warp_max(mine);
    if (top != -INFINITY) sum *= tc::ex2((mine - top) * kLog2e);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if ((tid & 31) == 0) red[tid >> 5] = make_float2(top, sum);
  }
  auto hits_of = [&](int u, auto wanted) {                     // which elements of a unit, a bit each (a NaN is never chosen)
    const uint4 raw = run[u];
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    const unsigned v = (unsigned)(unit0 + u) * kPer - lead;     // (of an element before the row: above every place)
    unsigned hits = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (wanted(fmaxf(W::at(w[i / W::kPer], i % W::kPer), -INFINITY)) && v + i < (unsigned)vocab) hits |= 1u << i;
    return hits;
  };
  // Few threads have anything to give: where they have many units, each one's are looked through by half of its warp.
  auto reach = [&](float bound, bool above, auto f) {
    bool more = true;
    auto take_unit = [&](int u) {
      for (unsigned hits = hits_of(u, [&](float x) { return above ? x > bound : x >= bound; }); hits != 0u && more; hits &= hits - 1u) {
        const int i = __ffs(hits) - 1;
        more = f(fmaxf(to_float<T>(reinterpret_cast<const T*>(run)[u * kPer + i]), -INFINITY), (int)((int64_t)(unit0 + u) * kPer - lead + i));
      }
    };
    const bool any = above ? mine > bound : mine >= bound;
    if (count <= 2 * kThreads) {
      for (int u = tid; u < count && any && more; u += kThreads) take_unit(u);
      return;
    }
    for (unsigned left = __ballot_sync(0xffffffffu, any); left != 0u;) {
      const unsigned rest = left & (left - 1u);
      const unsigned whose = (tid & 16) == 0 ? left : rest;
      if (whose != 0u)
        for (int u = (tid & ~31) + __ffs(whose) - 1 + (tid & 15) * kThreads; u < count && more; u += 16 * kThreads) take_unit(u);
      left = rest & (rest - 1u);
      __syncwarp();
    }
  };
  auto one = [&](auto f) {
    for (int u = tid; u < count; u += kThreads)
      for (unsigned hits = hits_of(u, [](float) { return true; }); hits != 0u; hits &= hits - 1u) {
        const int i = __ffs(hits) - 1;
        f(fmaxf(to_float<T>(reinterpret_cast<const T*>(run)[u * kPer + i]), -INFINITY), (int)((int64_t)(unit0 + u) * kPer - lead + i));
      }
  };
  auto equal = [&](float x, int need, auto f) {                // 256 units at a time, a prefix sum over the threads
    int found = 0;
    for (int base = 0; base < count && found < need; base += kThreads) {
      const int u = base + tid;
      const int64_t v = (int64_t)(unit0 + u) * kPer - lead;
      unsigned hits = u < count ? hits_of(u, [&](float y) { return y == x; }) : 0u;
      int upto = __popc(hits);
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, s);
        if ((tid & 31) >= s) upto += y;
      }
      if ((tid & 31) == 31) sums_s[tid >> 5] = upto;
      __syncthreads();
      int at = found + upto - __popc(hits);
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < (tid >> 5)) at += sums_s[w];
        found += sums_s[w];
      }
      for (; hits != 0u && at < need; hits &= hits - 1u, ++at) f(at, (int)(v + __ffs(hits) - 1));
      __syncthreads();
    }
    return true;
  };
  float* out_v = values + (int64_t)blockIdx.x * width;
  int* out_t = tokens + (int64_t)blockIdx.x * width;
  largest(sh, width, max(1, min(kThreads / 32, (count + 31) / 32)), mine, reach, one, equal, [&](int at, float v, int i) {
    out_v[at] = v;
    out_t[at] = i;
  });
  if (tid == kThreads - 32) {                                  // (barriers are behind it; the first warps are still ranking)
    float top = red[0].x, all = 0.f;
#pragma unroll
    for (int u = 1; u < kThreads / 32; ++u) top = fmaxf(top, red[u].x);
    const float from = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int u = 0; u < kThreads / 32; ++u) all += red[u].y * (red[u].x == top ? 1.f : tc::ex2((red[u].x - from) * kLog2e));
    sums[blockIdx.x] = make_float2(top, all);
  }
}

constexpr int kKept = 4;               // candidates of a thread of choose_kernel that are on their way while the sums are made

// MANY: more candidates than the threads keep at hand.  They are lists in order, WIDTH of each run, so the first of a list is its
// largest, and a list is read until it falls below the bound.  A run's list counts as 2^split of them, of every 2^split-th entry.
// (32 beams of 50,304, 13,312 candidates to a group, choose_kernel alone: 68 us with every candidate looked at, 14 us so.)
template <bool MANY>
__global__ void __launch_bounds__(kThreads) choose_kernel(const float* __restrict__ scores, int beams, int vocab, int width, int chunks, int split,
                                                          const float2* sums, const float* values, const int* tokens, float* __restrict__ out_scores,
                                                          int* __restrict__ out_rows, long long* __restrict__ out_tokens) {
  __shared__ Shared<double, long long> sh;
  __shared__ double base[kMaxBeams];                         // score - log-sum-exp of a beam; NaN: all of its scores are -inf
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  // element (a candidate, or a list of MANY) of this thread in every 256: a warp has every eighth, of all beams (of a poor beam alone,
  // its maximum would let all of the others' candidates pass)
  const int place = lane * (kThreads / 32) + (tid >> 5);
  const int per_beam = chunks * width, n = beams * per_beam;
  const int64_t first = (int64_t)g * n;
  float kept_v[kKept];
  int kept_t[kKept], kept_k[kKept];
  if constexpr (!MANY) {
#pragma unroll
    for (int u = 0; u < kKept; ++u) kept_k[u] = (place + u * kThreads) / per_beam;
  }
  int lanes = 32;                                            // of a beam
  while (lanes > 1 && lanes / 2 >= chunks && kThreads / lanes < beams) lanes /= 2;
  const int c0 = tid & (lanes - 1), k_first = tid / lanes;
  float score = k_first < beams ? scores[(int64_t)g * beams + k_first] : 0.f;      // (there before the logits are)
  tc::after_previous_kernel();
  const float2* all = sums + (int64_t)g * beams * chunks;
  float2 own = k_first < beams && c0 < chunks ? all[k_first * chunks + c0] : make_float2(-INFINITY, 0.f);
  if constexpr (!MANY) {
#pragma unroll
    for (int u = 0; u < kKept; ++u) {
      const int i = place + u * kThreads;
      kept_v[u] = i < n ? values[first + i] : 0.f;
      kept_t[u] = i < n ? tokens[first + i] : -1;
    }
  }
  for (int k0 = 0; k0 < beams; k0 += kThreads / lanes) {
    const int k = k0 + k_first;
    const float2* part = all + (int64_t)min(k, beams - 1) * chunks;
    if (k0 > 0) {
      score = scores[(int64_t)g * beams + min(k, beams - 1)];
      own = c0 < chunks ? part[c0] : make_float2(-INFINITY, 0.f);
    }
    float top = own.x;
    for (int c = c0 + lanes; c < chunks; c += lanes) top = fmaxf(top, part[c].x);
    for (int s = lanes / 2; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    auto term = [&](const float2& p) { return p.y != 0.f ? (double)p.y * exp2f((p.x - top) * kLog2e) : 0.0; };   // 0: nothing but -inf; a NaN stays
    double sum = term(own);
    for (int c = c0 + lanes; c < chunks; c += lanes) sum += term(part[c]);
    for (int s = lanes / 2; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    if (c0 == 0 && k < beams) {
      const double b = (double)score - ((double)top + log(sum));
      base[k] = isfinite(b) ? b : nan("");
    }
  }
  __syncthreads();
  auto one = [&](int i, int k, float value, int token, auto f) {    // f(score, place): beam in the upper half of the place, token in the lower
    if (isnan(base[k])) {                                     // equal ones: the lowest tokens stand for all
      const int v = i - k * per_beam;
      if (v < width && v < vocab) f(-(double)INFINITY, ((long long)k << 32) | v);
    } else if (token >= 0) {
      f(base[k] + (double)value, ((long long)k << 32) | token);
    }
  };
  auto each = [&](auto f) {
#pragma unroll
    for (int u = 0; u < kKept; ++u)
      if (place + u * kThreads < n) one(place + u * kThreads, kept_k[u], kept_v[u], kept_t[u], f);
  };
  // f(score, place) for the candidates of this thread's lists, of each until that says no
  auto lists = [&](auto f) {
    const int step = 1 << split, n_lists = (beams * chunks) << split;
#pragma unroll 4
    for (int l = place; l < n_lists; l += kThreads) {
      const int at = (l >> split) * width, k = (l >> split) / chunks;
      bool on = true;
      for (int e = l & (step - 1); e < width && on; e += step)
        one(at + e, k, values[first + at + e], tokens[first + at + e], [&](double x, long long i) { on = f(x, i); });
    }
  };
  double mine = -INFINITY;
  if constexpr (MANY) {
    lists([&](double x, long long) {
      mine = x > mine ? x : mine;
      return false;
    });
  } else {
    each([&](double x, long long) { mine = x > mine ? x : mine; });
  }
  auto reach = [&](double bound, bool above, auto f) {
    bool more = true;
    auto take = [&](double x, long long i) {
      const bool in = above ? x > bound : x >= bound;
      if (more && in) more = f(x, i);
      return more && in;
    };
    if constexpr (MANY) {
      if (above ? mine > bound : mine >= bound) lists(take);
    } else {
      each(take);
    }
  };
  auto equal = [](double, int, auto) { return false; };        // (places are not in order of their index)
  auto rest = [&](auto f) {
    if constexpr (MANY) lists([&](double x, long long i) { return !f(x, i); });
    else each(f);
  };
  largest(sh, width, kThreads / 32, mine, reach, rest, equal, [&](int at, double v, long long i) {
    const int64_t o = (int64_t)g * width + at;
    out_scores[o] = (float)v;
    out_rows[o] = g * beams + (int)(i >> 32);
    out_tokens[o] = i & 0xffffffffLL;
  });
}

// Runs of a beam's vocabulary, a CTA each: as many as make one wave of four CTAs an SM where they fit, none shorter than kLeastUnits.
constexpr int kLeastUnits = 512;
struct Runs { int chunks, units; };
Runs runs_of(int dtype, int rows, int vocab) {
  const int per = dtype == SA_F32 ? 4 : 8;
  const int total = (int)(((int64_t)vocab + per - 1 + per - 1) / per);      // a row may begin up to per - 1 elements into a unit
  const int most = (total + kLeastUnits - 1) / kLeastUnits, least = (total + kMostUnits - 1) / kMostUnits;
  const int chunks = max(least, min(most, max(1, 4 * kSms / rows)));
  const int units = (total + chunks - 1) / chunks;
  return Runs{(total + units - 1) / units, units};
}

}  // namespace

size_t workspace_bytes(int dtype, int groups, int beams, int vocab, int width) {
  return (size_t)groups * beams * runs_of(dtype, groups * beams, vocab).chunks * (8 + 8 * (size_t)width);
}

int select(const Select& p, cudaStream_t s) {
  const int rows = p.groups * p.beams;
  const Runs r = runs_of(p.dtype, rows, p.vocab);
  float2* sums = static_cast<float2*>(p.workspace);
  float* values = reinterpret_cast<float*>(sums + (size_t)rows * r.chunks);
  int* tokens = reinterpret_cast<int*>(values + (size_t)rows * r.chunks * p.width);
  tc::WaitCtx status;
  int st = tc::wait_ctx(&status);
  if (st != SA_OK) return st;
  auto launch = [&](auto kernel, auto ptr) -> int {
    const size_t smem = (size_t)r.units * 16;
    SA_CUDA_CHECK(allow_smem(kernel, smem));
    count_launch();
    kernel<<<(unsigned)rows * r.chunks, kThreads, smem, s>>>(ptr, p.group_stride, p.beam_stride, p.beams, p.vocab, p.width, r.chunks, r.units,
                                                             sums, values, tokens, status);
    SA_CUDA_CHECK(cudaGetLastError());
    return SA_OK;
  };
  switch (p.dtype) {
    case SA_F32: st = launch(candidates_kernel<float>, static_cast<const float*>(p.logits)); break;
    case SA_BF16: st = launch(candidates_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(p.logits)); break;
    case SA_F16: st = launch(candidates_kernel<__half>, static_cast<const __half*>(p.logits)); break;
    default: return SA_ERR_BAD_ARGUMENT;
  }
  if (st != SA_OK) return st;
  auto choose = [&](auto kernel, int split) {
    return launch_after(kernel, dim3(p.groups), kThreads, 0, s, p.scores, p.beams, p.vocab, p.width, r.chunks, split, (const float2*)sums,
                        (const float*)values, (const int*)tokens, p.out_scores, p.out_rows, p.out_tokens);
  };
  const int lists = p.beams * r.chunks;
  if (lists * p.width <= kKept * kThreads) return choose(choose_kernel<false>, 0);
  int split = 0;                                             // a list or more a thread, where that makes enough of them
  while ((lists << (split + 1)) <= kThreads && (2 << split) <= p.width) ++split;
  return choose(choose_kernel<true>, split);
}

}  // namespace beam
}  // namespace sa
