// Layer norm and the embedding: what sa_norm.cu, sa_embed.cu and the C entry points share.
#pragma once

#include "sa_common.cuh"
#include "sa_tc_ptx.cuh"

namespace sa {

namespace norm {
constexpr int kMaxWidth = 16384;
size_t backward_bytes(const sa_norm& p);
int forward(const sa_norm& p, cudaStream_t s);
int backward(const sa_norm& p, cudaStream_t s);
}  // namespace norm

namespace embed {
// out[v] = scale * the sum of factor[n] * dy[n] over the n with idx[n] = v, in their order, or that added to fp32 rows.
struct RowSums {
  const int64_t* idx;           // those outside [0, vocab), and `skip`, have no part
  int64_t skip;
  int tokens, vocab, width;
  const void* dy;
  int dtype;
  int64_t dy_stride;
  const float* factor;          // null: 1
  float scale;
  void* out;                    // (vocab, width), contiguous
  int out_dtype;
  bool add;
  void* workspace;              // sum_rows_bytes(), 16-byte aligned
};
size_t sum_rows_bytes(int tokens, int vocab, int width);
int sum_rows(const RowSums& r, cudaStream_t s);
size_t backward_bytes(const sa_embedding& p);
int forward(const sa_embedding& p, cudaStream_t s);
int backward(const sa_embedding& p, cudaStream_t s);
}  // namespace embed

// ---- rows of any type, eight values a thread at a time --------------------------------------------------------------------------
// Thread t of T holds NV x 8 values of a row.  VEC: eight neighbours, in one load of 16 or 32 bytes (the width is a multiple of 8, rows
// begin at multiples of those bytes); otherwise values T apart, so that a warp's loads are whole sectors all the same.
template <int T, bool VEC>
__device__ __forceinline__ int column_of(int chunk, int i, int t) {
  return VEC ? (chunk * T + t) * 8 + i : (chunk * 8 + i) * T + t;
}

// Whether a value lies in the row: with VEC one question for the eight.
template <int T, bool VEC>
__device__ __forceinline__ bool in_row(int chunk, int i, int t, int width) {
  return column_of<T, VEC>(chunk, VEC ? 0 : i, t) < width;
}

__device__ __forceinline__ void unpack_pair(uint32_t w, bool half, float* to) {
  if (half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    to[0] = f.x;
    to[1] = f.y;
  } else {
    to[0] = __uint_as_float(w << 16);
    to[1] = __uint_as_float(w & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void load_eight(const float* p, float (&v)[8]) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void store_eight(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, bool half) {
  if (half) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return tc::pack_bf16(lo, hi);
}

// The branch on the type is around all loads of a row, so that they are in flight together.
// SHARED: from shared memory, at a multiple of 16 bytes.
template <int NV, int T, bool VEC, bool SHARED = false>
__device__ __forceinline__ void load_row(float (&v)[NV][8], const void* base, int dtype, int64_t at, int width, int t) {
  if (dtype == SA_F32) {
    const float* p = static_cast<const float*>(base) + at;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      if (VEC) {
        if (column_of<T, VEC>(c, 0, t) >= width) continue;
        if (SHARED) {
          const float4* q = reinterpret_cast<const float4*>(p + column_of<T, VEC>(c, 0, t));
          const float4 a = q[0], b = q[1];
          v[c][0] = a.x; v[c][1] = a.y; v[c][2] = a.z; v[c][3] = a.w; v[c][4] = b.x; v[c][5] = b.y; v[c][6] = b.z; v[c][7] = b.w;
        } else {
          load_eight(p + column_of<T, VEC>(c, 0, t), v[c]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (column_of<T, VEC>(c, i, t) < width) v[c][i] = p[column_of<T, VEC>(c, i, t)];
      }
    }
    return;
  }
  const uint16_t* p = static_cast<const uint16_t*>(base) + at;
  const bool half = dtype == SA_F16;
  uint32_t raw[NV][4];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    if (VEC) {
      if (column_of<T, VEC>(c, 0, t) < width) {
        const uint4 q = *reinterpret_cast<const uint4*>(p + column_of<T, VEC>(c, 0, t));
        raw[c][0] = q.x; raw[c][1] = q.y; raw[c][2] = q.z; raw[c][3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = column_of<T, VEC>(c, 2 * i, t), b = column_of<T, VEC>(c, 2 * i + 1, t);
        raw[c][i] = (a < width ? p[a] : 0u) | ((b < width ? (uint32_t)p[b] : 0u) << 16);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < NV; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack_pair(raw[c][i], half, &v[c][2 * i]);
}

template <int NV, int T, bool VEC>
__device__ __forceinline__ void store_row(const float (&v)[NV][8], void* base, int dtype, int64_t at, int width, int t) {
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    if (VEC) {
      if (column_of<T, VEC>(c, 0, t) >= width) continue;
      if (dtype == SA_F32) {
        store_eight(static_cast<float*>(base) + at + column_of<T, VEC>(c, 0, t), v[c]);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_pair(v[c][2 * i], v[c][2 * i + 1], dtype == SA_F16);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at + column_of<T, VEC>(c, 0, t)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int col = column_of<T, VEC>(c, i, t);
        if (col >= width) continue;
        if (dtype == SA_F32) static_cast<float*>(base)[at + col] = v[c][i];
        else static_cast<uint16_t*>(base)[at + col] = (uint16_t)pack_pair(v[c][i], 0.f, dtype == SA_F16);
      }
    }
  }
}

__device__ __forceinline__ float rounded_to(float x, int dtype) {
  if (dtype == SA_BF16) return __bfloat162float(__float2bfloat16_rn(x));
  if (dtype == SA_F16) return __half2float(__float2half_rn(x));
  return x;
}

// Whether rows of a tensor can be read eight values at a time.
inline bool eights(const void* p, int dtype, int64_t stride, int64_t rows) {
  const int64_t bytes = dtype == SA_F32 ? 4 : 2;
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) % (8 * bytes)) == 0 && (rows <= 1 || stride % 8 == 0));
}

}  // namespace sa
