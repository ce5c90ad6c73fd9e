// Tensor-core engine, forward side (sm_100a: TMA loads, tcgen05 MMAs, fp32 accumulators in TMEM).
//
//   colsum_kernel   selection pass: for one 128-key tile and a run of 128-query tiles, the product
//                   K0 Q0^T with KEYS on the TMEM lanes, so a thread owns one key and the column sum of
//                   relu'd, masked logits over the tile's queries is a register reduction.  Writes
//                   COLSUM[b][query tile][key].
//   scan_kernel     exclusive prefix of COLSUM across query tiles, in place (-> CARRY), plus one extra
//                   row holding the grand total.  One thread per key column; bandwidth-bound.
//   forward_wide_kernel  flash-style forward for one 128-query tile of one head over 128-key steps, taken from
//                   the diagonal back to key 0: S = Q K^T and L0 = Q0 K0^T by MMA (Q, Q0 in TMEM); relu(L0) under
//                   the selection mask is written to shared memory as bf16 and the in-tile exclusive running
//                   sum over queries is one more MMA, (-strictly-lower-triangular ones) x selection,
//                   accumulated into S; then online softmax in the log2 domain with the cross-tile carry
//                   subtracted per key, and O += P V in TMEM.  Four arithmetic warpgroups and a control warp
//                   that issues every load and MMA; steps software-pipelined so the tensor pipe works under
//                   the exponentials.  head_dim 128, and head_dim 64 where two heads a CTA would leave SMs idle; few rows
//                   after many cached keys: a piece of the walk each, merged by the CTA that finishes last.
//                   Bound by the chain of a step (L0, selection, running sum, maximum over four warpgroups, exponentials,
//                   P V): 3.1 k cycles at head_dim 64, 3.7 k at 128 (one head per selector, whose single K tile is waited
//                   for: 5.0 k), counted over T = 16384 with the split walk in the same
//                   kernel (it is 1 to 5 % shorter without); the tensor pipe is busy 57 % of them at 128.
//
// Reference for the arithmetic: src/selective_attention/kernels.py:100-194 (selection, carry, forward).
#include <type_traits>

#include "sa_tc_fwd_wide.cuh"

namespace sa {
namespace tc {
namespace {

// ---------------------------------------------------------------------------------------------------
// selection column sums
// ---------------------------------------------------------------------------------------------------
// 128 threads own a key each; a fifth warp's elected lane issues the loads and MMAs, one tile ahead.  Bound by latency and
// issue: 128 compares and 64 packed additions a thread and tile.  (One accumulator and a block-wide barrier a tile, with the
// issuing thread among the 128, took 2.1 k cycles a tile and CTA: the additions alone were a chain of 512.)
constexpr int kColsumThreads = 160;

template <int D>
__global__ void __launch_bounds__(kColsumThreads) colsum_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                const __grid_constant__ CUtensorMap map_k,
                                                                float* __restrict__ carry, int seq, int ntiles, int exempt,
                                                                float scale, WaitCtx status, int q_offset, int mi_first,
                                                                int chunk) {
  constexpr int DK = D / 64;
  const int nj = blockIdx.x, b = blockIdx.z;
  // Query tiles from the key tile's own (the diagonal) on; in a prefill continuation from the first tile that holds a
  // new query on (rows before q_offset are not in the query tensor: TMA fills them with zeros, which select nothing).
  const int mi0 = max(nj, mi_first) + blockIdx.y * chunk;
  if (mi0 >= ntiles) return;
  const int count = min(chunk, ntiles - mi0);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* k0s = smem;                               // DK tiles [128 keys][64]
  uint8_t* q0s = smem + DK * kRowTile;               // 2 stages x DK tiles [128 queries][64]
  __shared__ uint64_t bar_k, bar_q[2], bar_mma[2], bar_read[2];
  __shared__ uint32_t tmem_base_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&bar_k, 1);
    for (int u = 0; u < 2; ++u) {
      mbar_init(&bar_q[u], 1);
      mbar_init(&bar_mma[u], 1);
      mbar_init(&bar_read[u], 4);
    }
    mbar_init_fence();
  }
  if (warp == 0) tmem_alloc(&tmem_base_s, 256);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_base_s;

  if (warp == 4) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc_bf16(128, 128, false, false);
      const uint32_t k_low = desc_low(smem_u32(k0s), 16), q_low = desc_low(smem_u32(q0s), 16);
      auto load_q = [&](int it) {
        uint64_t* bar = &bar_q[it & 1];
        mbar_expect_tx(bar, DK * kRowTile);
        for (int s = 0; s < DK; ++s)
          tma_load_4d(q0s + ((it & 1) * DK + s) * kRowTile, &map_q, bar, s * 64, (mi0 + it) * kTile - q_offset, 0, b);
      };
      mbar_expect_tx(&bar_k, DK * kRowTile);
      for (int s = 0; s < DK; ++s) tma_load_4d(k0s + s * kRowTile, &map_k, &bar_k, s * 64, nj * kTile, 0, b);
      load_q(0);
      if (count > 1) load_q(1);
      mbar_wait(&bar_k, 0, status, 201);
#pragma unroll 1
      for (int it = 0; it < count; ++it) {
        const int st = it & 1;
        const uint32_t ph = (uint32_t)((it >> 1) & 1);
        if (it >= 2) mbar_wait(&bar_read[st], ph ^ 1u, status, 203);      // the columns' last tile has been read
        mbar_wait(&bar_q[st], ph, status, 200);
        tc_fence_after_sync();
        for (int ks = 0; ks < 4 * DK; ++ks) {
          const uint32_t off = (uint32_t)((ks >> 2) * kRowTile + (ks & 3) * 32) >> 4;
          const uint32_t ql = q_low + (uint32_t)(st * DK * kRowTile >> 4) + off;
          if (ks == 0) mma_ss_low<false>(tmem + st * 128, k_low + off, ql, idesc);
          else mma_ss_low<true>(tmem + st * 128, k_low + off, ql, idesc);
        }
        mma_commit(&bar_mma[st]);
        if (it >= 1 && it + 1 < count) {                                  // the other stage: its MMA has completed
          mbar_wait(&bar_mma[st ^ 1], (uint32_t)(((it - 1) >> 1) & 1), status, 204);
          load_q(it + 1);
        }
      }
    }
    __syncwarp();
  } else {
    const uint32_t lane_base = tmem + ((uint32_t)(warp * 32) << 16);
    const int j = nj * kTile + tid;
    float* dst = carry + ((int64_t)b * (ntiles + 1) + mi0) * seq + j;
#pragma unroll 1
    for (int it = 0; it < count; ++it, dst += seq) {
      mbar_wait(&bar_mma[it & 1], (uint32_t)((it >> 1) & 1), status, 202);
      tc_fence_after_sync();
      const bool diag = mi0 + it == nj;
      float2 acc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] = make_float2(0.f, 0.f);
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t r[32];
        tmem_ld32(lane_base + (it & 1) * 128 + c0, r);
        tmem_ld_wait();
        if (diag) {                                                        // (key and query count from the same position)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (tid >= c0 + e) r[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          acc[(e >> 1) & 3] = __fadd2_rn(acc[(e >> 1) & 3], make_float2(fmaxf(__uint_as_float(r[e]), 0.f),
                                                                        fmaxf(__uint_as_float(r[e + 1]), 0.f)));
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_read[it & 1]);
      const float2 s2 = __fadd2_rn(__fadd2_rn(acc[0], acc[1]), __fadd2_rn(acc[2], acc[3]));
      if (j < seq) *dst = (j < exempt) ? 0.f : (s2.x + s2.y) * scale;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 256);
}

// One thread per key column: CARRY[b][mi][j] = sum of COLSUM[b][m'][j] over m' < mi, in place; row `ntiles`
// and total[b][j] receive the sum over all query tiles.  Only rows mi >= j / 128 exist.
__global__ void __launch_bounds__(256) scan_kernel(float* __restrict__ carry, float* total, int64_t total_stride, int seq,
                                                   int ntiles, int mi_first, const float* init,
                                                   int64_t init_stride, bool keep_init, unsigned int* tickets, int n_tickets) {
  if (blockIdx.x == 0 && blockIdx.y == 0 && (int)threadIdx.x < n_tickets) tickets[threadIdx.x] = 0u;   // of a split forward
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  const int b = blockIdx.y;
  if (j >= seq) return;
  float* col = carry + (int64_t)b * (ntiles + 1) * seq + j;
  const float before = init ? init[(int64_t)b * init_stride + j] : 0.f;   // what the key received before the first query given
  float run = before;
  int mi = max(j / kTile, mi_first);
  for (; mi + 8 <= ntiles; mi += 8) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = col[(int64_t)(mi + u) * seq];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      col[(int64_t)(mi + u) * seq] = run;
      run += x[u];
    }
  }
  for (; mi < ntiles; ++mi) {
    float x = col[(int64_t)mi * seq];
    col[(int64_t)mi * seq] = run;
    run += x;
  }
  col[(int64_t)ntiles * seq] = keep_init ? before : run;
  total[(int64_t)b * total_stride + j] = run;                    // (a continued prefill: where `init` was)
}

template <int D>
int forward_impl(const Problem& p, float* out, float* lse2, float* carry, float* total, cudaStream_t s) {
  const int ntiles = (p.seq + kTile - 1) / kTile;
  const int q_rows = p.seq - p.q_offset;                 // rows of the query tensor (all of them unless continuing a prefill)
  const int mi_first = p.q_offset / kTile;               // first query tile with a row to compute
  ForwardMaps m;
  int st = make_map_16bit(&m.q, p.q.ptr, D, q_rows, p.heads, p.batch, p.q.st, p.q.sh, p.q.sb, kTile);
  if (st != SA_OK) return st;
  st = make_map_16bit(&m.k, p.k.ptr, D, p.seq, p.heads, p.batch, p.k.st, p.k.sh, p.k.sb, kTile);
  if (st != SA_OK) return st;
  st = make_map_16bit(&m.v, p.v.ptr, D, p.seq, p.heads, p.batch, p.v.st, p.v.sh, p.v.sb, kTile);
  if (st != SA_OK) return st;
  // the selector's rows: (d, token, 1, batch)
  st = make_map_16bit(&m.q0, p.q0.ptr, D, q_rows, 1, p.batch, p.q0.st, 0, p.q0.sb, kTile);
  if (st != SA_OK) return st;
  st = make_map_16bit(&m.k0, p.k0.ptr, D, p.seq, 1, p.batch, p.k0.st, 0, p.k0.sb, kTile);
  if (st != SA_OK) return st;
  WaitCtx status;
  st = wait_ctx(&status);
  if (st != SA_OK) return st;

  constexpr int DK = D / 64;
  const int colsum_smem = 3 * DK * kRowTile + 1024;
  SA_CUDA_CHECK(allow_smem(colsum_kernel<D>, colsum_smem));
  // query tiles per CTA: 8, or 32 where that still gives every SM several CTAs (the key tile and the set-up are paid per CTA)
  const int64_t tiles = (int64_t)ntiles * (ntiles - mi_first) * p.batch;
  const int chunk = tiles >= 32 * 16 * kSms ? 32 : 8;
  dim3 gc(ntiles, (ntiles - mi_first + chunk - 1) / chunk, p.batch);
  {
    ProfileScope prof(SA_KERNEL_TC_COLSUM, s);
    count_launch();
    colsum_kernel<D><<<gc, kColsumThreads, colsum_smem, s>>>(m.q0, m.k0, carry, p.seq, ntiles, p.exempt, p.scale, status,
                                                             p.q_offset, mi_first, chunk);
  }
  SA_CUDA_CHECK(cudaGetLastError());
  const int pieces = p.split_scratch != nullptr ? prefill_split_pieces(p) : 1;
  const int64_t rows = (int64_t)p.batch * p.heads * q_rows;
  SplitWalk split{pieces, nullptr, nullptr, nullptr};
  if (pieces > 1) {
    split.tickets = reinterpret_cast<unsigned int*>(p.split_scratch);
    split.part = p.split_scratch + kSplitTickets;
    split.lse = split.part + pieces * rows * D;
  }
  dim3 gs((p.seq + 255) / 256, p.batch);
  {
    ProfileScope prof(SA_KERNEL_TC_SCAN, s);
    count_launch();
    scan_kernel<<<gs, 256, 0, s>>>(carry, total, p.total_stride, p.seq, ntiles, mi_first, p.carry_init, p.carry_init_stride,
                                    p.history_moved != nullptr, split.tickets, pieces > 1 ? kSplitTickets : 0);
  }
  SA_CUDA_CHECK(cudaGetLastError());
  if (p.history_moved != nullptr) *p.history_moved = true;

  const uint8_t* alive = nullptr;
  if (p.tile_table != nullptr && ntiles <= kMaxLiveTiles) {
    st = build_tile_table(p, carry, s);
    if (st != SA_OK) return st;
    alive = static_cast<const uint8_t*>(p.tile_table);
  }
  const bool self = self_selecting(p);
  // Heads that share a selector go two to a CTA: its selection is made once and the two overlap (1.3x a head-tile).  While
  // one head a CTA still fits the GPU in one wave, that is faster: a step of it takes 3.1 k cycles, of a pair 4.4 k.
  const int64_t ctas = (int64_t)(ntiles - mi_first) * p.batch * p.heads;
  if (D == 64 && !self && p.heads % 2 == 0 && ctas > kSms) return forward_pair(p, m, carry, out, lse2, status, alive, s);
  if (D == 64 && self && p.batch % 2 == 0 && ctas > kSms) return forward_self(p, m, carry, out, lse2, status, alive, s);
  const unsigned grid = (unsigned)(ntiles - mi_first) * p.batch * p.heads * pieces;
  const int wide_smem = WideSmem<D>::total + 1024;
  auto launch = [&](auto kernel) -> int {
    SA_CUDA_CHECK(allow_smem(kernel, wide_smem));
    ProfileScope prof(SA_KERNEL_TC_FORWARD, s);
    count_launch();
    kernel<<<grid, kWideThreads, wide_smem, s>>>(m.q, m.k, m.v, m.q0, m.k0, carry, out, lse2, p.heads, p.seq,
                                                 ntiles, p.exempt, p.scale, status,
                                                 static_cast<__nv_bfloat16*>(p.out_lowp), p.out_lowp_rows,
                                                 p.q_offset, alive, split, PagedWalk{});
    return SA_OK;
  };
  auto by_split = [&](auto self_tag, auto live_tag) {
    constexpr bool kSelf = decltype(self_tag)::value, kLive = decltype(live_tag)::value;
    return pieces > 1 ? launch(forward_wide_kernel<D, kSelf, kLive, true>) : launch(forward_wide_kernel<D, kSelf, kLive, false>);
  };
  const std::true_type yes;
  const std::false_type no;
  if (alive != nullptr) st = self ? by_split(yes, yes) : by_split(no, yes);
  else st = self ? by_split(yes, no) : by_split(no, no);
  if (st != SA_OK) return st;
  SA_CUDA_CHECK(cudaGetLastError());
  return SA_OK;
}

}  // namespace

// A short chunk after a long cache has few (query tile, head) pairs, each with a long walk: where half of the SMs or more would
// have nothing to do, a walk is cut into as many pieces as give each its SM, of at least 4 steps of 128 keys (a piece pays a
// set-up of about two, and the last one reads all of them).  A prompt is not cut: its rows do not depend on what follows them.
int prefill_split_pieces(const Problem& p) {
  if (p.q_offset == 0) return 1;
  const int ntiles = (p.seq + kTile - 1) / kTile;
  const int64_t ctas = (int64_t)(ntiles - p.q_offset / kTile) * p.batch * p.heads;
  const int64_t pieces = ctas > 0 ? kSms / ctas : 1;
  return (int)(pieces < ntiles / 4 ? (pieces > 1 ? pieces : 1) : (ntiles / 4 > 1 ? ntiles / 4 : 1));
}

int forward(const Problem& p, float* out, float* lse2, float* carry, float* total, cudaStream_t s) {
  if (p.head_dim == 64) return forward_impl<64>(p, out, lse2, carry, total, s);
  if (p.head_dim == 128) return forward_impl<128>(p, out, lse2, carry, total, s);
  return SA_ERR_UNSUPPORTED;
}

}  // namespace tc
}  // namespace sa
