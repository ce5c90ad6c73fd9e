// Two rows a CTA that select for themselves: the launch over contiguous keys and values (the kernel, and what bounds it:
// sa_tc_fwd_self.cuh).
#include "sa_tc_fwd_self.cuh"

namespace sa {
namespace tc {

int forward_self(const Problem& p, const ForwardMaps& m, const float* carry, float* out, float* lse2, const WaitCtx& status,
                 const uint8_t* alive, cudaStream_t s) {
  const int ntiles = (p.seq + kTile - 1) / kTile;
  const unsigned grid = (unsigned)(ntiles - p.q_offset / kTile) * (p.batch / 2);
  const int smem = SelfSmem::total;
  auto launch = [&](auto kernel) -> int {
    SA_CUDA_CHECK(allow_smem(kernel, smem));
    ProfileScope prof(SA_KERNEL_TC_FORWARD, s);
    count_launch();
    kernel<<<grid, kThreads, smem, s>>>(m.q, m.k, m.v, carry, out, lse2, p.seq, ntiles, p.exempt, p.scale, status,
                                        static_cast<__nv_bfloat16*>(p.out_lowp), p.out_lowp_rows, p.q_offset, alive, PagedWalk{});
    SA_CUDA_CHECK(cudaGetLastError());
    return SA_OK;
  };
  return alive != nullptr ? launch(forward_self_kernel<true>) : launch(forward_self_kernel<false>);
}

}  // namespace tc
}  // namespace sa
