// Two heads a CTA that select for themselves, over pages: the launch (the kernel, and what bounds it: sa_tc_fwd_self.cuh).
#include "sa_tc_fwd_self.cuh"

namespace sa {
namespace tc {

int forward_self_pages(const PagedWalk& walk, const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, const float* carry,
                       int items_max, int exempt, float scale, const WaitCtx& status, __nv_bfloat16* y, const RowLayout& y_rows, cudaStream_t s) {
  return launch_after(forward_self_kernel<false, true>, dim3((unsigned)items_max * (walk.heads / 2)), kThreads, SelfSmem::total, s, map_q,
                      map_k, map_v, carry, (float*)nullptr, (float*)nullptr, 0, 0, exempt, scale, status, y, y_rows, 0, (const uint8_t*)nullptr,
                      walk);
}

}  // namespace tc
}  // namespace sa
