// Attention over a paged cache, head dims up to 64 (paged_attention.cuh), and the dispatch by head dim.
#include "paged_attention.cuh"

namespace fa2 {

cudaError_t launch_paged_attention128(const PagedAttnLaunch& a, cudaStream_t stream);
cudaError_t launch_paged_attention128_rows(const PagedAttnLaunch& a, cudaStream_t stream);

cudaError_t launch_paged_attention(const PagedAttnLaunch& a, cudaStream_t stream) {
  return a.head_dim == 64 ? launch_paged_dim<64, false>(a, stream)
         : a.whole_rows   ? launch_paged_attention128_rows(a, stream)
                          : launch_paged_attention128(a, stream);
}

}  // namespace fa2
