// Attention over a paged cache, head dims up to 128 (paged_attention.cuh), a box of the cache per column block.
#include "paged_attention.cuh"

namespace fa2 {

cudaError_t launch_paged_attention128(const PagedAttnLaunch& a, cudaStream_t stream) {
  return launch_paged_dim<128, false>(a, stream);
}

}  // namespace fa2
