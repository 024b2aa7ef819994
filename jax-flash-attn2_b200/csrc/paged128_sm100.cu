// Attention over a paged cache, head dims up to 128 (paged_attention.cuh).
#include "paged_attention.cuh"

namespace fa2 {

cudaError_t launch_paged_attention128(const PagedAttnLaunch& a, cudaStream_t stream) {
  return launch_paged_dim<128>(a, stream);
}

}  // namespace fa2
