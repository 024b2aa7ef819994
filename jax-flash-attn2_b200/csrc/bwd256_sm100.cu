// Backward attention for head dim 256: instantiations of the kernels of bwd256_kernel.cuh and their dispatch.
#include "bwd256_kernel.cuh"

namespace fa2 {

template <bool kBf16>
static cudaError_t launch256_all(const BwdLaunch& a, cudaStream_t stream) {
  return launch256_passes<kBf16>(a, stream, [](const BwdLaunch& l, cudaStream_t s) {
    switch ((l.causal ? 2 : 0) | (l.feat ? 1 : 0)) {
      case 0: return launch256_main<kBf16, false, false>(l, s);
      case 1: return launch256_main<kBf16, false, true>(l, s);
      case 2: return launch256_main<kBf16, true, false>(l, s);
      default: return launch256_main<kBf16, true, true>(l, s);
    }
  });
}

cudaError_t launch_bwd256(const BwdLaunch& a, cudaStream_t stream) {
  return a.bf16 ? launch256_all<true>(a, stream) : launch256_all<false>(a, stream);
}

}  // namespace fa2
