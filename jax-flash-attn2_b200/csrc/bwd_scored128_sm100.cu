// Backward attention with changed scores (score_mod.cuh), head dim 128: instantiations of the kernels of bwd_kernel.cuh.
#include "bwd_kernel.cuh"

namespace fa2 {

template <bool kBf16>
static cudaError_t launch_scored(const BwdLaunch& a, int mod, cudaStream_t stream) {
  return launch_passes<128, kBf16>(a, stream, [mod](const BwdLaunch& l, cudaStream_t s) {
    switch (mod) {
      case 0: return launch_main<128, kBf16, false, false, 0>(l, s);
      case 1: return launch_main<128, kBf16, false, false, 1>(l, s);
      case 2: return launch_main<128, kBf16, false, false, 2>(l, s);
      default: return launch_main<128, kBf16, false, false, 3>(l, s);
    }
  });
}

cudaError_t launch_bwd_scored128(const BwdLaunch& a, int mod, cudaStream_t stream) {
  return a.bf16 ? launch_scored<true>(a, mod, stream) : launch_scored<false>(a, mod, stream);
}

}  // namespace fa2
