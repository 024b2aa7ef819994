// Backward attention with changed scores (score_mod.cuh), head dim 64: instantiations of the kernels of bwd_kernel.cuh.
#include "bwd_kernel.cuh"

namespace fa2 {

template <bool kBf16, bool kParts>
static cudaError_t launch_mod(const BwdLaunch& a, int mod, cudaStream_t stream) {
  switch (mod) {
    case 0: return launch_main<64, kBf16, false, false, 0, kParts>(a, stream);
    case 1: return launch_main<64, kBf16, false, false, 1, kParts>(a, stream);
    case 2: return launch_main<64, kBf16, false, false, 2, kParts>(a, stream);
    default: return launch_main<64, kBf16, false, false, 3, kParts>(a, stream);
  }
}

template <bool kBf16>
static cudaError_t launch_scored(const BwdLaunch& a, int mod, cudaStream_t stream) {
  return launch_passes<64, kBf16>(a, stream, [mod](const BwdLaunch& l, cudaStream_t s) {
    return l.parts > 1 ? launch_mod<kBf16, true>(l, mod, s) : launch_mod<kBf16, false>(l, mod, s);
  });
}

cudaError_t launch_bwd_scored64(const BwdLaunch& a, int mod, cudaStream_t stream) {
  return a.bf16 ? launch_scored<true>(a, mod, stream) : launch_scored<false>(a, mod, stream);
}

}  // namespace fa2
