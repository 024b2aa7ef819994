// Backward attention for head dims 64 and 128: instantiations of the kernels of bwd_kernel.cuh and their dispatch.
#include "bwd_kernel.cuh"

namespace fa2 {

template <int D, bool kBf16>
static cudaError_t launch_all(const BwdLaunch& a, cudaStream_t stream) {
  return launch_passes<D, kBf16>(a, stream, [](const BwdLaunch& l, cudaStream_t s) {
    switch ((l.causal ? 2 : 0) | (l.feat ? 1 : 0)) {
      case 0: return launch_main<D, kBf16, false, false>(l, s);
      case 1: return launch_main<D, kBf16, false, true>(l, s);
      case 2: return launch_main<D, kBf16, true, false>(l, s);
      default: return launch_main<D, kBf16, true, true>(l, s);
    }
  });
}

cudaError_t launch_bwd(const BwdLaunch& a, cudaStream_t stream) {
  if (a.head_dim == 64) return a.bf16 ? launch_all<64, true>(a, stream) : launch_all<64, false>(a, stream);
  if (a.head_dim == 128) return a.bf16 ? launch_all<128, true>(a, stream) : launch_all<128, false>(a, stream);
  if (a.head_dim == 256) return launch_bwd256(a, stream);
  return cudaErrorInvalidValue;
}

}  // namespace fa2
