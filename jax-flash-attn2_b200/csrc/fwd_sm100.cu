// Forward attention for head dims 64 and 128: instantiations of fwd_kernel (fwd_kernel.cuh) for every dtype,
// mask and feature set, and their dispatch.
#include "fwd_kernel.cuh"

namespace fa2 {

template <int D>
static cudaError_t launch_d(const FwdLaunch& a, cudaStream_t stream) {
  const int key = (a.bf16 ? 4 : 0) | (a.causal ? 2 : 0) | (a.feat ? 1 : 0);
  switch (key) {
    case 0: return launch_one<D, false, false, false>(a, stream);
    case 1: return launch_one<D, false, false, true>(a, stream);
    case 2: return launch_one<D, false, true, false>(a, stream);
    case 3: return launch_one<D, false, true, true>(a, stream);
    case 4: return launch_one<D, true, false, false>(a, stream);
    case 5: return launch_one<D, true, false, true>(a, stream);
    case 6: return launch_one<D, true, true, false>(a, stream);
    default: return launch_one<D, true, true, true>(a, stream);
  }
}

cudaError_t launch_fwd(const FwdLaunch& a, cudaStream_t stream) {
  switch (a.head_dim) {
    case 64: return launch_d<64>(a, stream);
    case 128: return launch_d<128>(a, stream);
    case 256: return launch_fwd256(a, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace fa2
