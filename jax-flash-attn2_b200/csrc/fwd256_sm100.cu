// Forward attention for head dim 256: instantiations of fwd256_kernel (fwd256_kernel.cuh) and their dispatch.
#include "fwd256_kernel.cuh"

namespace fa2 {

cudaError_t launch_fwd256(const FwdLaunch& a, cudaStream_t stream) {
  const int key = (a.bf16 ? 4 : 0) | (a.causal ? 2 : 0) | (a.feat ? 1 : 0);
  switch (key) {
    case 0: return launch256_one<false, false, false>(a, stream);
    case 1: return launch256_one<false, false, true>(a, stream);
    case 2: return launch256_one<false, true, false>(a, stream);
    case 3: return launch256_one<false, true, true>(a, stream);
    case 4: return launch256_one<true, false, false>(a, stream);
    case 5: return launch256_one<true, false, true>(a, stream);
    case 6: return launch256_one<true, true, false>(a, stream);
    default: return launch256_one<true, true, true>(a, stream);
  }
}

}  // namespace fa2
