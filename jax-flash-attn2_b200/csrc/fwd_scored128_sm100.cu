// Forward attention with changed scores (score_mod.cuh), head dim 128: instantiations of fwd_kernel (fwd_kernel.cuh).
#include "fwd_kernel.cuh"

namespace fa2 {

cudaError_t launch_fwd_scored128(const FwdLaunch& a, int mod, cudaStream_t stream) {
  switch ((a.bf16 ? 4 : 0) | mod) {
    case 0: return launch_one<128, false, false, false, 0>(a, stream);
    case 1: return launch_one<128, false, false, false, 1>(a, stream);
    case 2: return launch_one<128, false, false, false, 2>(a, stream);
    case 3: return launch_one<128, false, false, false, 3>(a, stream);
    case 4: return launch_one<128, true, false, false, 0>(a, stream);
    case 5: return launch_one<128, true, false, false, 1>(a, stream);
    case 6: return launch_one<128, true, false, false, 2>(a, stream);
    default: return launch_one<128, true, false, false, 3>(a, stream);
  }
}

}  // namespace fa2
