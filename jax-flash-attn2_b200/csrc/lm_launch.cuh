// Host-side launchers of the operators declared in fa2_b200_lm.h.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace fa2 {

cudaError_t launch_document_layout(const int* ids, long long stride_b, int B, int S, int* layout, cudaStream_t stream);

}  // namespace fa2
