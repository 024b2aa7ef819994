// Layout of packed documents: for every token the bounds of its document, and the bounds over every 128 tokens.
//
// A document is a run of equal ids. With c_s = 1 where the id of token s differs from that of s - 1,
//   first(s) = max { t <= s : c_t = 1 },   end(s) = min { t > s : c_t = 1 or t = S },
// a maximum scan from the left and a minimum scan from the right. One block per row: it walks the row in pieces
// of 4096 tokens (four per thread), scans a piece with warp shuffles and carries the result on. The work is a few
// reads and writes of 4 bytes per token and the kernel is bound by the latency of its piece-by-piece walk: about
// 2 us a piece, beside an attention call that grows with the square of the row.
#include <climits>

#include "lm_launch.cuh"

namespace fa2 {

namespace {

constexpr int kLayoutThreads = 1024;
constexpr int kPerThread = 4;
constexpr int kPiece = kLayoutThreads * kPerThread;

// Inclusive scan over the block, from thread 0 upwards or (kDown) from the last thread downwards; Op is max or min.
template <bool kDown, class Op>
__device__ __forceinline__ int block_scan(int v, Op op, int* warp_tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = kDown ? __shfl_down_sync(0xffffffffu, v, d) : __shfl_up_sync(0xffffffffu, v, d);
    if (kDown ? lane + d < 32 : lane >= d) v = op(v, o);
  }
  if (lane == (kDown ? 0 : 31)) warp_tot[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int t = warp_tot[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = kDown ? __shfl_down_sync(0xffffffffu, t, d) : __shfl_up_sync(0xffffffffu, t, d);
      if (kDown ? lane + d < 32 : lane >= d) t = op(t, o);
    }
    warp_tot[lane] = t;
  }
  __syncthreads();
  if (kDown ? warp < 31 : warp > 0) v = op(v, warp_tot[kDown ? warp + 1 : warp - 1]);
  return v;
}

__global__ void __launch_bounds__(kLayoutThreads)
document_layout_kernel(const int* __restrict__ ids, long long stride_b, int B, int S, int* __restrict__ layout) {
  __shared__ int warp_tot[32];
  __shared__ int carry;
  const int b = blockIdx.x, tid = threadIdx.x;
  const long long BS = static_cast<long long>(B) * S;
  const int nt = (S + 127) >> 7;
  int* tok_lo = layout + static_cast<long long>(b) * S;
  int* tok_hi = tok_lo + BS;
  int* tile_lo = layout + 2 * BS + static_cast<long long>(b) * nt;
  int* tile_hi = tile_lo + static_cast<long long>(B) * nt;
  const int* row = ids + b * stride_b;
  const int pieces = (S + kPiece - 1) / kPiece;

  auto begins = [&](int s) { return s == 0 || __ldg(row + s) != __ldg(row + s - 1); };
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int pc = 0; pc < pieces; ++pc) {
    const int s0 = pc * kPiece + tid * kPerThread;
    int own[kPerThread], last = -1;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      if (s0 + k < S && begins(s0 + k)) last = s0 + k;
      own[k] = last;
    }
    const int incl = block_scan<false>(last, [](int x, int y) { return max(x, y); }, warp_tot);
    // what lies before this thread's tokens: the scan up to the previous thread, or the piece before
    int before = __shfl_up_sync(0xffffffffu, incl, 1);
    if ((tid & 31) == 0) before = tid ? warp_tot[(tid >> 5) - 1] : -1;
    before = max(before, carry);
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (s0 + k < S) tok_lo[s0 + k] = __ldg(row + s0 + k) < 0 ? 0 : max(own[k], before);
    __syncthreads();                        // carry and warp_tot have been read
    if (tid == kLayoutThreads - 1) carry = max(incl, carry);
    __syncthreads();
  }
  if (tid == 0) carry = S;
  __syncthreads();
  for (int pc = pieces - 1; pc >= 0; --pc) {
    const int s0 = pc * kPiece + tid * kPerThread;
    int own[kPerThread], next = INT_MAX;    // first start at or behind token s0 + k, among this thread's tokens
#pragma unroll
    for (int k = kPerThread - 1; k >= 0; --k) {
      own[k] = next;                        // starts behind token s0 + k
      if (s0 + k < S && begins(s0 + k)) next = s0 + k;
    }
    const int incl = block_scan<true>(next, [](int x, int y) { return min(x, y); }, warp_tot);
    int behind = __shfl_down_sync(0xffffffffu, incl, 1);
    if ((tid & 31) == 31) behind = tid < kLayoutThreads - 1 ? warp_tot[(tid >> 5) + 1] : INT_MAX;
    behind = min(behind, carry);
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (s0 + k < S) tok_hi[s0 + k] = __ldg(row + s0 + k) < 0 ? 0 : min(own[k], behind);
    __syncthreads();
    if (tid == 0) carry = min(incl, carry);
    __syncthreads();
  }
  // (the block's own writes to tok_lo / tok_hi are visible to it behind the barrier)
  const int lane = tid & 31;
  for (int t = tid >> 5; t < nt; t += kLayoutThreads / 32) {
    int lo = INT_MAX, hi = 0;
    for (int s = t * 128 + lane; s < min(S, t * 128 + 128); s += 32) {
      const int h = tok_hi[s];
      if (h > 0) {
        lo = min(lo, tok_lo[s]);
        hi = max(hi, h);
      }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      tile_lo[t] = hi > 0 ? lo : 0;
      tile_hi[t] = hi;
    }
  }
}

}  // namespace

cudaError_t launch_document_layout(const int* ids, long long stride_b, int B, int S, int* layout, cudaStream_t stream) {
  document_layout_kernel<<<static_cast<unsigned>(B), kLayoutThreads, 0, stream>>>(ids, stride_b, B, S, layout);
  return cudaGetLastError();
}

}  // namespace fa2
