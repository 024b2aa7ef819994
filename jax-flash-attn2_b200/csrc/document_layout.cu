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

// Order in which the forward takes the blocks of 256 query rows: by the key tiles they walk over, longest first (as the
// forward deals them out in rounds of alternating direction, that evens out the SMs' shares: 4 rows of 4096 tokens with
// documents of 700 on average, 32 heads, 148 SMs: longest share 231 tiles in the order of the rows, 191 sorted, mean 189).
// The walk ends at the block's own last key, as under causal masking. A counting sort by one block; blocks of equal length
// land in any order, which changes no result.
constexpr int kOrderBins = 2048;
__global__ void __launch_bounds__(kLayoutThreads)
document_order_kernel(int B, int S, int* __restrict__ layout) {
  __shared__ int bins[kOrderBins];
  __shared__ int warp_tot[32];
  const long long BS = static_cast<long long>(B) * S;
  const int nt = (S + 127) >> 7, nq = (S + 255) >> 8, n = B * nq, tid = threadIdx.x;
  const int* tile_lo = layout + 2 * BS;
  const int* tile_hi = tile_lo + static_cast<long long>(B) * nt;
  int* order = layout + 2 * BS + 2 * static_cast<long long>(B) * nt;
  // bin of a block: 0 for the longest
  auto bin = [&](int i) {
    const int b = i / nq, q = i - b * nq;
    int first = INT_MAX, end = 0;
    for (int t = 2 * q; t < min(nt, 2 * q + 2); ++t) {
      const long long at = static_cast<long long>(b) * nt + t;
      const int hi = min(tile_hi[at], min(S, t * 128 + 128));
      if (hi > tile_lo[at]) {
        first = min(first, tile_lo[at]);
        end = max(end, hi);
      }
    }
    const int len = end > 0 ? ((end + 127) >> 7) - (first >> 7) : 0;
    return kOrderBins - 1 - min(len, kOrderBins - 1);
  };
  for (int k = tid; k < kOrderBins; k += kLayoutThreads) bins[k] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kLayoutThreads) atomicAdd(bins + bin(i), 1);
  __syncthreads();
  // exclusive sum over the bins, two per thread
  const int own0 = bins[2 * tid], own1 = bins[2 * tid + 1];
  const int incl = block_scan<false>(own0 + own1, [](int x, int y) { return x + y; }, warp_tot);
  __syncthreads();
  bins[2 * tid] = incl - own0 - own1;
  bins[2 * tid + 1] = incl - own1;
  __syncthreads();
  for (int i = tid; i < n; i += kLayoutThreads) order[atomicAdd(bins + bin(i), 1)] = i;
}
static_assert(kOrderBins == 2 * kLayoutThreads, "two bins per thread");

}  // namespace

cudaError_t launch_document_layout(const int* ids, long long stride_b, int B, int S, int* layout, cudaStream_t stream) {
  document_layout_kernel<<<static_cast<unsigned>(B), kLayoutThreads, 0, stream>>>(ids, stride_b, B, S, layout);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  document_order_kernel<<<1, kLayoutThreads, 0, stream>>>(B, S, layout);
  return cudaGetLastError();
}

}  // namespace fa2
