// The plan of a serving step over a paged key/value cache, and the write of its new keys and values.
//
// Request b has c_b tokens in the cache and brings n_b new ones; a page holds 2^s tokens.
//   cu_b   = n_0 + ... + n_(b-1)                       first row of its tokens in the packed tensors
//   have_b = ceil(c_b / 2^s),  need_b = ceil((c_b + n_b) / 2^s)
//   fresh_b = sum over the requests before b of need - have: its pages in the list of free ones start there
//   token i of it: position c_b + i, slot = page(position >> s) * 2^s + position mod 2^s
// and the work list of the attention: items of `item_tokens` query tokens with the number of 128-key tiles that each
// of them sees. All tiles of all items of all key/value heads form a line as long as their costs (lm_launch.cuh; an item
// begins with the cost of its start and end), which is cut into equal shares, one per SM. A border that falls next to
// an end of an item moves to that end, by at most snap_of (and half a share): an item that is cut costs partial rows of both
// sides, written and joined, about as much as two tiles of 256 rows or half a tile of a few.
// (36 x 4 items of two tiles and 256 rows, D = 64: 31 us with every border where it falls, 19 us with moved ones, 12 today.
// Prompts and single tokens over up to 3000 keys, 32/8 heads, D = 128: 95 us with these costs, 106 us with a tile of 256 rows
// counted as two of a few and two tiles for every start.)
//
// One launch. Every block scans the requests by itself in shared memory (a few thousand numbers: cheaper than a second
// launch that waits for the first), then block 0 writes the work list while the others place tokens, one per thread.
// A page that is new is entered into the table by the token that opens it. All of it is latency: a launch, two block
// scans and a dozen dependent shared-memory reads of a binary search (32 decodes 5.6 us, 700 requests 8.0 us; with the places of
// the items searched in global memory 7.3 and 10.0).
#include <climits>

#include "launch_util.cuh"
#include "lm_launch.cuh"

namespace fa2 {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kKnownItems = 4096;      // the items whose place in the line is kept in shared memory

// Exclusive scan over the block; returns the sum before this thread, `total` the sum of all.
template <class T>
__device__ __forceinline__ T block_exclusive(T v, T* warp_tot, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T o = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += o;
  }
  if (lane == 31) warp_tot[warp] = x;
  __syncthreads();
  if (warp == 0) {
    T t = warp_tot[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const T o = __shfl_up_sync(0xffffffffu, t, d);
      if (lane >= d) t += o;
    }
    warp_tot[lane] = t;
  }
  __syncthreads();
  const T before = warp ? warp_tot[warp - 1] : T(0);
  total = warp_tot[31];
  __syncthreads();      // warp_tot may be used again
  return before + x - v;
}

// How far a border may move, by the cost of the item's tiles.
__device__ __forceinline__ int snap_of(int cost) { return cost == kTileCost2 ? 2 * kTileCost2 : kTileCost1; }
__device__ __forceinline__ int item_cost(int cost) { return cost == kTileCost2 ? kItemCost2 : kItemCost1; }

// Largest index r in [0, n) with a[r] <= x (a ascends, a[0] <= x).
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads)
paged_plan_kernel(const PagedPlanDev p) {
  extern __shared__ int smem[];
  __shared__ long long warp_tot[32];
  __shared__ int item_before[kKnownItems];     // block 0: cost of the items before each of the first ones
  int* cu = smem;                    // [B + 1]
  int* fresh = smem + p.B + 1;       // [B]; block 0 then keeps the items' offsets here
  const int tid = threadIdx.x;
  const int per = (p.B + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(p.B, tid * per), r1 = min(p.B, r0 + per);
  const long long page = 1LL << p.page_shift;
  const long long capacity = static_cast<long long>(p.table_width) << p.page_shift;
  // (lengths below 0 count as 0; new tokens that the packed tensors have no row for are cut off)
  auto context = [&](int r) { return static_cast<long long>(max(0, __ldg(p.context_lens + r))); };
  auto pages = [&](long long tokens) { return (min(tokens, capacity) + page - 1) >> p.page_shift; };

  long long sum = 0, total;
  // (wanted after the first scan: on its way meanwhile)
  if (r0 < r1) asm volatile("prefetch.global.L1 [%0];" ::"l"(p.context_lens + r0));
  for (int r = r0; r < r1; ++r) sum += max(0, __ldg(p.new_lens + r));
  long long run = block_exclusive(sum, warp_tot, total);
  for (int r = r0; r < r1; ++r) {
    cu[r] = static_cast<int>(min(run, static_cast<long long>(p.num_tokens)));
    run += max(0, __ldg(p.new_lens + r));
  }
  if (tid == 0) cu[p.B] = static_cast<int>(min(total, static_cast<long long>(p.num_tokens)));
  __syncthreads();
  sum = 0;
  for (int r = r0; r < r1; ++r) sum += pages(context(r) + cu[r + 1] - cu[r]) - pages(context(r));
  run = block_exclusive(sum, warp_tot, total);
  for (int r = r0; r < r1; ++r) {
    fresh[r] = static_cast<int>(run);
    run += pages(context(r) + cu[r + 1] - cu[r]) - pages(context(r));
  }
  __syncthreads();

  if (blockIdx.x > 0) {
    // ---- tokens
    const int t = (static_cast<int>(blockIdx.x) - 1) * kPlanThreads + tid;
    if (t >= p.num_tokens) return;
    long long slot = -1, pos = 0;
    if (t < cu[p.B]) {
      // (requests without new tokens share their offset with the next one, which the search then finds)
      const int r = last_not_above(cu, p.B, t);
      const long long c = context(r);
      pos = c + t - cu[r];
      const long long pi = pos >> p.page_shift, have = pages(c);
      int* row = p.block_table + r * p.table_stride;
      if (pi < p.table_width) {
        int id = -1;
        if (pi < have) {
          id = row[pi];
        } else {
          const long long at = static_cast<long long>(p.free_start ? max(0, __ldg(p.free_start)) : 0) + fresh[r] + (pi - have);
          if (at < p.n_free) id = __ldg(p.free_pages + at);
          if ((pos & (page - 1)) == 0) row[pi] = id;
        }
        if (id >= 0) slot = (static_cast<long long>(id) << p.page_shift) + (pos & (page - 1));
      }
    }
    p.slot_map[t] = slot;
    p.positions[t] = static_cast<int>(min(pos, static_cast<long long>(INT_MAX)));
    return;
  }

  // ---- block 0: lengths and the work list
  if (tid == 0) p.pages_taken[0] = static_cast<int>(total);
  sum = 0;
  for (int r = r0; r < r1; ++r) {
    p.cu_seqlens[r] = cu[r];
    p.seqlens_k[r] = static_cast<int>(min(context(r) + cu[r + 1] - cu[r], static_cast<long long>(INT_MAX)));
    sum += (cu[r + 1] - cu[r] + p.item_tokens - 1) / p.item_tokens;
  }
  if (tid == 0) p.cu_seqlens[p.B] = cu[p.B];
  int* first_item = fresh;
  run = block_exclusive(sum, warp_tot, total);
  const int n_items = static_cast<int>(total);
  for (int r = r0; r < r1; ++r) {
    first_item[r] = static_cast<int>(run);
    run += (cu[r + 1] - cu[r] + p.item_tokens - 1) / p.item_tokens;
  }
  __syncthreads();
  long long carry = 0;
  int pairs = 0;                 // whether this thread has seen an item of two query tiles
  int4* items = reinterpret_cast<int4*>(p.work + p.items_at);
  for (int base = 0; base < n_items; base += kPlanThreads) {
    const int i = base + tid;
    int4 a = make_int4(0, 0, 0, 0);
    long long tiles = 0;
    int cost = kTileCost1;
    if (i < n_items) {
      const int r = last_not_above(first_item, p.B, i);
      const int t0 = (i - first_item[r]) * p.item_tokens;
      const int n = min(p.item_tokens, cu[r + 1] - cu[r] - t0);
      const long long pos0 = context(r) + t0;
      a = make_int4(cu[r] + t0, n, static_cast<int>(min(pos0, static_cast<long long>(INT_MAX / 2))), r);
      tiles = max(1LL, (min(pos0 + n, capacity) + 127) >> 7);
      cost = 2 * n > p.item_tokens ? kTileCost2 : kTileCost1;
      pairs |= cost == kTileCost2;
    }
    long long all;
    const long long before = carry + block_exclusive(i < n_items ? tiles * cost + item_cost(cost) : 0LL, warp_tot, all);
    if (i < n_items) {
      items[2 * i] = a;
      items[2 * i + 1] = make_int4(static_cast<int>(before), static_cast<int>(tiles), cost, 0);
      if (i < kKnownItems) item_before[i] = static_cast<int>(before);
    }
    carry += all;
  }
  // ---- shares (the items written above are visible to the block behind the barrier)
  const bool any_pair = __syncthreads_or(pairs) != 0;
  const long long per_head = carry, line = per_head * p.heads_kv;
  // (no more shares than key tiles, about: one without a tile costs the join the look at it)
  const int ctas = static_cast<int>(min(line / kTileCost1, static_cast<long long>(p.sms)));
  if (tid == 0) {
    p.work[0] = n_items;
    p.work[1] = ctas;
  }
  if (ctas == 0) return;
  // Single tokens alone: shares of whole key tiles (1 x 8000 keys, 32/8 heads, D = 128 18.7 us, 19.8 with halves of them);
  // with chunks among them as even as the costs allow (the second case above 95 us, 99 in whole tiles).
  const int unit = any_pair ? 1 : kTileCost1;
  const long long units = any_pair ? line : line / kTileCost1, share = units / ctas, extra = units - share * ctas;
  const int* prefix = p.work + p.items_at + 4;
  for (int c = tid; c <= ctas; c += kPlanThreads) {
    int4 start = make_int4(p.heads_kv, 0, 0, 0);
    if (c < ctas) {
      const long long g = unit * (share * c + min(static_cast<long long>(c), extra));
      const int hk = static_cast<int>(g / per_head);
      const int rem = static_cast<int>(g - hk * per_head);
      int lo = 0, hi = n_items;      // the item with the largest prefix not above rem
      if (n_items <= kKnownItems) {
        lo = last_not_above(item_before, n_items, rem);
      } else {
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (prefix[static_cast<long long>(mid) * kWorkItem] <= rem) lo = mid; else hi = mid;
        }
      }
      const int4 item = items[2 * static_cast<long long>(lo) + 1];
      const int cost = item.z, in = max(0, rem - item.x - item_cost(cost)), left = item.y * cost - in;
      const int snap = static_cast<int>(min(static_cast<long long>(snap_of(cost)), share * unit >> 1));
      int tile = (in + cost - 1) / cost;
      if (in <= snap && in <= left) tile = 0;
      else if (left <= snap) tile = item.y;
      start = make_int4(hk, lo, tile, cost == kTileCost2);
      if (tile >= item.y) start = lo + 1 < n_items ? make_int4(hk, lo + 1, 0, 0) : make_int4(hk + 1, 0, 0, 0);
    }
    reinterpret_cast<int4*>(p.work + kWorkHeader)[c] = start;
  }
}

// Copies a token's keys and values to its slot, 16 bytes of each per thread. HBM-bound: every byte is read and written
// once, consecutive threads take consecutive chunks of a token's heads.
__global__ void __launch_bounds__(256)
paged_write_kernel(const PagedWriteDev p) {
  const int per_token = p.heads * p.chunks_per_head;
  const long long idx = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const long long t = idx / per_token;
  if (t >= p.tokens) return;
  const int rest = static_cast<int>(idx - t * per_token);
  const int h = rest / p.chunks_per_head, c = rest - h * p.chunks_per_head;
  const long long slot = __ldg(p.slot_map + t);
  if (slot < 0 || slot >= p.slots) return;      // a row without a slot is not written
  const uint4 k = __ldg(reinterpret_cast<const uint4*>(p.k + t * p.k_st + h * p.k_sh) + c);
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(p.v + t * p.v_st + h * p.v_sh) + c);
  const long long pg = slot >> p.page_shift, in = slot & ((1LL << p.page_shift) - 1);
  reinterpret_cast<uint4*>(p.k_cache + pg * p.kc_sp + in * p.kc_ss + h * p.kc_sh)[c] = k;
  reinterpret_cast<uint4*>(p.v_cache + pg * p.vc_sp + in * p.vc_ss + h * p.vc_sh)[c] = v;
}

}  // namespace

cudaError_t launch_paged_plan(const PagedPlanDev& p, cudaStream_t stream) {
  const int bytes = (2 * p.B + 1) * static_cast<int>(sizeof(int));
  if (bytes > 48 * 1024 - kKnownItems * 4 - 512) {
    static bool opted_in[64] = {};
    const cudaError_t e = opt_in_dynamic_smem(paged_plan_kernel, 2 * 8192 * 4 + 64, opted_in);
    if (e != cudaSuccess) return e;
  }
  const unsigned grid = 1u + static_cast<unsigned>((p.num_tokens + kPlanThreads - 1LL) / kPlanThreads);
  paged_plan_kernel<<<grid, kPlanThreads, bytes, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_paged_write(const PagedWriteDev& p, cudaStream_t stream) {
  const long long threads = static_cast<long long>(p.tokens) * p.heads * p.chunks_per_head;
  paged_write_kernel<<<static_cast<unsigned>((threads + 255) / 256), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace fa2
