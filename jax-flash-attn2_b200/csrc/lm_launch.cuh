// Host-side launch records of the operators declared in fa2_b200_lm.h.
#pragma once
#include <cstdint>

#include <cuda.h>
#include <cuda_runtime.h>

namespace fa2 {

cudaError_t launch_document_layout(const int* ids, long long stride_b, int B, int S, int* layout, cudaStream_t stream);

// Work list of the paged attention (int32):
//   header     kWorkHeader words: 0: items, 1: CTAs that get a share
//   starts     where every CTA starts and, behind the last one, the end: 4 words (key/value head, item, key tile, 1 if it
//              starts inside an item of two query tiles) for each of the device's SMs and one more
//   items      kWorkItem words each: first row of the packed tensors, tokens, position of the first token, request, cost of
//              the items before it, key tiles of its own, cost of a key tile, 0
constexpr int kWorkHeader = 16;
constexpr int kWorkItem = 8;
// What the plan deals out in equal shares: the cost of a key tile of an item of one query tile and of two, and of the start and
// end of such an item. (From clock readings of every CTA, fitted: a key tile 2.1 and 2.9 thousand cycles at D = 64, 2.7 and
// 3.8 at D = 128, a start and end 5.3 and 5.9, 7.4 and 12.5; where memory is the bound, single tokens take less of both.)
constexpr int kTileCost1 = 2, kTileCost2 = 3, kItemCost1 = 4, kItemCost2 = 8;
inline int work_items_at(int sms) { return kWorkHeader + (4 * (sms + 1) + 7) / 8 * 8; }   // word of the first item

struct PagedPlanDev {
  const int *context_lens, *new_lens;
  int B;
  int* block_table;
  long long table_stride;
  int table_width;
  const int* free_pages;
  int n_free;
  const int* free_start;     // or null: 0
  int page_shift;
  int num_tokens;
  int item_tokens;           // query tokens per item of the work list
  int heads_kv, sms, items_at;
  int *cu_seqlens, *seqlens_k;
  long long* slot_map;
  int *positions, *pages_taken, *work;
};
cudaError_t launch_paged_plan(const PagedPlanDev& p, cudaStream_t stream);

struct PagedWriteDev {
  const uint16_t *k, *v;
  long long k_st, k_sh, v_st, v_sh;               // (token, head) element strides
  uint16_t *k_cache, *v_cache;
  long long kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh;   // (page, slot, head) element strides
  const long long* slot_map;
  long long slots;                                 // slots of the cache: pages << page_shift
  int tokens, heads, chunks_per_head;              // chunks of 8 elements
  int page_shift;
};
cudaError_t launch_paged_write(const PagedWriteDev& p, cudaStream_t stream);

struct PagedAttnDev {
  int T, Hq, Hkv, G;
  int tile_tokens;           // tokens of a 128-row tile: floor(128 / G)
  const int* work;
  int items_at;
  const int* block_table;
  long long table_stride;
  int table_width, page_shift, num_pages;
  int page_groups, page_heads;   // whole_rows: what a page adds to a box's fourth and fifth coordinate
  float scale_log2, cap2, arg2;
  const float* slopes;       // [Hq] or null
  uint16_t* out;
  long long out_st, out_sh;  // (token, head) element strides
  int blk;                   // real columns in each 64-column block
  float* lse;                // [T][Hq] natural log, or null
  float* part_o;             // [2 * CTAs][256][kernel head dim]
  float* part_lse;           // [2 * CTAs][256], log2
  int* status;
};
struct PagedAttnLaunch {
  CUtensorMap tmQ, tmK, tmV;
  PagedAttnDev p;
  int head_dim;              // 64 or 128
  bool whole_rows;           // (head dim 128) a box of K or V brings all columns of its keys
  bool bf16;
  int mod;                   // kModCap | kModSlope
};
cudaError_t launch_paged_attention(const PagedAttnLaunch& a, cudaStream_t stream);

}  // namespace fa2
