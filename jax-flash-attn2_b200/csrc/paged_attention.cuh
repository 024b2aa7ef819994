// Attention of new tokens over a paged key/value cache on sm_100a (head dims up to 128): chunks of prompts, single
// tokens and anything between in one launch.
//
//   out_t = softmax_j (score(q_t, k_j)) v_j over the keys j <= position(t) of t's request, found through its block table
//
// Rows. The G query heads that share a key/value head are rows of one tile, G consecutive rows per token, so that a key is
// read once per group: a 128-row tile holds floor(128 / G) tokens, an item (two tiles over one stream of keys, as in
// fwd_kernel.cuh) twice as many.
//
// Split. The plan deals the key tiles of all items of all key/value heads to the CTAs in one line, in equal shares whatever
// the lengths of the requests are (paged_plan.cu), and notes where each CTA starts. A CTA that has all key tiles of an item
// writes its rows; items cut by a border leave normalised partial rows and their log-sum-exp in
// float32 (at most two per CTA), which paged_combine_kernel joins in the order of the keys: the result does not depend on
// which CTA was faster.
//
// Few rows. An item whose tokens fit one query tile (every single token) is bound by the chain S -> softmax -> P V of a key
// tile, not by its work. It runs as two chains: the second warpgroup takes the odd key tiles of the same rows, with its own
// maximum, sum and accumulator, and the first one joins the two accumulators when it writes the rows, straight from tensor
// memory (the rows lie on the same lanes). 64 decodes over 128 .. 16384 keys (32/8 heads, D = 128): 161 us with one chain,
// 137 us with two (124 today); the cache alone is 646 MB, 98 us at the measured copy bandwidth.
//
// Keys. Pages hold 2^s tokens; a 128-key tile takes 128 / 2^s pieces of a page each (one if pages are larger), every piece
// one TMA box, issued by a lane of its own, or one per 64-column block where the cache's strides leave no dimension of a
// tensor map for the blocks (64 tokens over 9856 keys in pages of 16, 32/8 heads, D = 128: 414 us, 469 with a box per block, which
// is 2 KB; pages of 32 and more: no difference). Pages outside the request or the pool are fetched from
// an index behind the pool, which the TMA unit fills with zeros. Keys behind the last visible one in its page hold whatever
// was in memory: their scores are masked, and a spare warp zeroes their V rows, since 0 * NaN is NaN.
//
// Roles (12 warps): 0-3 and 4-7 softmax of the two query tiles, 8 MMA issue, 9 TMA, 10 clears V rows, 11 idle.
// Tensor memory: S0 128 | S1 128 | O0 D | O1 D columns, P over S, as in fwd_kernel.cuh.
#pragma once
#include "fwd_row.cuh"
#include "launch_util.cuh"
#include "lm_launch.cuh"
#include "ptx_sm100.cuh"
#include "score_mod.cuh"

namespace fa2 {

namespace {

constexpr int kPagedThreads = 384;
constexpr int kPagedRegsSoftmax = 208, kPagedRegsOther = 88;   // (2 * 208 + 88) / 3 = 168, the launch's share

template <int D>
struct PagedSmem {
  static constexpr int kQTileBytes = 128 * D * 2;
  static constexpr int kKVTileBytes = 128 * D * 2;
  static constexpr int kStages = D == 64 ? 10 : 5;
  static constexpr int kBlock = 128 * 128;             // one [128 rows][64 elements] block
  static constexpr int kQOff = 0;
  static constexpr int kKVOff = kQOff + 2 * kQTileBytes;
  static constexpr int kBarOff = kKVOff + kStages * kKVTileBytes;
  // q_full[2], q_free[2], kv_full[S], kv_empty[S], s_full[2], p_full[2][kPSplit], o_full[2], o_free[2], dirty, clean
  static constexpr int kNumBars = 4 + 2 * kStages + 2 + 2 * kPSplit + 4 + 2;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kStatOff = kMiscOff + 16;       // maximum and sum of the second chain's rows
  static constexpr int kNoteOff = kStatOff + 128 * 8;  // per softmax warp: see PagedNote
  static constexpr int kTotal = kNoteOff + 8 * 64;
  static constexpr int kDynamicBytes = kTotal + 1024;
  static_assert(kDynamicBytes <= 232448, "shared memory budget exceeded");
};

// A CTA's way from its start to the next CTA's. An item of two query tiles (part of a chunk, whose other items see the same
// keys) that it begins inside of comes last, so that the CTAs, which all begin with the first key tile of some item, walk over
// the keys of a long request side by side and share them in L2: 4096 new tokens of 64/8 heads, D = 128, over 65536 keys 8.55 ->
// 7.77 ms, over 32768 3.75 -> 3.67, over 8192 (which fit L2 either way) 0.678 -> 0.690. Single tokens share nothing, and are
// faster in the order of the line (64 over 2464 keys 135 us, 142 with the first piece last).
struct PagedWalk {
  int n_items;
  int hk, i, tile;
  int end_hk, end_i, end_tile;
  int late;                     // the stretch at the CTA's start is still to come
};

// One stretch of it: key tiles [ja, jb) of one item and head.
struct PagedSeg {
  int hk, row0, n_tok, pos0, req;
  int ja, jb, tiles;
  int seen;                     // keys the item's last token sees
  int n_t[2];                   // key tiles of this stretch that each warpgroup works on
  bool whole;                   // all key tiles of the item
  bool dual;                    // one query tile in two chains: warpgroup t takes the tiles ja + t, ja + t + 2, ...
};

// What a softmax warp needs between two stretches and at the end of one, but not in its loop over the key tiles, where the
// 128 scores of a row leave no registers for it: it stands in shared memory meanwhile. (Left to the compiler, some of the loop's
// own values were spilled: 4096 new tokens over 28k keys took 5.1 ms instead of 3.56 ms.)
struct PagedNote {
  PagedWalk w;
  int row0, hk;
  int slot;        // partial rows to write (2 * CTA or one more), or -1: the rows are complete
  int dual, other; // dual, and whether the second chain has an accumulator
};

__device__ __forceinline__ int4 paged_start_of(const int* work, int c) {
  return __ldg(reinterpret_cast<const int4*>(work + kWorkHeader) + c);
}

__device__ __forceinline__ void paged_advance(PagedWalk& w) {
  if (++w.i == w.n_items) {
    w.i = 0;
    ++w.hk;
  }
}

__device__ __forceinline__ void paged_start(const PagedAttnDev& p, PagedWalk& w) {
  w.n_items = __ldg(p.work);
  const int ctas = __ldg(p.work + 1), c = blockIdx.x;
  w.hk = w.i = w.tile = w.end_hk = w.end_i = w.end_tile = w.late = 0;
  if (c >= ctas) return;
  const int4 from = paged_start_of(p.work, c), to = paged_start_of(p.work, c + 1);
  w.hk = from.x; w.i = from.y; w.tile = from.z;
  w.end_hk = to.x; w.end_i = to.y; w.end_tile = to.z;
  if (from.w != 0 && w.tile > 0 && (w.hk != w.end_hk || w.i != w.end_i)) {
    w.late = 1;
    w.tile = 0;
    paged_advance(w);
  }
}

__device__ __forceinline__ bool paged_next(const PagedAttnDev& p, PagedWalk& w, PagedSeg& s) {
  bool in_last = w.hk == w.end_hk && w.i == w.end_i;
  int4 at = make_int4(w.hk, w.i, w.tile, 0);
  const bool done = in_last && w.tile >= w.end_tile;
  if (done) {
    if (!w.late) return false;
    w.late = 0;
    in_last = false;
    at = paged_start_of(p.work, blockIdx.x);
  }
  const int4* item = reinterpret_cast<const int4*>(p.work + p.items_at) + 2 * static_cast<long long>(at.y);
  const int4 a = __ldg(item);
  s.tiles = __ldg(&item[1].y);
  s.hk = at.x;
  s.row0 = a.x;
  s.n_tok = a.y;
  s.pos0 = a.z;
  s.req = a.w;
  s.ja = at.z;
  s.jb = in_last ? w.end_tile : s.tiles;
  s.seen = min(s.pos0 + s.n_tok, p.table_width << p.page_shift);
  s.whole = s.ja == 0 && s.jb == s.tiles;
  if (!done) {
    w.tile = s.jb;
    if (s.jb == s.tiles) {
      w.tile = 0;
      paged_advance(w);
    }
  }
  s.dual = s.n_tok <= p.tile_tokens;
  if (s.dual) {
    s.n_t[0] = (s.jb - s.ja + 1) >> 1;
    s.n_t[1] = (s.jb - s.ja) >> 1;
    return true;
  }
  const int n0 = p.tile_tokens;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int last = t == 0 ? n0 : s.n_tok;      // tokens up to the end of this query tile
    const int end = min(s.tiles, (s.pos0 + last + 127) >> 7);
    s.n_t[t] = max(0, min(end, s.jb) - s.ja);
  }
  return true;
}

}  // namespace

// kWhole: a box brings all columns of its keys.
template <int D, bool kBf16, int kMod, bool kWhole>
__global__ void __launch_bounds__(kPagedThreads, 1)
paged_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const PagedAttnDev p) {
  using L = PagedSmem<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t sQ = smem_base + L::kQOff, sKV = smem_base + L::kKVOff, bars = smem_base + L::kBarOff;
  auto bar_q_full = [&](int t) { return bars + 8u * t; };
  auto bar_q_free = [&](int t) { return bars + 8u * (2 + t); };
  auto bar_kv_full = [&](int s) { return bars + 8u * (4 + s); };
  auto bar_kv_empty = [&](int s) { return bars + 8u * (4 + L::kStages + s); };
  auto bar_s_full = [&](int t) { return bars + 8u * (4 + 2 * L::kStages + t); };
  auto bar_p_full = [&](int t, int hh) { return bars + 8u * (6 + 2 * L::kStages + kPSplit * t + hh); };
  auto bar_o_full = [&](int t) { return bars + 8u * (6 + 2 * L::kStages + 2 * kPSplit + t); };
  auto bar_o_free = [&](int t) { return bars + 8u * (8 + 2 * L::kStages + 2 * kPSplit + t); };
  // The MMA warp finds a V tile with rows to clear in its slot (dirty), a spare warp clears them (clean). The two take
  // turns, one tile at a time, so neither barrier can be a phase ahead of who waits for it.
  const uint32_t bar_dirty = bars + 8u * (10 + 2 * L::kStages + 2 * kPSplit), bar_clean = bar_dirty + 8u;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem_gen + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_gen + L::kMiscOff + 4);
  constexpr int kBlks = D / 64;
  // a K or V tile: groups of 8 keys, 1 KiB per column block; all groups of a block together, or (kWhole) all blocks of a group
  constexpr int group_stride = kWhole ? kBlks * 1024 : 1024, blk_stride = kWhole ? 1024 : L::kBlock;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 9 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  PagedWalk w;                 // (its loads are under way while the barriers are set up)
  paged_start(p, w);
  // (the combine kernel may be launched from here on; it waits for this kernel's end itself)
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    *abort_flag = 0;
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar_q_full(t), 1);
      mbar_init(bar_q_free(t), 1);
      mbar_init(bar_s_full(t), 1);
      for (int hh = 0; hh < kPSplit; ++hh) mbar_init(bar_p_full(t, hh), kBM);
      mbar_init(bar_o_full(t), 1);
      mbar_init(bar_o_free(t), kBM);
    }
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(bar_kv_full(s), 1);
      mbar_init(bar_kv_empty(s), 1);
    }
    mbar_init(bar_dirty, 1);
    mbar_init(bar_clean, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    __syncwarp();
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  constexpr uint32_t kColS = 0, kColO = 256;

  if (warp >= 8) setmaxnreg_dec<kPagedRegsOther>();
  if (warp == 11) {
    // idle
  } else if (warp == 10) {
    // =========================== clears V rows behind the last visible key ==================
    bool ok = true;
    uint32_t kv_count = 0, turn = 0;
    PagedSeg s;
    while (ok && paged_next(p, w, s)) {
      const int tail = s.seen & 127;
      kv_count += 2 * (s.jb - s.ja);
      if (s.jb != s.tiles || tail == 0) continue;
      const uint32_t last = kv_count - 1;                  // the stretch's last V tile
      const int slot = last % L::kStages;
      ok = mbar_wait_warp(bar_dirty, turn & 1u, abort_flag);
      ++turn;
      // (the tile has landed; waiting on its own barrier too orders the copy before the writes below)
      if (ok) ok = mbar_wait_warp(bar_kv_full(slot), (last / L::kStages) & 1u, abort_flag);
      if (!ok) break;
      // rows behind the end of the last page were filled with zeros by the TMA unit
      const int piece = min(128, 1 << p.page_shift);
      const int end = min(128, (tail + piece - 1) / piece * piece);
      uint8_t* v = smem_gen + L::kKVOff + slot * L::kKVTileBytes;
      for (int x = lane; x < (end - tail) * 8 * kBlks; x += 32) {
        const int blk = x / ((end - tail) * 8), y = x - blk * ((end - tail) * 8);
        const int row = tail + (y >> 3);
        *reinterpret_cast<uint4*>(v + blk * blk_stride + (row >> 3) * group_stride + (row & 7) * 128 + (y & 7) * 16) =
            make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_clean);
    }
    if (!ok && lane == 0) atomicOr(p.status, 512);
  } else if (warp == 9) {
    // =========================== TMA producer ================================================
    bool ok = true;
    uint32_t kv_count = 0, seg_idx = 0;
    PagedSeg s;
    const int piece_rows = min(128, 1 << p.page_shift), pieces = 128 / piece_rows;
    const int my_piece = lane % pieces, my_blk = lane / pieces;    // this lane's box of a K or V tile
    const bool issues = my_blk < (kWhole ? 1 : kBlks);
    const uint32_t box_dst = my_blk * L::kBlock + my_piece * piece_rows * (kWhole ? 128 * kBlks : 128);
    const int page_mask = (1 << p.page_shift) - 1;
    const uint32_t q_bytes = static_cast<uint32_t>(p.tile_tokens * p.G) * 128u * kBlks;
    for (; ok && paged_next(p, w, s); ++seg_idx) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ok = ok && mbar_wait_warp(bar_q_free(t), (seg_idx & 1u) ^ 1u, abort_flag);
        if (!ok) break;
        if (lane == 0 && t == 1 && s.dual) {
          mbar_arrive(bar_q_full(t));          // both chains read the first tile
        } else if (lane == 0) {
          mbar_arrive_expect_tx(bar_q_full(t), q_bytes);
#pragma unroll
          for (int blk = 0; blk < kBlks; ++blk)
            tma_load_5d(sQ + t * L::kQTileBytes + blk * L::kBlock, &tmQ, bar_q_full(t), 0, 0,
                        s.row0 + t * p.tile_tokens, blk, s.hk);
        }
      }
      // page of this lane's piece of key tile j: the pool's size (out of range, reads as zeros) where there is none
      const int* table = p.block_table + s.req * p.table_stride;
      auto page_of = [&](int j) {
        const int key = j * 128 + my_piece * piece_rows;
        int id = -1;
        if (issues && key < s.seen) id = __ldg(table + (key >> p.page_shift));
        return static_cast<unsigned>(id) < static_cast<unsigned>(p.num_pages) ? id : p.num_pages;
      };
      auto load = [&](const CUtensorMap* tm, int j, int page) {
        const int slot = kv_count % L::kStages;
        ok = ok && mbar_wait_warp(bar_kv_empty(slot), ((kv_count / L::kStages) & 1u) ^ 1u, abort_flag);
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(bar_kv_full(slot), L::kKVTileBytes);
        __syncwarp();
        const int place = (j * 128 + my_piece * piece_rows) & page_mask;
        if (kWhole && issues)
          tma_load_5d(sKV + slot * L::kKVTileBytes + box_dst, tm, bar_kv_full(slot), 0, 0, 0,
                      page * p.page_groups + (place >> 3), page * p.page_heads + s.hk);
        else if (issues)
          tma_load_5d(sKV + slot * L::kKVTileBytes + box_dst, tm, bar_kv_full(slot), 0, place, my_blk, s.hk, page);
        ++kv_count;
      };
      // in the order in which the MMA warp uses them (see there); pages are looked up two tiles ahead
      const int n = s.jb - s.ja, ahead = s.dual ? 2 : 1;
      int before2 = 0, before1 = 0, next = page_of(s.ja), after = n > 1 ? page_of(s.ja + 1) : 0;
      for (int j = -ahead; j < n && ok; ++j) {
        if (j >= 0) load(&tmV, s.ja + j, s.dual ? before2 : before1);
        if (j + ahead < n) load(&tmK, s.ja + j + ahead, next);
        before2 = before1;
        before1 = next;
        next = after;
        if (j + ahead + 2 < n) after = page_of(s.ja + j + ahead + 2);
      }
    }
    if (!ok && lane == 0) atomicOr(p.status, 1);
  } else if (warp == 8) {
    // =========================== MMA issuer ==================================================
    constexpr uint32_t idesc_s = make_idesc(kBf16, kBM, kBN, false, false);
    constexpr uint32_t idesc_o = make_idesc(kBf16, kBM, D, false, true);
    bool ok = true;
    const uint64_t dQ0 = make_sdesc(sQ, 16, 1024);
    const uint64_t dKV_k0 = make_sdesc(sKV, 16, group_stride);               // K tile, K-major
    const uint64_t dKV_mn0 = make_sdesc(sKV, blk_stride, group_stride);      // V tile, MN-major
    auto issue_s = [&](int t, int slot, int q_tile) {
      const uint64_t a0 = sdesc_advance(dQ0, q_tile * L::kQTileBytes);
      const uint64_t b0 = sdesc_advance(dKV_k0, slot * L::kKVTileBytes);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (k & 3) * 32;
        mma_ss_e(tmem_base + kColS + t * kBN, sdesc_advance(a0, (k >> 2) * L::kBlock + off),
                 sdesc_advance(b0, (k >> 2) * blk_stride + off), idesc_s, k > 0 ? 1u : 0u);
      }
      mma_commit_e(bar_s_full(t));
    };
    auto issue_o = [&](int t, int slot, bool first, int hh) {
      const uint64_t b0 = sdesc_advance(dKV_mn0, slot * L::kKVTileBytes);
#pragma unroll
      for (int k = hh * (kPCols / 16); k < (hh + 1) * (kPCols / 16); ++k)
        mma_ts_e(tmem_base + kColO + t * D, tmem_base + kColS + t * kBN + k * 8, sdesc_advance(b0, k * 2 * group_stride), idesc_o,
                 (first && k == 0) ? 0u : 1u);
    };
    uint32_t kv_count = 0, seg_idx = 0;
    uint32_t turn = 0;             // V tiles cleared so far
    uint32_t it_cnt[2] = {0, 0};
    PagedSeg s;
    for (; ok && paged_next(p, w, s); ++seg_idx) {
      const int n = s.jb - s.ja;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ok = ok && mbar_wait_warp(bar_q_full(t), seg_idx & 1u, abort_flag);
        if (ok && (s.n_t[t] == 0 || (s.dual && t == 1))) mma_commit_e(bar_q_free(t));
        if (ok && s.n_t[t] == 0) {       // a query tile without work keeps the hand-shakes in step
          ok = mbar_wait_warp(bar_o_free(t), (seg_idx & 1u) ^ 1u, abort_flag);
          if (ok) mma_commit_e(bar_o_full(t));
        }
      }
      if (!ok) break;
      // Step j: O_t += P_t V_j, then S_t = Q K of the key tile `ahead` further on, for every warpgroup t whose turn it is. Two
      // query tiles take every key tile each and look one tile ahead: while the softmax of one works, the MMAs of the other
      // run. One query tile in two chains: chain t takes the key tiles of its parity and looks two ahead.
      const int ahead = s.dual ? 2 : 1;
      for (int j = -ahead; j < n && ok; ++j) {
        const int jk = j + ahead;
        int slot_v = 0, slot_k = 0;
        if (j >= 0) {
          slot_v = kv_count % L::kStages;
          ok = mbar_wait_warp(bar_kv_full(slot_v), (kv_count / L::kStages) & 1u, abort_flag);
          ++kv_count;
          if (ok && j == n - 1 && s.jb == s.tiles && (s.seen & 127) != 0) {
            if (lane == 0) mbar_arrive(bar_dirty);
            __syncwarp();
            ok = mbar_wait_warp(bar_clean, turn & 1u, abort_flag);
            ++turn;
          }
        }
        if (ok && jk < n) {
          slot_k = kv_count % L::kStages;
          ok = mbar_wait_warp(bar_kv_full(slot_k), (kv_count / L::kStages) & 1u, abort_flag);
          ++kv_count;
        }
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bool mine = !s.dual || (j & 1) == t;
          const int last = s.dual ? n : s.n_t[t];            // key tiles this warpgroup works on end here
          const bool pv = mine && j >= 0 && j < last;
          if (pv) {
            if (j < ahead) ok = mbar_wait_warp(bar_o_free(t), (seg_idx & 1u) ^ 1u, abort_flag);   // O_t has been read out
#pragma unroll
            for (int hh = 0; hh < kPSplit; ++hh) {
              if (ok) ok = mbar_wait_warp(bar_p_full(t, hh), it_cnt[t] & 1u, abort_flag);
              if (!ok) break;
              tc_fence_after();
              issue_o(t, slot_v, j < ahead, hh);
            }
            if (!ok) break;
            ++it_cnt[t];
          }
          if (mine && jk < last) {
            issue_s(t, slot_k, s.dual ? 0 : t);
            if (s.dual ? jk == n - 1 : jk + 1 == last) mma_commit_e(bar_q_free(s.dual ? 0 : t));   // the last S of the Q tile
          }
          if (pv && jk >= last) mma_commit_e(bar_o_full(t));
        }
        if (!ok) break;
        if (j >= 0) mma_commit_e(bar_kv_empty(slot_v));
        if (jk < n) mma_commit_e(bar_kv_empty(slot_k));
      }
    }
    if (!ok && lane == 0) atomicOr(p.status, 2);
  } else {
    // =========================== softmax + epilogue ==========================================
    setmaxnreg_inc<kPagedRegsSoftmax>();
    const int t = warp >> 2, r = tid & (kBM - 1);
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem_base + lane_base + kColS + t * kBN;
    const uint32_t tO = tmem_base + lane_base + kColO + t * D;
    const float sc = ModTerms<kMod>::sc(p.scale_log2, p.cap2);
    static_assert(sizeof(PagedNote) <= 64, "the notes overlap");
    volatile PagedNote* note = reinterpret_cast<volatile PagedNote*>(smem_gen + L::kNoteOff + warp * 64);
    FwdKernelParams none;                              // softmax_tile_row reads nothing of it without score terms
    const KeepBitsDropout keep{false, make_uint4(0u, 0u, 0u, 0u)};
    uint32_t it_cnt = 0, o_cnt = 0;
    bool ok = true;
    if (lane == 0) {
      note->w.n_items = w.n_items;
      note->w.hk = w.hk; note->w.i = w.i; note->w.tile = w.tile;
      note->w.end_hk = w.end_hk; note->w.end_i = w.end_i; note->w.end_tile = w.end_tile;
      note->w.late = w.late;
    }
    __syncwarp();
    while (true) {
      int nt, row_lim, tile, tile_step, pos;
      float slope_h = 0.f;
      bool live;
      {
        w.n_items = note->w.n_items;
        w.hk = note->w.hk; w.i = note->w.i; w.tile = note->w.tile;
        w.end_hk = note->w.end_hk; w.end_i = note->w.end_i; w.end_tile = note->w.end_tile;
        w.late = note->w.late;
        PagedSeg s;
        if (!paged_next(p, w, s)) break;
        const int tok = r / p.G, head = r - tok * p.G;     // this row's token in the tile and head in the group
        const int tok0 = s.dual ? 0 : t * p.tile_tokens;   // first token of this query tile
        const int tokens = min(p.tile_tokens, max(0, s.n_tok - tok0));
        const bool valid = tok < tokens;
        live = 32 * (warp & 3) < tokens * p.G;             // some row of the warp is
        nt = s.n_t[t];
        tile = s.dual ? s.ja + t : s.ja;
        tile_step = s.dual ? 2 : 1;
        pos = s.pos0 + tok0 + tok;
        row_lim = valid ? min(pos, s.seen - 1) : -1;
        if (has_slope(kMod) && valid) slope_h = __ldg(p.slopes + s.hk * p.G + head);
        __syncwarp();
        if (lane == 0) {
          note->w.hk = w.hk; note->w.i = w.i; note->w.tile = w.tile;
          note->w.late = w.late;
          note->row0 = s.row0 + tok0;
          note->hk = s.hk;
          // the first stretch of a CTA that begins inside an item, the last one that ends inside one
          note->slot = s.whole ? -1 : 2 * static_cast<int>(blockIdx.x) + (s.ja > 0 ? 0 : 1);
          note->dual = s.dual;
          note->other = s.dual && s.n_t[1] > 0;
        }
        __syncwarp();
      }
      float m = -INFINITY, l = 0.f;
      const ModTerms<kMod> terms(p.scale_log2, p.arg2, p.cap2, slope_h, pos);
      for (int j = 0; j < nt && ok; ++j, ++it_cnt, tile += tile_step) {
        ok = mbar_wait(bar_s_full(t), it_cnt & 1u, abort_flag);
        if (!ok) break;
        if (live) {
          softmax_tile_row<D, kBf16, false, true>(tS, tO, tile, j > 0, none, row_lim, sc, false, m, l, [] {},
                                                  [&](int hh) { mbar_arrive(bar_p_full(t, hh)); }, terms, keep, 0);
        } else {
          // rows nobody asked for: whatever stands in their P only reaches rows of O that are not read
#pragma unroll
          for (int hh = 0; hh < kPSplit; ++hh) mbar_arrive(bar_p_full(t, hh));
        }
      }
      if (ok) ok = mbar_wait(bar_o_full(t), o_cnt & 1u, abort_flag);   // once per stretch, work or not
      ++o_cnt;
      tc_fence_after();
      float mine = 1.f, other = 0.f;       // factors of the two chains' accumulators
      const bool dual = note->dual != 0;
      if (dual) {
        // (a thread whose wait gave up meets the others here all the same)
        float2* stat = reinterpret_cast<float2*>(smem_gen + L::kStatOff);
        if (t == 1) stat[r] = make_float2(m, l);
        named_bar_sync(1, 256);
        if (t == 1) continue;              // the first warpgroup writes the rows and hands both accumulators back
        const float2 o = stat[r];
        const float top = fmaxf(m, o.x);
        if (top > -INFINITY) {
          mine = ex2_approx((m - top) * sc);
          other = ex2_approx((o.x - top) * sc);
        }
        m = top;
        l = l * mine + o.y * other;
      }
      const float inv = l > 0.f ? 1.f / l : 0.f;
      const float lse2 = l > 0.f ? m * sc + lg2_approx(l) : -INFINITY;
      const int tok = r / p.G, h = note->hk * p.G + (r - tok * p.G), slot = note->slot;
      const bool valid = row_lim >= 0, whole = slot < 0, join = note->other != 0;
      const long long token = note->row0 + tok;
      const long long prow = static_cast<long long>(slot) * 256 + t * kBM + r;
      if (ok && valid) {
        if (whole) {
          if (p.lse) p.lse[token * p.Hq + h] = lse2 * kLn2;
        } else {
          p.part_lse[prow] = lse2;
        }
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (nt > 0 && live) {
          tmem_ld32(tO + c * 32, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
        if (join && live) {
          uint32_t o1[32];
          tmem_ld32(tO + D + c * 32, o1);
          tc_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; ++k)
            o[k] = __float_as_uint(__uint_as_float(o[k]) * mine + __uint_as_float(o1[k]) * other);
        }
        if (c == D / 32 - 1) {
          tc_fence_before();
          mbar_arrive(bar_o_free(t));
          if (dual) mbar_arrive(bar_o_free(1));
        }
        if (ok && valid) {
          if (whole) {
            const int col = (c & 1) * 32;                       // column inside the 64-column block
            uint4* dst = reinterpret_cast<uint4*>(p.out + token * p.out_st + h * p.out_sh + (c >> 1) * p.blk + col);
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
              if (col + 8 * q4 < p.blk) {
                uint4 v;
                v.x = pack2<kBf16>(__uint_as_float(o[8 * q4 + 0]) * inv, __uint_as_float(o[8 * q4 + 1]) * inv);
                v.y = pack2<kBf16>(__uint_as_float(o[8 * q4 + 2]) * inv, __uint_as_float(o[8 * q4 + 3]) * inv);
                v.z = pack2<kBf16>(__uint_as_float(o[8 * q4 + 4]) * inv, __uint_as_float(o[8 * q4 + 5]) * inv);
                v.w = pack2<kBf16>(__uint_as_float(o[8 * q4 + 6]) * inv, __uint_as_float(o[8 * q4 + 7]) * inv);
                dst[q4] = v;
              }
          } else {
            store_partial_row(p.part_o + prow * D + c * 32, o, inv);
          }
        }
      }
    }
    if (!ok && r == 0) atomicOr(p.status, 4);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Which of the CTAs base .. base + 31 have a part of the item that is cut first at the start of CTA c and reaches to CTA `last`:
// one without a tile of its own (its start is the next one's) has none, the first one, c - 1, always has.
__device__ __forceinline__ unsigned paged_parts(const PagedAttnDev& p, int base, int c, int last, int lane) {
  bool here = base + lane <= last;
  if (here && base + lane >= c) {
    const int4 from = paged_start_of(p.work, base + lane), to = paged_start_of(p.work, base + lane + 1);
    here = from.x != to.x || from.y != to.y || from.z != to.z;
  }
  return __ballot_sync(0xffffffffu, here);
}

// kRows rows of an item at a time, x0, x0 + stride, ...; the parts of CTAs c - 1 .. last that there are (32 CTAs at a time, the
// first ones known already), kParts of them with their loads under way at once: a part's row comes from L2, and one after
// the other they would cost its latency each.
template <int D, bool kBf16, int kRows, int kParts>
__device__ __forceinline__ void paged_join_rows(const PagedAttnDev& p, int hk, int row0, int rows, int x0, int stride, int c,
                                                int last, unsigned first_parts, int lane) {
  constexpr int kVec = D / 32;
  const int row_tile = p.tile_tokens * p.G;
  int row[kRows];                   // inside a part
  float m[kRows], acc[kRows][kVec], sum[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int x = min(x0 + k * stride, rows - 1);        // a row too many is computed again and not written
    row[k] = x < row_tile ? x : kBM + x - row_tile;
    m[k] = -INFINITY;
    sum[k] = 0.f;
#pragma unroll
    for (int e = 0; e < kVec; ++e) acc[k][e] = 0.f;
  }
  for (int base = c - 1; base <= last; base += 32) {
    unsigned parts = base == c - 1 ? first_parts : paged_parts(p, base, c, last, lane);
    while (parts) {
      float lse[kParts][kRows], v[kParts][kRows][kVec];
#pragma unroll
      for (int q = 0; q < kParts; ++q) {
        const bool any = parts != 0;
        const int cc = any ? base + __ffs(parts) - 1 : c - 1;
        if (any) parts &= parts - 1;
        // part c - 1 is its CTA's last stretch, the others are first ones
        const long long slot = (cc == c - 1 ? 2LL * cc + 1 : 2LL * cc) * 256;
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          lse[q][k] = any ? __ldcg(p.part_lse + slot + row[k]) : -INFINITY;
          const float* src = p.part_o + (slot + row[k]) * D + lane * kVec;
          if constexpr (kVec == 4) {
            const float4 f = __ldcg(reinterpret_cast<const float4*>(src));
            v[q][k][0] = f.x; v[q][k][1] = f.y; v[q][k][2] = f.z; v[q][k][3] = f.w;
          } else {
            const float2 f = __ldcg(reinterpret_cast<const float2*>(src));
            v[q][k][0] = f.x; v[q][k][1] = f.y;
          }
        }
      }
#pragma unroll
      for (int q = 0; q < kParts; ++q) {
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
          if (lse[q][k] == -INFINITY) continue;       // no part, or the row sees none of its keys
          const float top = fmaxf(m[k], lse[q][k]);
          const float keep = ex2_approx(m[k] - top), wgt = ex2_approx(lse[q][k] - top);
          m[k] = top;
          sum[k] = sum[k] * keep + wgt;
#pragma unroll
          for (int e = 0; e < kVec; ++e) acc[k][e] = fmaf(acc[k][e], keep, wgt * v[q][k][e]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const int x = x0 + k * stride;
    if (x >= rows) break;
    const int tok = x / p.G, h = hk * p.G + (x - tok * p.G);
    const float inv = sum[k] > 0.f ? 1.f / sum[k] : 0.f;
    const long long token = row0 + tok;
    if (p.lse && lane == 0) p.lse[token * p.Hq + h] = sum[k] > 0.f ? (m[k] + lg2_approx(sum[k])) * kLn2 : -INFINITY;
    const int col = lane * kVec, in = col & 63;
    if (in < p.blk) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + token * p.out_st + h * p.out_sh + (col >> 6) * p.blk + in);
#pragma unroll
      for (int e = 0; e < kVec; e += 2) dst[e >> 1] = pack2<kBf16>(acc[k][e] * inv, acc[k][e + 1] * inv);
    }
  }
}

// Joins the partial rows of an item cut by CTA borders: with the parts' log2 sums L_c,
//   out = sum_c 2^(L_c - L) o_c,   L = log2 sum_c 2^L_c,
// in the order of the keys. Block (c, y) looks at the start of CTA c + 1 and works iff that is the first border inside its
// item; rows are dealt over the y blocks and their warps. Each partial row is read once. It is launched while the main
// kernel still runs (programmatic dependent launch) and waits for its results only after it has found its item.
template <int D, bool kBf16>
__global__ void __launch_bounds__(256)
paged_combine_kernel(const PagedAttnDev p) {
  const int ctas = __ldg(p.work + 1), c = blockIdx.x + 1, lane = threadIdx.x & 31;
  int last = c;                       // last CTA with a part of the item
  bool first_inside = false;
  int4 a = make_int4(0, 0, 0, 0), at = a;
  if (c < ctas) {
    at = paged_start_of(p.work, c);
    const int4 before = paged_start_of(p.work, c - 1);
    first_inside = at.z > 0 && !(before.x == at.x && before.y == at.y && before.z > 0);
    if (first_inside) {
      a = __ldg(reinterpret_cast<const int4*>(p.work + p.items_at) + 2 * static_cast<long long>(at.y));
      while (true) {
        const int cc = last + 1 + lane;
        bool same = false;
        if (cc < ctas) {
          const int4 x = paged_start_of(p.work, cc);
          same = x.x == at.x && x.y == at.y;
        }
        const unsigned votes = __ballot_sync(0xffffffffu, same);
        const int n = votes == 0xffffffffu ? 32 : __ffs(~votes) - 1;
        last += n;
        if (n < 32) break;
      }
    }
  }
  const unsigned parts = first_inside ? paged_parts(p, c - 1, c, last, lane) : 0u;
  // (every block waits, so that this kernel never ends before the main one)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!first_inside) return;
  const int rows = a.y * p.G, stride = 8 * gridDim.y;
  int x = (threadIdx.x >> 5) + 8 * blockIdx.y;
  if (rows <= stride) {
    if (x < rows) paged_join_rows<D, kBf16, 1, 8>(p, at.x, a.x, rows, x, stride, c, last, parts, lane);
  } else {
    for (; x < rows; x += 4 * stride) paged_join_rows<D, kBf16, 4, 2>(p, at.x, a.x, rows, x, stride, c, last, parts, lane);
  }
}

template <int D, bool kBf16, int kMod, bool kWhole>
static cudaError_t launch_paged_one(const PagedAttnLaunch& a, cudaStream_t stream) {
  using L = PagedSmem<D>;
  auto kern = paged_attention_kernel<D, kBf16, kMod, kWhole>;
  static bool smem_opted_in[64] = {};
  cudaError_t e = opt_in_dynamic_smem(kern, L::kDynamicBytes, smem_opted_in);
  if (e != cudaSuccess) return e;
  const int grid = sm_count();
  kern<<<grid, kPagedThreads, L::kDynamicBytes, stream>>>(a.tmQ, a.tmK, a.tmV, a.p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (grid < 2) return cudaSuccess;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid - 1, 4);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_combine_kernel<D, kBf16>, a.p);
}

template <int D, bool kWhole>
static cudaError_t launch_paged_dim(const PagedAttnLaunch& a, cudaStream_t stream) {
  switch ((a.bf16 ? 4 : 0) | a.mod) {
    case 0: return launch_paged_one<D, false, 0, kWhole>(a, stream);
    case 1: return launch_paged_one<D, false, 1, kWhole>(a, stream);
    case 2: return launch_paged_one<D, false, 2, kWhole>(a, stream);
    case 3: return launch_paged_one<D, false, 3, kWhole>(a, stream);
    case 4: return launch_paged_one<D, true, 0, kWhole>(a, stream);
    case 5: return launch_paged_one<D, true, 1, kWhole>(a, stream);
    case 6: return launch_paged_one<D, true, 2, kWhole>(a, stream);
    default: return launch_paged_one<D, true, 3, kWhole>(a, stream);
  }
}

}  // namespace fa2
