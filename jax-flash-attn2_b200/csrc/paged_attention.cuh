// Attention of new tokens over a paged key/value cache on sm_100a (head dims up to 128): chunks of prompts, single
// tokens and anything between in one launch.
//
//   out_t = softmax_j (score(q_t, k_j)) v_j over the keys j <= position(t) of t's request, found through its block table
//
// Rows. The G query heads that share a key/value head are rows of one tile, G consecutive rows per token, so that a key is
// read once per group: a 128-row tile holds floor(128 / G) tokens, an item (two tiles over one stream of keys, as in
// fwd_kernel.cuh) twice as many.
//
// Split. The key tiles of all items of all key/value heads are numbered through, W in all, and CTA c works on the tiles
// [c W / n, (c + 1) W / n): every SM streams the same number of tiles whatever the lengths of the requests are. A CTA that
// has all key tiles of an item writes its rows; items cut by a border leave normalised partial rows and their log-sum-exp in
// float32 (at most two per CTA), which paged_combine_kernel joins in the order of the keys: the result does not depend on
// which CTA was faster.
//
// Keys. Pages hold 2^s tokens; a 128-key tile takes 128 / 2^s pieces of a page each (one if pages are larger), every piece
// and 64-column block one TMA box, issued by a lane of its own. Pages outside the request or the pool are fetched from
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
  static constexpr int kStages = D == 64 ? 8 : 4;
  static constexpr int kBlock = 128 * 128;             // one [128 rows][64 elements] block
  static constexpr int kQOff = 0;
  static constexpr int kKVOff = kQOff + 2 * kQTileBytes;
  static constexpr int kBarOff = kKVOff + kStages * kKVTileBytes;
  // q_full[2], q_free[2], kv_full[S], kv_empty[S], s_full[2], p_full[2][kPSplit], o_full[2], o_free[2], dirty, clean
  static constexpr int kNumBars = 4 + 2 * kStages + 2 + 2 * kPSplit + 4 + 2;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kTotal = kMiscOff + 16;
  static constexpr int kDynamicBytes = kTotal + 1024;
  static_assert(kDynamicBytes <= 232448, "shared memory budget exceeded");
};

// A CTA's way through its share of the numbered key tiles.
struct PagedWalk {
  int n_items, per_head;        // items; key tiles of all items for one key/value head
  long long g, g_end;           // numbered tiles left: [g, g_end)
  int hk, i, rem;               // where g lies: head, item, tile among per_head
};

// One stretch of it: key tiles [ja, jb) of one item and head.
struct PagedSeg {
  int hk, row0, n_tok, pos0, req;
  int ja, jb, tiles;
  int seen;                     // keys the item's last token sees
  int n_t[2];                   // key tiles of this stretch that each query tile works on
  bool whole;                   // all key tiles of the item
};

__device__ __forceinline__ int paged_ctas(long long total, int grid) {
  return static_cast<int>(total < grid ? total : grid);
}
__device__ __forceinline__ long long paged_border(long long total, int ctas, int c) { return total * c / ctas; }

// Item with the largest prefix not above `rem`.
__device__ __forceinline__ int paged_find(const int* work, int n_items, int rem) {
  const int* prefix = work + kWorkHeader + 4;
  int lo = 0, hi = n_items;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(prefix + static_cast<long long>(mid) * kWorkItem) <= rem) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void paged_start(const PagedAttnDev& p, PagedWalk& w) {
  w.n_items = __ldg(p.work);
  w.per_head = __ldg(p.work + 1);
  const long long total = static_cast<long long>(w.per_head) * p.Hkv;
  const int ctas = paged_ctas(total, gridDim.x), c = blockIdx.x;
  w.g = w.g_end = 0;
  if (c >= ctas) return;
  w.g = paged_border(total, ctas, c);
  w.g_end = paged_border(total, ctas, c + 1);
  w.hk = static_cast<int>(w.g / w.per_head);
  w.rem = static_cast<int>(w.g - static_cast<long long>(w.hk) * w.per_head);
  w.i = paged_find(p.work, w.n_items, w.rem);
}

__device__ __forceinline__ bool paged_next(const PagedAttnDev& p, PagedWalk& w, PagedSeg& s) {
  if (w.g >= w.g_end) return false;
  const int4* item = reinterpret_cast<const int4*>(p.work + kWorkHeader) + 2 * static_cast<long long>(w.i);
  const int4 a = __ldg(item), b = __ldg(item + 1);
  s.hk = w.hk;
  s.row0 = a.x;
  s.n_tok = a.y;
  s.pos0 = a.z;
  s.req = a.w;
  s.tiles = b.y;
  s.ja = w.rem - b.x;
  s.jb = static_cast<int>(min(static_cast<long long>(s.tiles), s.ja + (w.g_end - w.g)));
  s.seen = min(s.pos0 + s.n_tok, p.table_width << p.page_shift);
  s.whole = s.ja == 0 && s.jb == s.tiles;
  const int n0 = min(s.n_tok, p.tile_tokens);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int last = t == 0 ? n0 : s.n_tok;      // tokens up to the end of this query tile
    const int end = t == 0 || s.n_tok > n0 ? min(s.tiles, (s.pos0 + last + 127) >> 7) : 0;
    s.n_t[t] = max(0, min(end, s.jb) - s.ja);
  }
  const int n = s.jb - s.ja;
  w.g += n;
  w.rem += n;
  if (s.jb == s.tiles && ++w.i == w.n_items) {
    w.i = 0;
    w.rem = 0;
    ++w.hk;
  }
  return true;
}

}  // namespace

template <int D, bool kBf16, int kMod>
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

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

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
  if (warp == 9 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
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
    PagedWalk w;
    PagedSeg s;
    paged_start(p, w);
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
        *reinterpret_cast<uint4*>(v + blk * L::kBlock + tail * 128 + y * 16) = make_uint4(0u, 0u, 0u, 0u);
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
    PagedWalk w;
    PagedSeg s;
    paged_start(p, w);
    const int piece_rows = min(128, 1 << p.page_shift), pieces = 128 / piece_rows;
    const int my_piece = lane % pieces, my_blk = lane / pieces;    // this lane's box of a K or V tile
    const bool issues = my_blk < kBlks;
    const uint32_t box_dst = my_blk * L::kBlock + my_piece * piece_rows * 128;
    const int page_mask = (1 << p.page_shift) - 1;
    const uint32_t q_bytes = static_cast<uint32_t>(p.tile_tokens * p.G) * 128u * kBlks;
    for (; ok && paged_next(p, w, s); ++seg_idx) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ok = ok && mbar_wait_warp(bar_q_free(t), (seg_idx & 1u) ^ 1u, abort_flag);
        if (!ok) break;
        if (lane == 0) {
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
      int next_page = page_of(s.ja);
      for (int j = s.ja; j < s.jb && ok; ++j) {
        const int page = next_page;
        if (j + 1 < s.jb) next_page = page_of(j + 1);
        const int row = (j * 128 + my_piece * piece_rows) & page_mask;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++kv_count) {
          const int slot = kv_count % L::kStages;
          ok = mbar_wait_warp(bar_kv_empty(slot), ((kv_count / L::kStages) & 1u) ^ 1u, abort_flag);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(bar_kv_full(slot), L::kKVTileBytes);
          __syncwarp();
          if (issues)
            tma_load_5d(sKV + slot * L::kKVTileBytes + box_dst, kv ? &tmV : &tmK, bar_kv_full(slot), 0, row, my_blk, s.hk,
                        page);
        }
      }
    }
    if (!ok && lane == 0) atomicOr(p.status, 1);
  } else if (warp == 8) {
    // =========================== MMA issuer ==================================================
    constexpr uint32_t idesc_s = make_idesc(kBf16, kBM, kBN, false, false);
    constexpr uint32_t idesc_o = make_idesc(kBf16, kBM, D, false, true);
    bool ok = true;
    const uint64_t dQ0 = make_sdesc(sQ, 16, 1024);
    const uint64_t dKV_k0 = make_sdesc(sKV, 16, 1024);               // K tile, K-major
    const uint64_t dKV_mn0 = make_sdesc(sKV, L::kBlock, 1024);       // V tile, MN-major
    auto issue_s = [&](int t, int slot) {
      const uint64_t a0 = sdesc_advance(dQ0, t * L::kQTileBytes);
      const uint64_t b0 = sdesc_advance(dKV_k0, slot * L::kKVTileBytes);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (k >> 2) * L::kBlock + (k & 3) * 32;
        mma_ss_e(tmem_base + kColS + t * kBN, sdesc_advance(a0, off), sdesc_advance(b0, off), idesc_s, k > 0 ? 1u : 0u);
      }
      mma_commit_e(bar_s_full(t));
    };
    auto issue_o = [&](int t, int slot, bool first, int hh) {
      const uint64_t b0 = sdesc_advance(dKV_mn0, slot * L::kKVTileBytes);
#pragma unroll
      for (int k = hh * (kPCols / 16); k < (hh + 1) * (kPCols / 16); ++k)
        mma_ts_e(tmem_base + kColO + t * D, tmem_base + kColS + t * kBN + k * 8, sdesc_advance(b0, k * 2048), idesc_o,
                 (first && k == 0) ? 0u : 1u);
    };
    uint32_t kv_count = 0, seg_idx = 0;
    uint32_t turn = 0;             // V tiles cleared so far
    uint32_t it_cnt[2] = {0, 0};
    PagedWalk w;
    PagedSeg s;
    paged_start(p, w);
    for (; ok && paged_next(p, w, s); ++seg_idx) {
      const int n = s.jb - s.ja;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ok = ok && mbar_wait_warp(bar_q_full(t), seg_idx & 1u, abort_flag);
        if (ok && s.n_t[t] == 0) {       // a query tile without work keeps the hand-shakes in step
          mma_commit_e(bar_q_free(t));
          ok = mbar_wait_warp(bar_o_free(t), (seg_idx & 1u) ^ 1u, abort_flag);
          if (ok) mma_commit_e(bar_o_full(t));
        }
      }
      if (!ok) break;
      {
        const int slot = kv_count % L::kStages;
        ok = mbar_wait_warp(bar_kv_full(slot), (kv_count / L::kStages) & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (s.n_t[t] > 0) {
            issue_s(t, slot);
            if (s.n_t[t] == 1) mma_commit_e(bar_q_free(t));   // that was the last S of tile t
          }
        }
        mma_commit_e(bar_kv_empty(slot));
        ++kv_count;
      }
      for (int j = 0; j < n && ok; ++j) {
        const bool has_next = j + 1 < n;
        const int slot_v = kv_count % L::kStages, slot_k = (kv_count + 1) % L::kStages;
        ok = mbar_wait_warp(bar_kv_full(slot_v), (kv_count / L::kStages) & 1u, abort_flag);
        if (ok && has_next) ok = mbar_wait_warp(bar_kv_full(slot_k), ((kv_count + 1) / L::kStages) & 1u, abort_flag);
        if (ok && !has_next && s.jb == s.tiles && (s.seen & 127) != 0) {
          if (lane == 0) mbar_arrive(bar_dirty);
          __syncwarp();
          ok = mbar_wait_warp(bar_clean, turn & 1u, abort_flag);
          ++turn;
        }
        if (!ok) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (j < s.n_t[t]) {
            if (j == 0) {      // the epilogue of the previous stretch has read O_t out of tensor memory
              ok = mbar_wait_warp(bar_o_free(t), (seg_idx & 1u) ^ 1u, abort_flag);
              if (!ok) break;
            }
#pragma unroll
            for (int hh = 0; hh < kPSplit; ++hh) {
              ok = mbar_wait_warp(bar_p_full(t, hh), it_cnt[t] & 1u, abort_flag);
              if (!ok) break;
              tc_fence_after();
              issue_o(t, slot_v, j == 0, hh);
            }
            if (!ok) break;
            ++it_cnt[t];
            if (j + 1 < s.n_t[t]) {
              issue_s(t, slot_k);
              if (j + 2 == s.n_t[t]) mma_commit_e(bar_q_free(t));   // last S of tile t issued
            } else {
              mma_commit_e(bar_o_full(t));
            }
          }
        }
        if (!ok) break;
        mma_commit_e(bar_kv_empty(slot_v));
        if (has_next) mma_commit_e(bar_kv_empty(slot_k));
        kv_count += has_next ? 2 : 1;
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
    const int tok = r / p.G, head = r - tok * p.G;     // this row's token in the tile and head in the group
    FwdKernelParams none;                              // softmax_tile_row reads nothing of it without score terms
    const KeepBitsDropout keep{false, make_uint4(0u, 0u, 0u, 0u)};
    uint32_t it_cnt = 0, o_cnt = 0;
    bool ok = true;
    PagedWalk w;
    PagedSeg s;
    paged_start(p, w);
    while (paged_next(p, w, s)) {
      const int nt = s.n_t[t];
      const int tokens = min(p.tile_tokens, max(0, s.n_tok - t * p.tile_tokens));   // of this query tile
      const bool valid = tok < tokens;
      const bool live = 32 * (warp & 3) < tokens * p.G;    // some row of the warp is
      const int pos = s.pos0 + t * p.tile_tokens + tok;
      const int row_lim = valid ? min(pos, s.seen - 1) : -1;
      const int h = s.hk * p.G + head;
      float m = -INFINITY, l = 0.f;
      const ModTerms<kMod> terms(p.scale_log2, p.arg2, p.cap2, has_slope(kMod) && valid ? __ldg(p.slopes + h) : 0.f, pos);
      for (int j = 0; j < nt && ok; ++j, ++it_cnt) {
        ok = mbar_wait(bar_s_full(t), it_cnt & 1u, abort_flag);
        if (!ok) break;
        if (live) {
          softmax_tile_row<D, kBf16, false, true>(tS, tO, s.ja + j, j > 0, none, row_lim, sc, false, m, l, [] {},
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
      const float inv = l > 0.f ? 1.f / l : 0.f;
      const float lse2 = l > 0.f ? m * sc + lg2_approx(l) : -INFINITY;
      const long long token = s.row0 + t * p.tile_tokens + tok;
      // partial results: the first stretch of a CTA that begins inside an item, the last one that ends inside one
      const long long prow = (2LL * blockIdx.x + (s.ja > 0 ? 0 : 1)) * 256 + t * kBM + r;
      if (ok && valid) {
        if (s.whole) {
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
        if (c == D / 32 - 1) {
          tc_fence_before();
          mbar_arrive(bar_o_free(t));
        }
        if (ok && valid) {
          if (s.whole) {
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

// Joins the partial rows of an item cut by CTA borders: with the parts' log2 sums L_c,
//   out = sum_c 2^(L_c - L) o_c,   L = log2 sum_c 2^L_c,
// in the order of the keys. Block (c, y) looks at the border between CTA c and c + 1 and works iff that border is the first
// inside its item; one warp per row, rows dealt over the y blocks. Reads each partial row once.
template <int D, bool kBf16>
__global__ void __launch_bounds__(256)
paged_combine_kernel(const PagedAttnDev p, int main_grid) {
  const int n_items = __ldg(p.work), per_head = __ldg(p.work + 1);
  const long long total = static_cast<long long>(per_head) * p.Hkv;
  const int ctas = paged_ctas(total, main_grid);
  const int c = blockIdx.x + 1;
  if (c >= ctas) return;
  const long long g = paged_border(total, ctas, c);
  const int hk = static_cast<int>(g / per_head);
  const int rem = static_cast<int>(g - static_cast<long long>(hk) * per_head);
  const int i = paged_find(p.work, n_items, rem);
  const int4* item = reinterpret_cast<const int4*>(p.work + kWorkHeader) + 2 * static_cast<long long>(i);
  const int4 a = __ldg(item), b = __ldg(item + 1);
  const long long begin = static_cast<long long>(hk) * per_head + b.x, end = begin + b.y;
  if (g == begin || paged_border(total, ctas, c - 1) > begin) return;
  int last = c;      // last CTA with a part of the item
  while (last + 1 < ctas && paged_border(total, ctas, last + 1) < end) ++last;

  const int lane = threadIdx.x & 31;
  const int rows = a.y * p.G;
  constexpr int kVec = D / 32;
  for (int x = (threadIdx.x >> 5) * gridDim.y + blockIdx.y; x < rows; x += 8 * gridDim.y) {
    const int tok = x / p.G, h = hk * p.G + (x - tok * p.G);
    const int t = tok >= p.tile_tokens ? 1 : 0;
    const int r = t * kBM + x - t * p.tile_tokens * p.G;     // row inside the parts
    auto row_of = [&](int cc) { return (cc == c - 1 ? 2LL * cc + 1 : 2LL * cc) * 256 + r; };
    float m = -INFINITY;
    for (int cc = c - 1 + lane; cc <= last; cc += 32) m = fmaxf(m, __ldg(p.part_lse + row_of(cc)));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    float acc[kVec], sum = 0.f;
#pragma unroll
    for (int k = 0; k < kVec; ++k) acc[k] = 0.f;
    if (m > -INFINITY) {
#pragma unroll 4
      for (int cc = c - 1; cc <= last; ++cc) {
        const float wgt = ex2_approx(__ldg(p.part_lse + row_of(cc)) - m);
        const float* src = p.part_o + row_of(cc) * D + lane * kVec;
        sum += wgt;
        if constexpr (kVec == 4) {
          const float4 v = __ldg(reinterpret_cast<const float4*>(src));
          acc[0] = fmaf(wgt, v.x, acc[0]);
          acc[1] = fmaf(wgt, v.y, acc[1]);
          acc[2] = fmaf(wgt, v.z, acc[2]);
          acc[3] = fmaf(wgt, v.w, acc[3]);
        } else {
          const float2 v = __ldg(reinterpret_cast<const float2*>(src));
          acc[0] = fmaf(wgt, v.x, acc[0]);
          acc[1] = fmaf(wgt, v.y, acc[1]);
        }
      }
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const long long token = a.x + tok;
    if (p.lse && lane == 0) p.lse[token * p.Hq + h] = sum > 0.f ? (m + lg2_approx(sum)) * kLn2 : -INFINITY;
    const int col = lane * kVec, in = col & 63;
    if (in < p.blk) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + token * p.out_st + h * p.out_sh + (col >> 6) * p.blk + in);
#pragma unroll
      for (int k = 0; k < kVec; k += 2) dst[k >> 1] = pack2<kBf16>(acc[k] * inv, acc[k + 1] * inv);
    }
  }
}

template <int D, bool kBf16, int kMod>
static cudaError_t launch_paged_one(const PagedAttnLaunch& a, cudaStream_t stream) {
  using L = PagedSmem<D>;
  auto kern = paged_attention_kernel<D, kBf16, kMod>;
  static bool smem_opted_in[64] = {};
  cudaError_t e = opt_in_dynamic_smem(kern, L::kDynamicBytes, smem_opted_in);
  if (e != cudaSuccess) return e;
  const int grid = sm_count();
  kern<<<grid, kPagedThreads, L::kDynamicBytes, stream>>>(a.tmQ, a.tmK, a.tmV, a.p);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (grid > 1) paged_combine_kernel<D, kBf16><<<dim3(grid - 1, 4), 256, 0, stream>>>(a.p, grid);
  return cudaGetLastError();
}

template <int D>
static cudaError_t launch_paged_dim(const PagedAttnLaunch& a, cudaStream_t stream) {
  switch ((a.bf16 ? 4 : 0) | a.mod) {
    case 0: return launch_paged_one<D, false, 0>(a, stream);
    case 1: return launch_paged_one<D, false, 1>(a, stream);
    case 2: return launch_paged_one<D, false, 2>(a, stream);
    case 3: return launch_paged_one<D, false, 3>(a, stream);
    case 4: return launch_paged_one<D, true, 0>(a, stream);
    case 5: return launch_paged_one<D, true, 1>(a, stream);
    case 6: return launch_paged_one<D, true, 2>(a, stream);
    default: return launch_paged_one<D, true, 3>(a, stream);
  }
}

}  // namespace fa2
