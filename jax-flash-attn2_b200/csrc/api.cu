// C ABI of the library: argument validation, tensor-map construction, kernel dispatch.
// Host half of the reference's launchers _fwd_attention_kernel_call
// (jax_flash_attn2/flash_attention_triton/_forward_triton.py:462-592) and
// _bwd_attention_kernel_call (_backward_triton.py:948-1173); the shape and broadcast rules
// follow calc_bias_strides (flash_attention_triton/_utils.py:151-193).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "../../include/fa2_b200.h"
#include "../../include/fa2_b200_debug.h"
#include "../../include/fa2_b200_lm.h"
#include "bwd_launch.cuh"
#include "fwd_launch.cuh"
#include "launch_util.cuh"
#include "lm_launch.cuh"
#include "score_mod.cuh"

namespace fa2 {
namespace {

thread_local char g_err[512] = "";
thread_local cudaEvent_t g_bwd_events[4] = {nullptr, nullptr, nullptr, nullptr};

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

__device__ int g_status_word;   // set by kernels whose bounded wait ran out

int* status_ptr() {
  // Looked up per call: the address differs per device and the caller chooses the device.
  int* p = nullptr;
  if (cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_status_word) != cudaSuccess) return nullptr;
  return p;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn get_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(sym);
  });
  return fn;
}

// The kernels exist for head dims 64, 128 and 256 (1, 2 and 4 blocks of 64 columns). Any other
// head dim is cut into the same number of equal blocks of D / nblk columns, each padded with zeros
// to 64: the tensor maps below give the first dimension the extent D / nblk while the box stays 64
// wide, so the TMA unit zero-fills the padding on loads and clips it on stores. Every operand is
// cut the same way, so the dot products over the head dim are unchanged, and outputs leave through
// the same kind of map, which puts their columns back in place. The block stride must be a multiple
// of 16 bytes, hence D % 8 == 0 up to 64, D % 16 == 0 up to 128, D % 32 == 0 up to 256.
struct HeadDim {
  int padded;   // 64, 128 or 256: selects the kernel
  int nblk;     // padded / 64
  int blk;      // real columns per block (64 when the head dim is one the kernels are built for)
};
bool split_head_dim(int D, HeadDim* hd) {
  if (D <= 0 || D > 256) return false;
  hd->padded = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  hd->nblk = hd->padded / 64;
  if (D % (8 * hd->nblk) != 0) return false;
  hd->blk = D / hd->nblk;
  return true;
}

// Tensor map of a [B, S, H, D] operand (any strides, unit head-dim stride) viewed as the 5-D
// tensor (D/nblk, S, nblk, H, B); one box is (64, rows, nblk, 1, 1) and lands in shared memory as
// nblk consecutive [rows][64] blocks with the 128-byte swizzle the MMA descriptors expect.
int make_tmap(CUtensorMap* tm, const void* ptr, bool bf16, int B, int S, int H, const HeadDim& hd,
              const fa2_strides& st, int box_rows, const char* what, int box_dblocks = 0) {
  if (box_dblocks == 0) box_dblocks = hd.nblk;   // default: the full head dim
  const int D = hd.blk * hd.nblk;
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return fail(FA2_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  if ((reinterpret_cast<uintptr_t>(ptr) & 15) != 0)
    return fail(FA2_ERR_UNSUPPORTED, "%s: pointer must be 16-byte aligned", what);
  if ((st.b % 8) || (st.s % 8) || (st.h % 8))
    return fail(FA2_ERR_UNSUPPORTED, "%s: strides must be multiples of 8 elements", what);
  if (st.s <= 0 || (H > 1 && st.h <= 0) || (B > 1 && st.b <= 0))
    return fail(FA2_ERR_INVALID_ARG, "%s: strides must be positive", what);
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(hd.blk), static_cast<cuuint64_t>(S),
                              static_cast<cuuint64_t>(hd.nblk), static_cast<cuuint64_t>(H),
                              static_cast<cuuint64_t>(B)};
  // A dimension of extent 1 still needs a legal (multiple of 16 bytes) stride.
  const cuuint64_t sh = static_cast<cuuint64_t>(st.h > 0 ? st.h : D) * 2;
  const cuuint64_t sb = static_cast<cuuint64_t>(st.b > 0 ? st.b : static_cast<int64_t>(D)) * 2;
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(st.s) * 2,
                                 static_cast<cuuint64_t>(hd.blk) * 2, sh, sb};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(box_rows),
                             static_cast<cuuint32_t>(box_dblocks), 1, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r =
      enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
          const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(FA2_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed with CUresult %d", what,
                static_cast<int>(r));
  return FA2_OK;
}

int check_problem(const fa2_problem& p) {
  if (p.batch <= 0 || p.seqlen_q <= 0 || p.seqlen_k <= 0 || p.heads_q <= 0 || p.heads_kv <= 0)
    return fail(FA2_ERR_INVALID_ARG, "batch, sequence lengths and head counts must be positive");
  if (p.heads_q % p.heads_kv != 0)
    return fail(FA2_ERR_INVALID_ARG, "query heads (%d) must be divisible by key/value heads (%d)",
                p.heads_q, p.heads_kv);
  if (p.dtype != FA2_FP16 && p.dtype != FA2_BF16)
    return fail(FA2_ERR_UNSUPPORTED, "only fp16 and bf16 inputs are supported");
  HeadDim hd;
  if (!split_head_dim(p.head_dim, &hd))
    return fail(FA2_ERR_UNSUPPORTED,
                "head_dim %d is not supported (multiples of 8 up to 64, of 16 up to 128, of 32 up to 256 are)",
                p.head_dim);
  if (!(p.dropout_p >= 0.f) || !(p.dropout_p < 1.f))
    return fail(FA2_ERR_INVALID_ARG, "dropout_p must be in [0, 1)");
  if (!std::isfinite(p.softmax_scale))
    return fail(FA2_ERR_INVALID_ARG, "softmax_scale must be finite");
  if (p.dropout_p > 0.f && (p.heads_q_global < p.head_offset + p.heads_q || p.batch_offset < 0 ||
                            p.head_offset < 0))
    return fail(FA2_ERR_INVALID_ARG, "dropout offsets: head_offset + heads_q exceeds heads_q_global");
  // The kernels count work items and blocks in 32-bit integers (one item per 128 query rows and
  // query head at most, times up to 32 key splits): refuse what would not fit instead of wrapping.
  const long long q_tiles = (static_cast<long long>(p.seqlen_q) + 127) / 128;
  const long long k_tiles = (static_cast<long long>(p.seqlen_k) + 127) / 128;
  const long long bh = static_cast<long long>(p.batch) * p.heads_q;
  if (bh > INT_MAX || bh * q_tiles * 32 > INT_MAX || bh * k_tiles * 2 > INT_MAX ||
      bh * p.seqlen_q > INT_MAX)
    return fail(FA2_ERR_UNSUPPORTED,
                "problem too large: batch * heads_q * max(seqlen_q, 64 * ceil(seqlen / 128)) must stay below 2^31");
  return FA2_OK;
}

int make_score_term(ScoreTermDev* out, const fa2_score_term& t, const fa2_problem& p,
                    const char* what) {
  std::memset(out, 0, sizeof(*out));
  out->head_div = 1;
  if (!t.ptr) return FA2_OK;
  if (t.head_div < 0 || (t.head_div > 1 && p.heads_q % t.head_div != 0))
    return fail(FA2_ERR_INVALID_ARG, "%s: head_div must divide heads_q", what);
  out->head_div = t.head_div > 1 ? t.head_div : 1;
  if (t.dtype != p.dtype && t.dtype != FA2_FP32)
    return fail(FA2_ERR_UNSUPPORTED, "%s: dtype must be the q dtype or fp32", what);
  if (t.stride_b < 0 || t.stride_h < 0 || t.stride_q < 0)
    return fail(FA2_ERR_INVALID_ARG, "%s: strides must be non-negative", what);
  out->ptr = t.ptr;
  out->sb = t.stride_b;
  out->sh = t.stride_h;
  out->sq = t.stride_q;
  out->is_f32 = (t.dtype == FA2_FP32);
  const int vec = out->is_f32 ? 4 : 8;
  out->vec_ok = ((reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0) && (t.stride_b % vec == 0) &&
                (t.stride_h % vec == 0) && (t.stride_q % vec == 0);
  return FA2_OK;
}

// Tensor map of an additive score term for the kernels that stage it in shared memory: the 4-D
// tensor (Sk, Sq, heads, batch) of 16-bit elements, broadcast dimensions with extent 1, box
// (64 keys, box_rows query rows). Sets t->staged when the term qualifies: the q dtype, a real query
// dimension, 16-byte aligned base and strides (the TMA unit's rules). Otherwise the term stays on
// the direct-load path and the map is left untouched.
void try_stage_term(CUtensorMap* tm, ScoreTermDev* t, const fa2_problem& p, int box_rows) {
  t->staged = 0;
  if (!t->ptr || t->is_f32 || t->sq <= 0) return;
  if ((reinterpret_cast<uintptr_t>(t->ptr) & 15) || (t->sq % 8) || (t->sh % 8) || (t->sb % 8)) return;
  if (p.seqlen_k < 8) return;
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return;
  const cuuint64_t nh = t->sh ? static_cast<cuuint64_t>(p.heads_q / t->head_div) : 1;
  const cuuint64_t nb = t->sb ? static_cast<cuuint64_t>(p.batch) : 1;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.seqlen_k), static_cast<cuuint64_t>(p.seqlen_q), nh, nb};
  // a dimension of extent 1 still needs a legal stride: the natural one
  const cuuint64_t s_q = static_cast<cuuint64_t>(t->sq) * 2;
  const cuuint64_t s_h = t->sh ? static_cast<cuuint64_t>(t->sh) * 2 : s_q * dims[1];
  const cuuint64_t s_b = t->sb ? static_cast<cuuint64_t>(t->sb) * 2 : s_h * nh;
  const cuuint64_t strides[3] = {s_q, s_h, s_b};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      enc(tm, p.dtype == FA2_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
          const_cast<void*>(t->ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) t->staged = 1;
}

void make_dropout(DropoutDev* d, const fa2_problem& p) {
  std::memset(d, 0, sizeof(*d));
  d->enabled = p.dropout_p > 0.f;
  d->inv_keep = 1.f;
  if (!d->enabled) return;
  // 16-bit draws: the drop probability is realised in steps of 2^-16
  const double thr = std::floor(static_cast<double>(p.dropout_p) * 65536.0 + 0.5);
  d->threshold = thr >= 65535.0 ? 65535u : static_cast<uint32_t>(thr);
  d->inv_keep = static_cast<float>(1.0 / (1.0 - static_cast<double>(p.dropout_p)));
  d->seed_lo = static_cast<uint32_t>(p.dropout_seed & 0xffffffffu);
  d->seed_hi = static_cast<uint32_t>(p.dropout_seed >> 32);
  d->b_off = p.batch_offset;
  d->h_off = p.head_offset;
  d->hq_global = p.heads_q_global;
}

size_t dropout_bits_bytes(const fa2_problem& p) {
  if (!(p.dropout_p > 0.f)) return 0;
  const size_t nqt = (static_cast<size_t>(p.seqlen_q) + 127) / 128, nkt = (static_cast<size_t>(p.seqlen_k) + 127) / 128;
  return static_cast<size_t>(p.batch) * p.heads_q * nqt * nkt * 2048;
}

// The optional record of the keep bits (written by the forward, read by the backward).
int set_dropout_bits(DropoutDev* d, const fa2_problem& p, const uint32_t* bits, size_t bytes) {
  d->bits = nullptr;
  if (!bits || !d->enabled) return FA2_OK;
  if (reinterpret_cast<uintptr_t>(bits) & 15)
    return fail(FA2_ERR_INVALID_ARG, "dropout_bits must be 16-byte aligned");
  if (bytes < dropout_bits_bytes(p))
    return fail(FA2_ERR_INVALID_ARG, "dropout_bits must hold %zu bytes", dropout_bits_bytes(p));
  d->bits = const_cast<uint32_t*>(bits);
  d->bits_nqt = (p.seqlen_q + 127) / 128;
  d->bits_nkt = (p.seqlen_k + 127) / 128;
  return FA2_OK;
}

// The optional device-resident operands of the dropout stream (seed, shard offsets).
int set_dropout_operands(DropoutDev* d, const uint64_t* seed_dev, const int32_t* offsets_dev) {
  if (seed_dev && (reinterpret_cast<uintptr_t>(seed_dev) & 7))
    return fail(FA2_ERR_INVALID_ARG, "dropout_seed_dev must be 8-byte aligned");
  if (offsets_dev && (reinterpret_cast<uintptr_t>(offsets_dev) & 3))
    return fail(FA2_ERR_INVALID_ARG, "offsets_dev must be 4-byte aligned");
  d->seed_dev = reinterpret_cast<const unsigned long long*>(seed_dev);
  d->offsets_dev = offsets_dev;
  return FA2_OK;
}

// What the kernels need of a scratch pointer: 16-byte bulk copies and float4 accesses; 128 bytes is
// what allocators of every framework (XLA's sub-allocated temporaries included) guarantee.
constexpr uintptr_t kWorkspaceAlign = 128;

// Bytes of Q, dO and dq-accumulator tiles that one chunk of the backward's launch order may span.
// Measured on B=8, S=4096, Hq=32, Hkv=8, D=128 causal (16 MiB per group): main kernel 2.76 ms with
// chunks of 1 or 2 groups, 2.58-2.63 ms with 4, 8 or 16; only a few of a chunk's key tiles run at
// any time, so the live set stays well below this figure.
constexpr size_t kSchedL2Bytes = 128u << 20;

size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

struct BwdWorkspace {
  size_t delta_off, dq_off, absmax_off, xstats_off, order_off, total;
  int sq_pad;
  // attention with changed scores: the parts of the query heads and their dK and dV behind all else
  int parts;
  size_t parts_off, parts_total;
};
// Parts into which the backward of attention with changed scores deals the query heads of a key/value head: as many (a
// divisor of them) as find an SM each, if that takes at least 2 of the 128-query steps off a key tile's way; joining the parts
// costs about as much as one step, 2 to 3 us. Measured (causal, bf16, whole backward, one part -> parts): 4096 queries, 16/2
// heads, D = 128 633 -> 346 us, 16/1 heads, D = 64 915 -> 251 us; 1 x 512, 32/8 heads, D = 128 63 -> 40 us; 1 x 1024, 8/1 heads,
// D = 256 256 -> 64 us; two steps less: 1 x 256, 8/4 heads, D = 128 33 -> 31 us; one less: 1 x 128, 8/4 heads, D = 128 28 -> 33 us
// (with a join of twice today's time).
int bwd_parts(const fa2_problem& p, const HeadDim& hd) {
  const int64_t tiles = static_cast<int64_t>(p.batch) * p.heads_kv * ((p.seqlen_k + 127) / 128) * (hd.padded == 256 ? 2 : 1);
  const int64_t group = p.heads_q / p.heads_kv, room = sm_count() / tiles;
  int64_t parts = 1;
  for (int64_t d = 2; d <= std::min(group, room); ++d)
    if (group % d == 0) parts = d;
  const int64_t steps = (static_cast<int64_t>(p.seqlen_q) + 127) / 128 * group;
  return steps - steps / parts >= 2 ? static_cast<int>(parts) : 1;
}
BwdWorkspace bwd_workspace(const fa2_problem& p, bool scored = false) {
  BwdWorkspace w;
  w.sq_pad = (p.seqlen_q + 127) / 128 * 128;
  const size_t rows = static_cast<size_t>(p.batch) * p.heads_q * w.sq_pad;
  w.delta_off = 0;
  w.dq_off = align_up(2 * rows * sizeof(float), 256);   // (lse2, delta) per row
  HeadDim hd;
  split_head_dim(p.head_dim, &hd);   // checked by the callers
  w.absmax_off = w.dq_off + align_up(rows * hd.padded * sizeof(float), 256);
  w.xstats_off = w.absmax_off + 256;   // one word: max|dO| of the call (fp16 range guard)
  // the row statistics once more as MMA operand tiles, 4 KiB per 128 rows (head dim 128)
  const bool fold = hd.padded == 128;
  w.order_off = w.xstats_off + (fold ? rows / 128 * 4096 : 0);
  // counters for the bit-reproducible mode: one per 128-row dQ tile, at head dim 256 one per
  // 64 rows and half of the head dim
  w.total = w.order_off + align_up(rows / 128 * (hd.padded <= 128 ? 1 : 4) * sizeof(int), 256);
  w.parts = scored ? bwd_parts(p, hd) : 1;
  w.parts_off = w.total;
  const size_t kv_rows = static_cast<size_t>(p.batch) * p.heads_kv * ((static_cast<size_t>(p.seqlen_k) + 127) / 128 * 128);
  w.parts_total = w.total + (w.parts > 1 ? 2 * w.parts * kv_rows * hd.padded * sizeof(float) : 0);
  return w;
}

// Split-KV plan of the forward: how many parts the key sequence is
// cut into and how many K/V tiles each part gets. A problem is split when its (query block,
// batch, head) items would leave more than half of the SMs idle and the key sequence is long
// enough to share out.
struct SplitPlan {
  int n_splits, split_tiles;
  int sq_k, hq_k;          // the problem as the kernel sees it (after packing grouped heads)
  size_t part_o_bytes, part_lse_off, total;
};
SplitPlan plan_splits(const fa2_problem& p, const HeadDim& hd, bool pack_heads) {
  SplitPlan s{};
  s.n_splits = 1;
  s.sq_k = pack_heads ? p.heads_q / p.heads_kv : p.seqlen_q;
  s.hq_k = pack_heads ? p.heads_kv : p.heads_q;
  const int n_tiles = (p.seqlen_k + 127) / 128;
  // work items: 256 query rows per item in the head dim <= 128 kernel, 128 in the head dim 256 one
  const int item_rows = hd.padded > 128 ? 128 : 256;
  const long long items = static_cast<long long>((s.sq_k + item_rows - 1) / item_rows) * p.batch * s.hq_k;
  const int sms = sm_count();
  if (n_tiles < 8 || items * 2 > sms) return s;
  int want = static_cast<int>(std::min<long long>(std::min<long long>(sms / items, n_tiles / 4), 32));
  if (want < 2) return s;
  s.split_tiles = (n_tiles + want - 1) / want;
  s.n_splits = (n_tiles + s.split_tiles - 1) / s.split_tiles;
  if (s.n_splits < 2) {
    s.n_splits = 1;
    return s;
  }
  const size_t rows = static_cast<size_t>(s.n_splits) * p.batch * s.sq_k * s.hq_k;
  s.part_o_bytes = align_up(rows * hd.padded * sizeof(float), 256);
  s.part_lse_off = s.part_o_bytes;
  const size_t sq_pad = static_cast<size_t>((s.sq_k + 127) / 128) * 128;
  s.total = s.part_lse_off + align_up(static_cast<size_t>(s.n_splits) * p.batch * s.hq_k * sq_pad * 4, 256);
  return s;
}

bool can_pack_heads(const fa2_problem& p) {
  const int group = p.heads_kv > 0 ? p.heads_q / p.heads_kv : 0;
  return p.seqlen_q == 1 && group > 1 && group <= 128 && !(p.dropout_p > 0.f);
}

// Sizes and parts of a document layout (int32): token bounds [B][S] twice, tile bounds [B][ceil(S/128)] twice, order of the
// blocks of 256 rows [B * ceil(S/256)].
size_t document_layout_ints(int64_t batch, int64_t seqlen) {
  const size_t s = static_cast<size_t>(seqlen);
  return static_cast<size_t>(batch) * (2 * s + 2 * ((s + 127) / 128) + (s + 255) / 256);
}

constexpr float kMinSoftcap = 1.f / 1024.f, kMaxSoftcap = 1024.f;

int check_softcap(float cap) {
  if (cap != 0.f && !(cap >= kMinSoftcap && cap <= kMaxSoftcap))
    return fail(FA2_ERR_INVALID_ARG, "softcap must be 0 (none) or in [2^-10, 1024]");
  return FA2_OK;
}

// Checks the score changes of a call and fills the kernels' record; `mode` receives kModCap | kModSlope.
int make_score_mod(ScoreModDev* out, int* mode, const fa2_score_mod& m, const fa2_problem& p) {
  std::memset(out, 0, sizeof(*out));
  const int rc = check_softcap(m.softcap);
  if (rc) return rc;
  if (!(p.softmax_scale >= 1e-30f))
    return fail(FA2_ERR_INVALID_ARG, "softmax_scale must be positive in attention with changed scores");
  if (p.dropout_p > 0.f) return fail(FA2_ERR_UNSUPPORTED, "dropout is not supported in attention with changed scores");
  if (m.prefix_lens && !p.causal) return fail(FA2_ERR_INVALID_ARG, "prefix_lens needs causal masking");
  if (m.document_layout && p.seqlen_q != p.seqlen_k)
    return fail(FA2_ERR_INVALID_ARG, "documents require seqlen_q == seqlen_k");
  if ((reinterpret_cast<uintptr_t>(m.alibi_slopes) | reinterpret_cast<uintptr_t>(m.prefix_lens) |
       reinterpret_cast<uintptr_t>(m.document_layout)) & 3)
    return fail(FA2_ERR_INVALID_ARG, "alibi_slopes, prefix_lens and document_layout must be 4-byte aligned");
  *mode = 0;
  if (m.softcap > 0.f) {
    *mode |= kModCap;
    out->cap2 = static_cast<float>(m.softcap * 1.4426950408889634);
    out->arg2 = static_cast<float>(2.0 * p.softmax_scale * 1.4426950408889634 / m.softcap);
    if (!std::isfinite(out->arg2)) return fail(FA2_ERR_INVALID_ARG, "softmax_scale / softcap overflows");
  }
  if (m.alibi_slopes) *mode |= kModSlope;
  out->slopes = m.alibi_slopes;
  out->prefix_lens = m.prefix_lens;
  out->causal = p.causal != 0;
  if (m.document_layout) {
    const size_t tokens = static_cast<size_t>(p.batch) * p.seqlen_q;
    const size_t tiles = static_cast<size_t>(p.batch) * ((static_cast<size_t>(p.seqlen_q) + 127) / 128);
    out->tok_lo = m.document_layout;
    out->tok_hi = out->tok_lo + tokens;
    out->tile_lo = out->tok_hi + tokens;
    out->tile_hi = out->tile_lo + tiles;
    out->order = out->tile_hi + tiles;
  }
  if (m.o_rest) {
    if (reinterpret_cast<uintptr_t>(m.o_rest) & 15) return fail(FA2_ERR_UNSUPPORTED, "o_rest must be 16-byte aligned");
    if ((m.o_rest_strides.b % 8) || (m.o_rest_strides.s % 8) || (m.o_rest_strides.h % 8))
      return fail(FA2_ERR_UNSUPPORTED, "o_rest: strides must be multiples of 8 elements");
    HeadDim hd;
    split_head_dim(p.head_dim, &hd);
    out->rest = static_cast<uint16_t*>(m.o_rest);
    out->rest_sb = m.o_rest_strides.b;
    out->rest_ss = m.o_rest_strides.s;
    out->rest_sh = m.o_rest_strides.h;
    out->rest_blk = hd.blk;
  }
  return FA2_OK;
}

cudaError_t launch_fwd_scored(const FwdLaunch& a, int mode, cudaStream_t stream) {
  return a.head_dim == 64    ? launch_fwd_scored64(a, mode, stream)
         : a.head_dim == 128 ? launch_fwd_scored128(a, mode, stream)
                             : launch_fwd_scored256(a, mode, stream);
}
cudaError_t launch_bwd_scored(const BwdLaunch& a, int mode, cudaStream_t stream) {
  return a.head_dim == 64    ? launch_bwd_scored64(a, mode, stream)
         : a.head_dim == 128 ? launch_bwd_scored128(a, mode, stream)
                             : launch_bwd_scored256(a, mode, stream);
}

int fwd_impl(const fa2_fwd_params* a, const fa2_score_mod* mod, void* cuda_stream);
int bwd_impl(const fa2_bwd_params* a, const fa2_score_mod* mod, void* cuda_stream);

}  // namespace
}  // namespace fa2

using namespace fa2;

extern "C" {

int fa2_version(void) { return FA2_ABI_VERSION; }

const char* fa2_last_error(void) { return g_err; }

int fa2_debug_device_status(void* cuda_stream) {
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  int* dptr = status_ptr();
  if (!dptr) return fail(FA2_ERR_CUDA, "status word is not addressable");
  int v = 0;
  if (cudaStreamSynchronize(stream) != cudaSuccess ||
      cudaMemcpy(&v, dptr, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess)
    return fail(FA2_ERR_CUDA, "reading the status word failed: %s",
                cudaGetErrorString(cudaGetLastError()));
  if (v != 0) cudaMemset(dptr, 0, sizeof(int));
  return v;
}

int fa2_debug_bwd_stage_events(void* const* events) {
  for (int i = 0; i < 4; ++i) g_bwd_events[i] = events ? static_cast<cudaEvent_t>(events[i]) : nullptr;
  return FA2_OK;
}

int fa2_fwd(const fa2_fwd_params* a, void* cuda_stream) { return fwd_impl(a, nullptr, cuda_stream); }

size_t fa2_fwd_workspace_bytes(const fa2_problem* problem) {
  if (!problem || check_problem(*problem)) return 0;
  HeadDim hd;
  split_head_dim(problem->head_dim, &hd);
  // whether grouped heads get packed also depends on operands this function does not see
  // (bias, mask, lengths): report what the larger of the two plans needs
  size_t need = plan_splits(*problem, hd, false).total;
  if (can_pack_heads(*problem)) need = std::max(need, plan_splits(*problem, hd, true).total);
  return need;
}

size_t fa2_dropout_bits_bytes(const fa2_problem* problem) {
  if (!problem || check_problem(*problem)) return 0;
  return dropout_bits_bytes(*problem);
}

size_t fa2_bwd_workspace_bytes(const fa2_problem* problem) {
  if (!problem || check_problem(*problem)) return 0;
  return bwd_workspace(*problem).total;
}

int fa2_bwd(const fa2_bwd_params* a, void* cuda_stream) { return bwd_impl(a, nullptr, cuda_stream); }

// ---------------------------------------------------------------------------------------------
// Backward without a caller-provided workspace
// ---------------------------------------------------------------------------------------------
namespace {
// Scratch of the backward (row statistics + fp32 dq accumulator) for callers that cannot hand
// in device memory of their own. One array per GPU that loads the library, held until exit.
static __device__ __align__(256) unsigned char g_bwd_static_scratch[FA2_BWD_STATIC_SCRATCH_BYTES];

constexpr int kMaxDevices = 64;
void* g_static_scratch_ptr[kMaxDevices] = {};
std::mutex g_static_scratch_mutex;

// Device address of the array on the current device. In host code the array's name is only a
// handle for the runtime, not an address a kernel could use, so the address is looked up once per
// device (with that device current) and cached.
int static_scratch_address(void** out) {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices)
    return fail(FA2_ERR_CUDA, "cannot identify the current CUDA device");
  std::lock_guard<std::mutex> lock(g_static_scratch_mutex);
  if (!g_static_scratch_ptr[dev]) {
    void* ptr = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&ptr, g_bwd_static_scratch);
    if (e != cudaSuccess || !ptr)
      return fail(FA2_ERR_CUDA, "cudaGetSymbolAddress failed for the static scratch: %s",
                  cudaGetErrorString(e));
    g_static_scratch_ptr[dev] = ptr;
  }
  *out = g_static_scratch_ptr[dev];
  return FA2_OK;
}
}  // namespace

int fa2_bwd_static_scratch(const fa2_bwd_params* a, void* cuda_stream) {
  if (!a) return fail(FA2_ERR_INVALID_ARG, "params is null");
  const int rc = check_problem(a->p);
  if (rc) return rc;
  const size_t need = bwd_workspace(a->p).total;
  if (need > static_cast<size_t>(FA2_BWD_STATIC_SCRATCH_BYTES))
    return fail(FA2_ERR_WORKSPACE,
                "this problem needs %zu bytes of scratch; the built-in scratch holds %zu bytes "
                "(batch * heads_q * ceil(seqlen_q/128)*128 * (head_dim + 2) * 4 must not exceed it); "
                "use fa2_bwd with a workspace instead",
                need, static_cast<size_t>(FA2_BWD_STATIC_SCRATCH_BYTES));
  void* scratch = nullptr;
  const int rs = static_scratch_address(&scratch);
  if (rs) return rs;
  fa2_bwd_params b = *a;
  b.workspace = scratch;
  b.workspace_bytes = FA2_BWD_STATIC_SCRATCH_BYTES;
  return fa2_bwd(&b, cuda_stream);
}

// ---------------------------------------------------------------------------------------------
// Attention with changed scores (fa2_b200_lm.h)
// ---------------------------------------------------------------------------------------------
int fa2_lm_version(void) { return FA2_LM_ABI_VERSION; }

int fa2_scored_fwd(const fa2_fwd_params* a, const fa2_score_mod* mod, void* cuda_stream) {
  if (!mod) return fail(FA2_ERR_INVALID_ARG, "mod is null");
  return fwd_impl(a, mod, cuda_stream);
}

size_t fa2_scored_bwd_workspace_bytes(const fa2_problem* problem) {
  if (!problem || check_problem(*problem)) return 0;
  return bwd_workspace(*problem, true).parts_total;
}

int fa2_scored_bwd(const fa2_bwd_params* a, const fa2_score_mod* mod, void* cuda_stream) {
  if (!mod) return fail(FA2_ERR_INVALID_ARG, "mod is null");
  return bwd_impl(a, mod, cuda_stream);
}

size_t fa2_document_layout_bytes(int32_t batch, int32_t seqlen) {
  if (batch <= 0 || seqlen <= 0) return 0;
  return document_layout_ints(batch, seqlen) * sizeof(int32_t);
}

int fa2_document_layout(const int32_t* document_ids, int64_t stride_b, int32_t batch, int32_t seqlen, int32_t* layout,
                        size_t layout_bytes, void* cuda_stream) {
  if (!document_ids || !layout) return fail(FA2_ERR_INVALID_ARG, "document_ids and layout must be non-null");
  if (batch <= 0 || seqlen <= 0) return fail(FA2_ERR_INVALID_ARG, "batch and seqlen must be positive");
  if (seqlen > INT_MAX - 8192) return fail(FA2_ERR_UNSUPPORTED, "seqlen must stay below 2^31 - 8192");
  if (stride_b < 0) return fail(FA2_ERR_INVALID_ARG, "the stride of document_ids must be non-negative");
  if (reinterpret_cast<uintptr_t>(document_ids) & 3)
    return fail(FA2_ERR_INVALID_ARG, "document_ids must be 4-byte aligned");
  if (reinterpret_cast<uintptr_t>(layout) & 15) return fail(FA2_ERR_INVALID_ARG, "layout must be 16-byte aligned");
  if (static_cast<int64_t>(batch) * ((seqlen + 255) / 256) > INT_MAX)
    return fail(FA2_ERR_UNSUPPORTED, "batch * seqlen is too large");
  const size_t need = document_layout_ints(batch, seqlen) * sizeof(int32_t);
  if (layout_bytes < need) return fail(FA2_ERR_INVALID_ARG, "layout must hold %zu bytes", need);
  const cudaError_t e =
      launch_document_layout(document_ids, stride_b, batch, seqlen, layout, static_cast<cudaStream_t>(cuda_stream));
  if (e != cudaSuccess) return fail(FA2_ERR_CUDA, "document layout launch failed: %s", cudaGetErrorString(e));
  return FA2_OK;
}

// ---------------------------------------------------------------------------------------------
// Serving with a paged cache (fa2_b200_lm.h)
// ---------------------------------------------------------------------------------------------
namespace {
constexpr int kMaxRequests = 8192;
constexpr int64_t kMaxContext = 1 << 30;   // keys a table can hold: positions and tile counts stay within 32 bits

int check_groups(int32_t heads_q, int32_t heads_kv) {
  if (heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv != 0)
    return fail(FA2_ERR_INVALID_ARG, "query heads (%d) must be divisible by key/value heads (%d)", heads_q, heads_kv);
  if (heads_q / heads_kv > 128)
    return fail(FA2_ERR_UNSUPPORTED, "at most 128 query heads per key/value head are supported");
  return FA2_OK;
}
// log2 of a page size, or -1
int page_shift_of(int32_t page_size) {
  if (page_size < 8 || page_size > (1 << 20) || (page_size & (page_size - 1))) return -1;
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}
int item_tokens_of(int32_t heads_q, int32_t heads_kv) { return 2 * (128 / (heads_q / heads_kv)); }
int64_t max_items(int64_t requests, int64_t tokens, int64_t item_tokens) {
  return std::min(tokens, tokens / item_tokens + requests);
}

int check_cache(const fa2_paged_cache& c, const char* what) {
  if (!c.ptr) return fail(FA2_ERR_INVALID_ARG, "%s must be non-null", what);
  if (reinterpret_cast<uintptr_t>(c.ptr) & 15) return fail(FA2_ERR_UNSUPPORTED, "%s: pointer must be 16-byte aligned", what);
  if (c.stride_page <= 0 || c.stride_slot <= 0 || c.stride_head <= 0)
    return fail(FA2_ERR_INVALID_ARG, "%s: strides must be positive", what);
  if ((c.stride_page % 8) || (c.stride_slot % 8) || (c.stride_head % 8))
    return fail(FA2_ERR_UNSUPPORTED, "%s: strides must be multiples of 8 elements", what);
  return FA2_OK;
}

// 5-D map of 16-bit elements with a 128-byte swizzle.
int encode_map(CUtensorMap* tm, const void* ptr, bool bf16, const cuuint64_t (&dims)[5], const cuuint64_t (&strides)[4],
               const cuuint32_t (&box)[5], CUtensorMapL2promotion promotion, const char* what) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return fail(FA2_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                         const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(FA2_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed with CUresult %d", what, static_cast<int>(r));
  return FA2_OK;
}
}  // namespace

size_t fa2_paged_work_bytes(int32_t requests, int32_t num_tokens, int32_t heads_q, int32_t heads_kv) {
  if (requests <= 0 || num_tokens < 0 || check_groups(heads_q, heads_kv)) return 0;
  return (work_items_at(sm_count()) +
          kWorkItem * static_cast<size_t>(max_items(requests, num_tokens, item_tokens_of(heads_q, heads_kv)))) * sizeof(int32_t);
}

int fa2_paged_plan(const fa2_paged_plan_params* a, void* cuda_stream) {
  if (!a) return fail(FA2_ERR_INVALID_ARG, "params is null");
  if (a->requests <= 0 || a->num_tokens < 0 || a->table_width <= 0 || a->n_free < 0)
    return fail(FA2_ERR_INVALID_ARG, "requests and table_width must be positive, num_tokens and n_free not negative");
  if (a->requests > kMaxRequests) return fail(FA2_ERR_UNSUPPORTED, "at most %d requests are supported", kMaxRequests);
  const int rc = check_groups(a->heads_q, a->heads_kv);
  if (rc) return rc;
  const int shift = page_shift_of(a->page_size);
  if (shift < 0) return fail(FA2_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 2^20");
  if (!a->context_lens || !a->new_lens || !a->block_table || (!a->free_pages && a->n_free > 0) || !a->cu_seqlens ||
      !a->seqlens_k || (a->num_tokens > 0 && (!a->slot_map || !a->positions)) || !a->pages_taken || !a->work)
    return fail(FA2_ERR_INVALID_ARG, "the plan's arrays must be non-null");
  if (a->table_stride < a->table_width) return fail(FA2_ERR_INVALID_ARG, "table_stride must be at least table_width");
  if ((static_cast<int64_t>(a->table_width) << shift) > kMaxContext)
    return fail(FA2_ERR_UNSUPPORTED, "table_width * page_size must not exceed 2^30");
  if ((reinterpret_cast<uintptr_t>(a->context_lens) | reinterpret_cast<uintptr_t>(a->new_lens) |
       reinterpret_cast<uintptr_t>(a->block_table) | reinterpret_cast<uintptr_t>(a->free_pages) |
       reinterpret_cast<uintptr_t>(a->free_start) | reinterpret_cast<uintptr_t>(a->cu_seqlens) |
       reinterpret_cast<uintptr_t>(a->seqlens_k) | reinterpret_cast<uintptr_t>(a->positions) |
       reinterpret_cast<uintptr_t>(a->pages_taken)) & 3)
    return fail(FA2_ERR_INVALID_ARG, "the plan's int32 arrays must be 4-byte aligned");
  if ((reinterpret_cast<uintptr_t>(a->slot_map) & 7) || (reinterpret_cast<uintptr_t>(a->work) & 15))
    return fail(FA2_ERR_INVALID_ARG, "slot_map must be 8-byte and work 16-byte aligned");
  const int item_tokens = item_tokens_of(a->heads_q, a->heads_kv);
  const int64_t items = max_items(a->requests, a->num_tokens, item_tokens);
  if (a->work_bytes < (work_items_at(sm_count()) + kWorkItem * static_cast<size_t>(items)) * sizeof(int32_t))
    return fail(FA2_ERR_WORKSPACE, "work must hold fa2_paged_work_bytes bytes");
  const int64_t tiles = ((static_cast<int64_t>(a->table_width) << shift) + 127) / 128;
  if (items * (kTileCost2 * tiles + kItemCost2) > INT_MAX)
    return fail(FA2_ERR_UNSUPPORTED, "problem too large: %lld items of up to %lld key tiles must stay below 2^29",
                static_cast<long long>(items), static_cast<long long>(tiles));
  PagedPlanDev d;
  d.context_lens = a->context_lens;
  d.new_lens = a->new_lens;
  d.B = a->requests;
  d.block_table = a->block_table;
  d.table_stride = a->table_stride;
  d.table_width = a->table_width;
  d.free_pages = a->free_pages;
  d.n_free = a->n_free;
  d.free_start = a->free_start;
  d.page_shift = shift;
  d.num_tokens = a->num_tokens;
  d.item_tokens = item_tokens;
  d.heads_kv = a->heads_kv;
  d.sms = sm_count();
  d.items_at = work_items_at(d.sms);
  d.cu_seqlens = a->cu_seqlens;
  d.seqlens_k = a->seqlens_k;
  d.slot_map = reinterpret_cast<long long*>(a->slot_map);
  d.positions = a->positions;
  d.pages_taken = a->pages_taken;
  d.work = a->work;
  const cudaError_t e = launch_paged_plan(d, static_cast<cudaStream_t>(cuda_stream));
  if (e != cudaSuccess) return fail(FA2_ERR_CUDA, "plan launch failed: %s", cudaGetErrorString(e));
  return FA2_OK;
}

int fa2_paged_cache_write(const fa2_paged_write_params* a, void* cuda_stream) {
  if (!a) return fail(FA2_ERR_INVALID_ARG, "params is null");
  if (a->tokens < 0 || a->heads <= 0 || a->head_dim <= 0 || a->pages <= 0)
    return fail(FA2_ERR_INVALID_ARG, "heads, head_dim and pages must be positive, tokens not negative");
  const int shift = page_shift_of(a->page_size);
  if (shift < 0) return fail(FA2_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 2^20");
  if (a->head_dim % 8) return fail(FA2_ERR_UNSUPPORTED, "head_dim must be a multiple of 8");
  int rc = check_cache(a->k_cache, "k_cache");
  if (!rc) rc = check_cache(a->v_cache, "v_cache");
  if (rc) return rc;
  if (a->tokens == 0) return FA2_OK;
  if (!a->k || !a->v || !a->slot_map) return fail(FA2_ERR_INVALID_ARG, "k, v and slot_map must be non-null");
  if ((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) & 15)
    return fail(FA2_ERR_UNSUPPORTED, "k and v must be 16-byte aligned");
  if ((a->k_stride_t % 8) || (a->k_stride_h % 8) || (a->v_stride_t % 8) || (a->v_stride_h % 8))
    return fail(FA2_ERR_UNSUPPORTED, "k and v: strides must be multiples of 8 elements");
  if (a->k_stride_t < 0 || a->k_stride_h < 0 || a->v_stride_t < 0 || a->v_stride_h < 0)
    return fail(FA2_ERR_INVALID_ARG, "k and v: strides must not be negative");
  if (reinterpret_cast<uintptr_t>(a->slot_map) & 7) return fail(FA2_ERR_INVALID_ARG, "slot_map must be 8-byte aligned");
  const int64_t per_token = static_cast<int64_t>(a->heads) * (a->head_dim / 8);
  if (per_token > INT_MAX || a->tokens * per_token > 256LL * INT_MAX)
    return fail(FA2_ERR_UNSUPPORTED, "tokens * heads * head_dim is too large");
  PagedWriteDev d;
  d.k = static_cast<const uint16_t*>(a->k);
  d.v = static_cast<const uint16_t*>(a->v);
  d.k_st = a->k_stride_t; d.k_sh = a->k_stride_h;
  d.v_st = a->v_stride_t; d.v_sh = a->v_stride_h;
  d.k_cache = static_cast<uint16_t*>(const_cast<void*>(a->k_cache.ptr));
  d.v_cache = static_cast<uint16_t*>(const_cast<void*>(a->v_cache.ptr));
  d.kc_sp = a->k_cache.stride_page; d.kc_ss = a->k_cache.stride_slot; d.kc_sh = a->k_cache.stride_head;
  d.vc_sp = a->v_cache.stride_page; d.vc_ss = a->v_cache.stride_slot; d.vc_sh = a->v_cache.stride_head;
  d.slot_map = reinterpret_cast<const long long*>(a->slot_map);
  d.slots = static_cast<long long>(a->pages) << shift;
  d.tokens = a->tokens;
  d.heads = a->heads;
  d.chunks_per_head = a->head_dim / 8;
  d.page_shift = shift;
  const cudaError_t e = launch_paged_write(d, static_cast<cudaStream_t>(cuda_stream));
  if (e != cudaSuccess) return fail(FA2_ERR_CUDA, "cache write launch failed: %s", cudaGetErrorString(e));
  return FA2_OK;
}

size_t fa2_paged_workspace_bytes(int32_t head_dim) {
  HeadDim hd;
  if (!split_head_dim(head_dim, &hd) || hd.padded > 128) return 0;
  // two partial items of 256 rows per CTA: the rows, then their log-sum-exp
  return static_cast<size_t>(2) * sm_count() * 256 * (hd.padded + 1) * sizeof(float);
}

int fa2_paged_attention(const fa2_paged_attention_params* a, void* cuda_stream) {
  if (!a) return fail(FA2_ERR_INVALID_ARG, "params is null");
  if (a->tokens < 0 || a->requests <= 0 || a->table_width <= 0 || a->pages <= 0)
    return fail(FA2_ERR_INVALID_ARG, "requests, table_width and pages must be positive, tokens not negative");
  int rc = check_groups(a->heads_q, a->heads_kv);
  if (rc) return rc;
  if (a->dtype != FA2_FP16 && a->dtype != FA2_BF16)
    return fail(FA2_ERR_UNSUPPORTED, "only fp16 and bf16 inputs are supported");
  HeadDim hd;
  if (!split_head_dim(a->head_dim, &hd) || hd.padded > 128)
    return fail(FA2_ERR_UNSUPPORTED, "head_dim %d is not supported (multiples of 8 up to 64, of 16 up to 128 are)", a->head_dim);
  const int shift = page_shift_of(a->page_size);
  if (shift < 0) return fail(FA2_ERR_UNSUPPORTED, "page_size must be a power of two from 8 to 2^20");
  if ((static_cast<int64_t>(a->table_width) << shift) > kMaxContext)
    return fail(FA2_ERR_UNSUPPORTED, "table_width * page_size must not exceed 2^30");
  if (!(a->softmax_scale >= 1e-30f) || !std::isfinite(a->softmax_scale))
    return fail(FA2_ERR_INVALID_ARG, "softmax_scale must be positive and finite");
  if ((rc = check_softcap(a->softcap))) return rc;
  if ((rc = check_cache(a->k_cache, "k_cache")) || (rc = check_cache(a->v_cache, "v_cache"))) return rc;
  if (a->tokens == 0) return FA2_OK;
  if (!a->q || !a->o || !a->block_table || !a->work)
    return fail(FA2_ERR_INVALID_ARG, "q, o, block_table and work must be non-null");
  if (a->table_stride < a->table_width) return fail(FA2_ERR_INVALID_ARG, "table_stride must be at least table_width");
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->o)) & 15)
    return fail(FA2_ERR_UNSUPPORTED, "q and o must be 16-byte aligned");
  if ((a->q_stride_t % 8) || (a->q_stride_h % 8) || (a->o_stride_t % 8) || (a->o_stride_h % 8))
    return fail(FA2_ERR_UNSUPPORTED, "q and o: strides must be multiples of 8 elements");
  if (a->q_stride_t <= 0 || a->q_stride_h <= 0 || a->o_stride_t <= 0 || a->o_stride_h <= 0)
    return fail(FA2_ERR_INVALID_ARG, "q and o: strides must be positive");
  if ((reinterpret_cast<uintptr_t>(a->work) & 15) || ((reinterpret_cast<uintptr_t>(a->block_table) |
       reinterpret_cast<uintptr_t>(a->lse) | reinterpret_cast<uintptr_t>(a->alibi_slopes)) & 3))
    return fail(FA2_ERR_INVALID_ARG, "work must be 16-byte, block_table, lse and alibi_slopes 4-byte aligned");
  // a runtime call before the driver-level tensor-map encoder: see fwd_impl
  int* const status_word = status_ptr();
  if (!status_word) return fail(FA2_ERR_CUDA, "status word is not addressable");
  const size_t need = fa2_paged_workspace_bytes(a->head_dim);
  if (!a->workspace || a->workspace_bytes < need) return fail(FA2_ERR_WORKSPACE, "workspace must hold %zu bytes", need);
  if (reinterpret_cast<uintptr_t>(a->workspace) & (kWorkspaceAlign - 1))
    return fail(FA2_ERR_WORKSPACE, "workspace must be 128-byte aligned");

  PagedAttnLaunch L;
  std::memset(&L, 0, sizeof(L));
  const bool bf16 = a->dtype == FA2_BF16;
  const int group = a->heads_q / a->heads_kv, tile_tokens = 128 / group;
  const auto bytes = [](int64_t elements) { return static_cast<cuuint64_t>(elements) * 2; };
  {
    // (columns, heads of a group, tokens, column blocks, key/value heads): a box is the rows of one query tile
    const cuuint64_t dims[5] = {static_cast<cuuint64_t>(hd.blk), static_cast<cuuint64_t>(group),
                                static_cast<cuuint64_t>(a->tokens), static_cast<cuuint64_t>(hd.nblk),
                                static_cast<cuuint64_t>(a->heads_kv)};
    const cuuint64_t st[4] = {bytes(a->q_stride_h), bytes(a->q_stride_t), bytes(hd.blk), bytes(a->q_stride_h * group)};
    const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(tile_tokens), 1, 1};
    if ((rc = encode_map(&L.tmQ, a->q, bf16, dims, st, box, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, "q"))) return rc;
  }
  // Two column blocks in one box: the places of a page count as groups of 8, and one dimension serves for two where pages lie
  // one behind the other (groups of all pages) or the heads of all pages do.
  const int64_t page_groups = a->page_size / 8, all_groups = page_groups * (a->pages + INT64_C(1)),
                all_heads = a->heads_kv * (a->pages + INT64_C(1));
  const auto pages_in_line = [&](const fa2_paged_cache& c) { return c.stride_page == c.stride_slot * a->page_size; };
  const auto heads_in_line = [&](const fa2_paged_cache& c) { return c.stride_page == c.stride_head * a->heads_kv; };
  const bool by_groups = all_groups <= INT_MAX && pages_in_line(a->k_cache) && pages_in_line(a->v_cache);
  const bool by_heads = !by_groups && all_heads <= INT_MAX && heads_in_line(a->k_cache) && heads_in_line(a->v_cache);
  const bool whole_rows = hd.padded == 128 && (by_groups || by_heads);
  for (int x = 0; x < 2; ++x) {
    // (columns, places in a page, column blocks, heads, pages): a box is a piece of a page of at most 128 rows
    const fa2_paged_cache& c = x ? a->v_cache : a->k_cache;
    const cuuint64_t dims[5] = {static_cast<cuuint64_t>(hd.blk), static_cast<cuuint64_t>(a->page_size),
                                static_cast<cuuint64_t>(hd.nblk), static_cast<cuuint64_t>(a->heads_kv),
                                static_cast<cuuint64_t>(a->pages)};
    const cuuint64_t st[4] = {bytes(c.stride_slot), bytes(hd.blk), bytes(c.stride_head), bytes(c.stride_page)};
    const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(std::min(a->page_size, 128)), 1, 1, 1};
    // Up to 64 columns a key takes 128 bytes: fetching 256 would bring the next head's into L2, where it is not needed
    // before another CTA comes there (16 decodes over 16000 keys, 16/8 heads, D = 64, pages of 64: 138 us, 121 with 128).
    const CUtensorMapL2promotion promotion =
        hd.padded == 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_256B;
    if (whole_rows) {
      // (columns, 8 places, column blocks, groups of 8 places, heads)
      const cuuint64_t dims_w[5] = {static_cast<cuuint64_t>(hd.blk), 8, static_cast<cuuint64_t>(hd.nblk),
                                    static_cast<cuuint64_t>(by_groups ? page_groups * a->pages : page_groups),
                                    static_cast<cuuint64_t>(by_groups ? a->heads_kv : static_cast<int64_t>(a->heads_kv) * a->pages)};
      const cuuint64_t st_w[4] = {bytes(c.stride_slot), bytes(hd.blk), bytes(c.stride_slot * 8), bytes(c.stride_head)};
      const cuuint32_t box_w[5] = {64, 8, 2, static_cast<cuuint32_t>(std::min(a->page_size, 128) / 8), 1};
      if ((rc = encode_map(x ? &L.tmV : &L.tmK, c.ptr, bf16, dims_w, st_w, box_w, promotion, x ? "v_cache" : "k_cache"))) return rc;
      continue;
    }
    if ((rc = encode_map(x ? &L.tmV : &L.tmK, c.ptr, bf16, dims, st, box, promotion, x ? "v_cache" : "k_cache"))) return rc;
  }
  PagedAttnDev& d = L.p;
  d.T = a->tokens; d.Hq = a->heads_q; d.Hkv = a->heads_kv; d.G = group;
  d.tile_tokens = tile_tokens;
  d.work = a->work;
  d.items_at = work_items_at(sm_count());
  d.block_table = a->block_table;
  d.table_stride = a->table_stride;
  d.table_width = a->table_width;
  d.page_shift = shift;
  d.num_pages = a->pages;
  d.page_groups = by_groups ? static_cast<int>(page_groups) : 0;
  d.page_heads = by_groups ? 0 : a->heads_kv;
  d.scale_log2 = static_cast<float>(a->softmax_scale * 1.4426950408889634);
  L.mod = 0;
  if (a->softcap > 0.f) {
    L.mod |= kModCap;
    d.cap2 = static_cast<float>(a->softcap * 1.4426950408889634);
    d.arg2 = static_cast<float>(2.0 * a->softmax_scale * 1.4426950408889634 / a->softcap);
    if (!std::isfinite(d.arg2)) return fail(FA2_ERR_INVALID_ARG, "softmax_scale / softcap overflows");
  }
  if (a->alibi_slopes) L.mod |= kModSlope;
  d.slopes = a->alibi_slopes;
  d.out = static_cast<uint16_t*>(a->o);
  d.out_st = a->o_stride_t; d.out_sh = a->o_stride_h;
  d.blk = hd.blk;
  d.lse = a->lse;
  d.part_o = static_cast<float*>(a->workspace);
  d.part_lse = d.part_o + static_cast<size_t>(2) * sm_count() * 256 * hd.padded;
  d.status = status_word;
  L.head_dim = hd.padded;
  L.whole_rows = whole_rows;
  L.bf16 = bf16;
  const cudaError_t e = launch_paged_attention(L, static_cast<cudaStream_t>(cuda_stream));
  if (e != cudaSuccess) return fail(FA2_ERR_CUDA, "paged attention launch failed: %s", cudaGetErrorString(e));
  return FA2_OK;
}

}  // extern "C"

namespace fa2 {
namespace {

// fa2_fwd, or with `mod` fa2_scored_fwd.
int fwd_impl(const fa2_fwd_params* a, const fa2_score_mod* mod, void* cuda_stream) {
  if (!a) return fail(FA2_ERR_INVALID_ARG, "params is null");
  const fa2_problem& p = a->p;
  int rc = check_problem(p);
  if (rc) return rc;
  if (!a->q || !a->k || !a->v || !a->o || !a->lse)
    return fail(FA2_ERR_INVALID_ARG, "q, k, v, o and lse must be non-null");
  if (a->lse_stride_h < p.seqlen_q || a->lse_stride_b < 0)
    return fail(FA2_ERR_INVALID_ARG, "lse_stride_h must be at least seqlen_q");
  ScoreModDev mod_dev;
  int mod_mode = 0;
  if (mod) {
    if (a->bias.ptr || a->mask.ptr || a->seqlens || a->dropout_bits)
      return fail(FA2_ERR_UNSUPPORTED, "bias, mask, seqlens and dropout are not supported in attention with changed scores");
    if ((rc = make_score_mod(&mod_dev, &mod_mode, *mod, p))) return rc;
  }
  // First CUDA call of the entry point, on purpose a runtime call: it makes the device's primary
  // context current on a host thread that has not touched the runtime yet (a framework's worker
  // thread served from a memory cache), which the driver-level tensor-map encoder below needs.
  int* const status_word = status_ptr();
  if (!status_word) return fail(FA2_ERR_CUDA, "status word is not addressable");

  FwdLaunch L;
  std::memset(&L, 0, sizeof(L));
  const bool bf16 = p.dtype == FA2_BF16;
  HeadDim hd;
  split_head_dim(p.head_dim, &hd);
  const int D = hd.padded;
  // The problem as the kernel sees it. Decode shape (one query row per head, grouped heads,
  // nothing that depends on the (query, head) position): the G query heads of a key/value head
  // become G query rows of one head through the strides alone, so K and V are streamed once per
  // group instead of once per query head, by one CTA instead of G. A single row sees every key
  // whether the call is causal or not (bottom-right alignment).
  const int group = p.heads_q / p.heads_kv;
  const bool pack_heads = can_pack_heads(p) && !mod && !a->bias.ptr && !a->mask.ptr && !a->seqlens &&
                          a->q_strides.h > 0 && a->o_strides.h > 0;
  int sq_k = p.seqlen_q, hq_k = p.heads_q;
  fa2_strides q_st = a->q_strides, o_st = a->o_strides;
  long long lse_sh = a->lse_stride_h, lse_sq = 1;
  bool causal = p.causal != 0;
  if (pack_heads) {
    sq_k = group;
    hq_k = p.heads_kv;
    q_st.s = a->q_strides.h;  q_st.h = a->q_strides.h * group;
    o_st.s = a->o_strides.h;  o_st.h = a->o_strides.h * group;
    lse_sq = a->lse_stride_h; lse_sh = a->lse_stride_h * group;
    causal = false;
  }
  // Split-KV: the kernel writes per-split partial results into the workspace (as batch elements
  // split * B + b of a contiguous fp32 [n_splits * B, Sq, Hq, kernel head dim] output and its lse),
  // merged afterwards; o itself is written by the merge alone.
  SplitPlan sp = plan_splits(p, hd, pack_heads);
  if (sp.n_splits > 1 && (!a->workspace || a->workspace_bytes < sp.total ||
                          (reinterpret_cast<uintptr_t>(a->workspace) & (kWorkspaceAlign - 1))))
    sp.n_splits = 1;   // not enough scratch: run unsplit
  const bool split = sp.n_splits > 1;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  // head dim 256: K arrives in halves of the head dim, V in halves of the 128 key rows
  if ((rc = make_tmap(&L.tmQ, a->q, bf16, p.batch, sq_k, hq_k, hd, q_st, 128, "q")) ||
      (rc = make_tmap(&L.tmK, a->k, bf16, p.batch, p.seqlen_k, p.heads_kv, hd, a->k_strides, 128, "k",
                      D == 256 ? 4 / kKV256Parts : 0)) ||
      (rc = make_tmap(&L.tmV, a->v, bf16, p.batch, p.seqlen_k, p.heads_kv, hd, a->v_strides,
                      D == 256 ? 128 / kKV256Parts : 128, "v")) ||
      (rc = make_tmap(&L.tmO, a->o, bf16, p.batch, sq_k, hq_k, hd, o_st, 128, "o")) ||
      (rc = make_tmap(&L.tmO1, a->o, bf16, p.batch, sq_k, hq_k, hd, o_st, 128, "o", 1)))
    return rc;

  FwdKernelParams& kp = L.kp;
  kp.B = p.batch; kp.Sq = sq_k; kp.Sk = p.seqlen_k;
  kp.Hq = hq_k; kp.Hkv = p.heads_kv; kp.G = hq_k / p.heads_kv;
  kp.causal_off = p.seqlen_k - sq_k;
  kp.scale_log2 = p.softmax_scale * 1.4426950408889634f;
  kp.lse = a->lse; kp.lse_sb = a->lse_stride_b; kp.lse_sh = lse_sh; kp.lse_sq = lse_sq;
  kp.n_splits = 1;
  kp.split_tiles = 0;
  kp.part_o = nullptr;
  const int sq_pad = (sq_k + 127) / 128 * 128;
  if (split) {
    kp.n_splits = sp.n_splits;
    kp.split_tiles = sp.split_tiles;
    kp.part_o = reinterpret_cast<float*>(ws);
    kp.lse = reinterpret_cast<float*>(ws + sp.part_lse_off);
    kp.lse_sq = 1;
    kp.lse_sh = sq_pad;
    kp.lse_sb = static_cast<long long>(hq_k) * sq_pad;
  }
  if ((rc = make_score_term(&kp.bias, a->bias, p, "bias")) ||
      (rc = make_score_term(&kp.mask, a->mask, p, "mask")))
    return rc;
  make_dropout(&kp.drop, p);
  if (a->seqlens && p.seqlen_q != p.seqlen_k)
    return fail(FA2_ERR_INVALID_ARG, "seqlens requires seqlen_q == seqlen_k");
  if (a->seqlens && (reinterpret_cast<uintptr_t>(a->seqlens) & 3))
    return fail(FA2_ERR_INVALID_ARG, "seqlens must be 4-byte aligned");
  kp.seqlens = a->seqlens;
  if ((rc = set_dropout_operands(&kp.drop, a->dropout_seed_dev, a->offsets_dev))) return rc;
  // (grouped decode rows are only packed without dropout, so the record's row / head indices are
  // always those of the caller's problem)
  if ((rc = set_dropout_bits(&kp.drop, p, a->dropout_bits, a->dropout_bits_bytes))) return rc;
  kp.n_qblk = (sq_k + 255) / 256;
  kp.status = status_word;

  L.head_dim = D;
  L.bf16 = bf16;
  L.causal = causal;
  // The plain path assumes a positive scale (it takes the row maximum before scaling).
  L.feat = kp.bias.ptr || kp.mask.ptr || kp.drop.enabled || !(p.softmax_scale > 0.f);
  if (L.feat && D == 64) {
    // the head-dim-64 kernel streams 16-bit bias / mask tiles through shared memory
    try_stage_term(&L.tmBias, &kp.bias, p, 32);
    try_stage_term(&L.tmMask, &kp.mask, p, 32);
  }

  if (mod) kp.mod = mod_dev;
  cudaError_t e = mod ? launch_fwd_scored(L, mod_mode, static_cast<cudaStream_t>(cuda_stream))
                      : launch_fwd(L, static_cast<cudaStream_t>(cuda_stream));
  if (e != cudaSuccess)
    return fail(FA2_ERR_CUDA, "forward launch failed: %s", cudaGetErrorString(e));
  if (split) {
    FwdCombine c{};
    c.part_o = reinterpret_cast<const float*>(ws);
    c.part_lse = reinterpret_cast<const float*>(ws + sp.part_lse_off);
    c.o = a->o;
    c.o_strides[0] = o_st.b; c.o_strides[1] = o_st.s; c.o_strides[2] = o_st.h;
    c.lse = a->lse;
    c.lse_sb = a->lse_stride_b; c.lse_sh = lse_sh; c.lse_sq = lse_sq;
    c.n_splits = sp.n_splits; c.B = p.batch; c.Sq = sq_k; c.Hq = hq_k; c.D = p.head_dim;
    c.D_part = D;
    c.d_blk = hd.blk;
    c.sq_pad = sq_pad;
    c.bf16 = bf16;
    if (mod) {
      c.rest = mod_dev.rest;
      c.rest_strides[0] = mod_dev.rest_sb; c.rest_strides[1] = mod_dev.rest_ss; c.rest_strides[2] = mod_dev.rest_sh;
    }
    e = launch_fwd_combine(c, static_cast<cudaStream_t>(cuda_stream));
    if (e != cudaSuccess)
      return fail(FA2_ERR_CUDA, "split-KV merge launch failed: %s", cudaGetErrorString(e));
  }
  return FA2_OK;
}

// fa2_bwd, or with `mod` fa2_scored_bwd.
int bwd_impl(const fa2_bwd_params* a, const fa2_score_mod* mod, void* cuda_stream) {
  if (!a) return fail(FA2_ERR_INVALID_ARG, "params is null");
  const fa2_problem& p = a->p;
  int rc = check_problem(p);
  if (rc) return rc;
  if (!a->q || !a->k || !a->v || !a->o || !a->d_o || !a->lse || !a->dq || !a->dk || !a->dv)
    return fail(FA2_ERR_INVALID_ARG, "q, k, v, o, d_o, lse, dq, dk and dv must be non-null");
  if (a->lse_stride_h < p.seqlen_q || a->lse_stride_b < 0)
    return fail(FA2_ERR_INVALID_ARG, "lse_stride_h must be at least seqlen_q");
  const BwdWorkspace w = bwd_workspace(p, mod != nullptr);
  if (!a->workspace || a->workspace_bytes < w.total)
    return fail(FA2_ERR_WORKSPACE, "workspace must hold %zu bytes", w.total);
  if (reinterpret_cast<uintptr_t>(a->workspace) & (kWorkspaceAlign - 1))
    return fail(FA2_ERR_WORKSPACE, "workspace must be 128-byte aligned");
  if (a->dbias.ptr) {
    if (!a->bias.ptr) return fail(FA2_ERR_INVALID_ARG, "dbias is given but bias is not");
    if ((a->dbias.batch != 1 && a->dbias.batch != p.batch) ||
        (a->dbias.heads != 1 && a->dbias.heads != p.heads_kv && a->dbias.heads != p.heads_q))
      return fail(FA2_ERR_INVALID_ARG, "dbias: batch must be 1 or %d and heads 1, %d or %d", p.batch,
                  p.heads_kv, p.heads_q);
    if (reinterpret_cast<uintptr_t>(a->dbias.ptr) & 3)
      return fail(FA2_ERR_INVALID_ARG, "dbias must be 4-byte aligned");
  }

  ScoreModDev mod_dev;
  int mod_mode = 0;
  if (mod) {
    if (a->bias.ptr || a->mask.ptr || a->seqlens || a->dropout_bits || a->dbias.ptr)
      return fail(FA2_ERR_UNSUPPORTED, "bias, mask, seqlens and dropout are not supported in attention with changed scores");
    if ((rc = make_score_mod(&mod_dev, &mod_mode, *mod, p))) return rc;
  }
  // a runtime call before the driver-level tensor-map encoder: see fa2_fwd
  int* const status_word = status_ptr();
  if (!status_word) return fail(FA2_ERR_CUDA, "status word is not addressable");

  BwdLaunch L;
  std::memset(&L, 0, sizeof(L));
  const bool bf16 = p.dtype == FA2_BF16;
  HeadDim hd;
  split_head_dim(p.head_dim, &hd);
  const int D = hd.padded;
  // head dim 256: 64-row query tiles, and dk / dv leave in halves of the head dim
  const int q_rows = (D == 256) ? 64 : 128;
  const int dkv_blocks = (D == 256) ? 2 : D / 64;
  if ((rc = make_tmap(&L.tmQ, a->q, bf16, p.batch, p.seqlen_q, p.heads_q, hd, a->q_strides, q_rows, "q")) ||
      // head dim 256: K is loaded in halves of the head dim (two 64-column blocks per copy)
      (rc = make_tmap(&L.tmK, a->k, bf16, p.batch, p.seqlen_k, p.heads_kv, hd, a->k_strides, 128, "k",
                      D == 256 ? 2 : 0)) ||
      (rc = make_tmap(&L.tmV, a->v, bf16, p.batch, p.seqlen_k, p.heads_kv, hd, a->v_strides, 128, "v")) ||
      (rc = make_tmap(&L.tmdO, a->d_o, bf16, p.batch, p.seqlen_q, p.heads_q, hd, a->do_strides, q_rows, "d_o")) ||
      (rc = make_tmap(&L.tmdK, a->dk, bf16, p.batch, p.seqlen_k, p.heads_kv, hd, a->dk_strides, 128, "dk", dkv_blocks)) ||
      (rc = make_tmap(&L.tmdV, a->dv, bf16, p.batch, p.seqlen_k, p.heads_kv, hd, a->dv_strides, 128, "dv", dkv_blocks)))
    return rc;
  if ((a->o_strides.b % 8) || (a->o_strides.s % 8) || (a->o_strides.h % 8) ||
      (a->dq_strides.b % 8) || (a->dq_strides.s % 8) || (a->dq_strides.h % 8) ||
      (reinterpret_cast<uintptr_t>(a->o) & 15) || (reinterpret_cast<uintptr_t>(a->dq) & 15))
    return fail(FA2_ERR_UNSUPPORTED, "o / dq: 16-byte aligned pointers and strides in multiples of 8 are required");

  BwdKernelParams& kp = L.kp;
  kp.B = p.batch; kp.Sq = p.seqlen_q; kp.Sk = p.seqlen_k;
  kp.Hq = p.heads_q; kp.Hkv = p.heads_kv; kp.G = p.heads_q / p.heads_kv;
  kp.causal_off = p.seqlen_k - p.seqlen_q;
  kp.scale = p.softmax_scale;
  kp.scale_log2 = p.softmax_scale * 1.4426950408889634f;
  kp.lse = a->lse; kp.lse_sb = a->lse_stride_b; kp.lse_sh = a->lse_stride_h;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  kp.delta = reinterpret_cast<float*>(ws + w.delta_off);
  kp.dq_acc = reinterpret_cast<float*>(ws + w.dq_off);
  kp.Sq_pad = w.sq_pad;
  kp.do_absmax_bits = reinterpret_cast<const unsigned*>(ws + w.absmax_off);
  if ((rc = make_score_term(&kp.bias, a->bias, p, "bias")) ||
      (rc = make_score_term(&kp.mask, a->mask, p, "mask")))
    return rc;
  make_dropout(&kp.drop, p);
  if (a->seqlens && p.seqlen_q != p.seqlen_k)
    return fail(FA2_ERR_INVALID_ARG, "seqlens requires seqlen_q == seqlen_k");
  if (a->seqlens && (reinterpret_cast<uintptr_t>(a->seqlens) & 3))
    return fail(FA2_ERR_INVALID_ARG, "seqlens must be 4-byte aligned");
  kp.seqlens = a->seqlens;
  if ((rc = set_dropout_operands(&kp.drop, a->dropout_seed_dev, a->offsets_dev))) return rc;
  if ((rc = set_dropout_bits(&kp.drop, p, a->dropout_bits, a->dropout_bits_bytes))) return rc;
  kp.n_kvblk = (p.seqlen_k + 127) / 128;
  // Launch order (bwd_work_item): causal problems take as many (batch, kv head) groups per chunk as
  // keep a chunk's Q, dO and fp32 dq accumulator tiles within a share of L2; uniform problems keep
  // the group-after-group order.
  kp.sched_groups = 1;
  if (p.causal) {
    const size_t per_group = static_cast<size_t>(kp.G) * p.seqlen_q * D * (2 + 2 + 4);
    const size_t budget = kSchedL2Bytes;
    const long long groups = static_cast<long long>(p.batch) * p.heads_kv;
    kp.sched_groups = static_cast<int>(std::max<long long>(1, std::min<long long>(groups, budget / std::max<size_t>(per_group, 1))));
  }
  kp.status = status_word;

  L.head_dim = D;
  L.bf16 = bf16;
  L.causal = p.causal != 0;
  // (the plain head-dim-128 kernel divides the log-sum-exp by the scale once, in the pre-pass)
  L.feat = kp.bias.ptr || kp.mask.ptr || kp.drop.enabled || !(std::fabs(p.softmax_scale) >= 1e-30f);
  // (a capped score takes no statistics through the MMAs, see bwd_kernel.cuh)
  kp.xstats = (!L.feat && D == 128 && !(mod && has_cap(mod_mode))) ? reinterpret_cast<const uint4*>(ws + w.xstats_off) : nullptr;
  kp.dq_order = a->deterministic ? reinterpret_cast<int*>(ws + w.order_off) : nullptr;
  if (L.feat && D == 64) {
    // the head-dim-64 kernel brings 16-bit bias / mask tiles in through the TMA unit
    try_stage_term(&L.tmBias, &kp.bias, p, 128);
    try_stage_term(&L.tmMask, &kp.mask, p, 128);
  }
  if (a->dbias.ptr) {
    const long long plane = static_cast<long long>(p.seqlen_q) * p.seqlen_k;
    kp.dbias.ptr = a->dbias.ptr;
    kp.dbias.sh = a->dbias.heads == 1 ? 0 : plane;
    kp.dbias.sb = a->dbias.batch == 1 ? 0 : plane * a->dbias.heads;
    kp.dbias.head_div = a->dbias.heads == p.heads_q ? 1 : p.heads_q / p.heads_kv;
    // entries no step touches (above the causal diagonal, behind a batch element's length) stay 0
    const cudaError_t ez = cudaMemsetAsync(a->dbias.ptr, 0, sizeof(float) * plane * a->dbias.heads * a->dbias.batch,
                                           static_cast<cudaStream_t>(cuda_stream));
    if (ez != cudaSuccess)
      return fail(FA2_ERR_CUDA, "clearing dbias failed: %s", cudaGetErrorString(ez));
  }
  L.o = a->o; L.o_strides[0] = a->o_strides.b; L.o_strides[1] = a->o_strides.s; L.o_strides[2] = a->o_strides.h;
  L.d_o = a->d_o; L.do_strides[0] = a->do_strides.b; L.do_strides[1] = a->do_strides.s; L.do_strides[2] = a->do_strides.h;
  L.dq = a->dq; L.dq_strides[0] = a->dq_strides.b; L.dq_strides[1] = a->dq_strides.s; L.dq_strides[2] = a->dq_strides.h;
  L.parts = 1;
  if (w.parts > 1 && a->workspace_bytes >= w.parts_total) {
    L.parts = w.parts;
    kp.part_kv = reinterpret_cast<float*>(ws + w.parts_off);
    L.dk = a->dk; L.dk_strides[0] = a->dk_strides.b; L.dk_strides[1] = a->dk_strides.s; L.dk_strides[2] = a->dk_strides.h;
    L.dv = a->dv; L.dv_strides[0] = a->dv_strides.b; L.dv_strides[1] = a->dv_strides.s; L.dv_strides[2] = a->dv_strides.h;
  }
  L.delta = reinterpret_cast<float*>(ws + w.delta_off);
  L.dq_acc_bytes = w.absmax_off - w.dq_off;
  L.head_dim_real = p.head_dim;
  L.head_blk = hd.blk;

  for (int i = 0; i < 4; ++i) {
    L.stage_events[i] = g_bwd_events[i];
    g_bwd_events[i] = nullptr;   // armed for one call only
  }
  if (mod) kp.mod = mod_dev;
  const cudaError_t e = mod ? launch_bwd_scored(L, mod_mode, static_cast<cudaStream_t>(cuda_stream))
                            : launch_bwd(L, static_cast<cudaStream_t>(cuda_stream));
  if (e != cudaSuccess)
    return fail(FA2_ERR_CUDA, "backward launch failed: %s", cudaGetErrorString(e));
  return FA2_OK;
}

}  // namespace
}  // namespace fa2
