// Attention scores changed by a tanh cap or a distance bias, and masks that leave a query an interval of keys.
//
//   s = softmax_scale * q.k ;   cap:   s <- cap * tanh(s / cap) ;   slopes:  s <- s - slope_h * |i + Sk - Sq - j|
//
// and query i sees key j iff  lo_i <= j < hi_i.  Every mask offered here is such an interval: a causal query sees
// j <= i + Sk - Sq, a prefix of length p raises that end to p, a document [first, end) cuts both ends. The set
// of queries that see a key is an interval for the same reason, so a row of a tile needs two compares at most, and
// whole tiles outside the interval are never loaded.
//
// With t = tanh(s / cap) the derivative of a capped score is 1 - t^2.
#pragma once
#include "kernel_params.cuh"
#include "ptx_sm100.cuh"

namespace fa2 {

// Template argument of the scored kernels: which score changes are compiled in. kNoMod: the plain kernels.
constexpr int kNoMod = -1;
constexpr int kModCap = 1;
constexpr int kModSlope = 2;

constexpr bool has_cap(int mod) { return mod > 0 && (mod & kModCap); }
constexpr bool has_slope(int mod) { return mod > 0 && (mod & kModSlope); }

constexpr float kLog2eMod = 1.4426950408889634f;
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Interval of keys that query row `qi` (< Sq) of batch element `b` sees; empty: hi <= lo.
__device__ __forceinline__ void query_interval(const ScoreModDev& m, int b, int qi, int Sq, int Sk, int causal_off,
                                               int& lo, int& hi) {
  lo = 0;
  hi = Sk;
  if (m.tok_lo != nullptr) {
    const long long at = static_cast<long long>(b) * Sq + qi;
    lo = __ldg(m.tok_lo + at);
    hi = __ldg(m.tok_hi + at);
  }
  if (m.causal) {
    const int prefix = m.prefix_lens != nullptr ? __ldg(m.prefix_lens + b) : 0;
    hi = min(hi, max(qi + causal_off + 1, prefix));
  }
}

// Interval of queries that see key `kj` (< Sk).
__device__ __forceinline__ void key_interval(const ScoreModDev& m, int b, int kj, int Sq, int causal_off, int& lo,
                                             int& hi) {
  lo = 0;
  hi = Sq;
  if (m.tok_lo != nullptr) {
    const long long at = static_cast<long long>(b) * Sq + kj;
    lo = __ldg(m.tok_lo + at);
    hi = __ldg(m.tok_hi + at);
  }
  if (m.causal) {
    const int prefix = m.prefix_lens != nullptr ? __ldg(m.prefix_lens + b) : 0;
    if (kj >= prefix) lo = max(lo, kj - causal_off);
  }
}

// Key tiles [lo, hi) (128 keys each) that some of the 128 query rows of tile `qt` sees; none: lo == hi == 0.
__device__ __forceinline__ void query_tile_range(const ScoreModDev& m, int b, int qt, int Sq, int Sk, int causal_off,
                                                 int& lo, int& hi) {
  const int nq = (Sq + 127) >> 7;
  int first = 0, end = Sk;
  if (qt >= nq) {
    end = 0;
  } else {
    if (m.tile_lo != nullptr) {
      first = __ldg(m.tile_lo + static_cast<long long>(b) * nq + qt);
      end = __ldg(m.tile_hi + static_cast<long long>(b) * nq + qt);
    }
    if (m.causal) {
      const int prefix = m.prefix_lens != nullptr ? __ldg(m.prefix_lens + b) : 0;
      end = min(end, max(min(qt * 128 + 127, Sq - 1) + causal_off + 1, prefix));
    }
  }
  lo = hi = 0;
  if (end > first) {
    lo = first >> 7;
    hi = (end + 127) >> 7;
  }
}

// Query tiles [lo, hi) (kRows rows each) that see some of the 128 keys of tile `kt`; none: lo == hi.
template <int kRows>
__device__ __forceinline__ void key_tile_range(const ScoreModDev& m, int b, int kt, int Sq, int causal_off, int& lo,
                                               int& hi) {
  int first = 0, end = Sq;
  if (m.tile_lo != nullptr) {
    const long long at = static_cast<long long>(b) * ((Sq + 127) >> 7) + kt;
    first = __ldg(m.tile_lo + at);
    end = __ldg(m.tile_hi + at);
  }
  if (m.causal) {
    const int prefix = m.prefix_lens != nullptr ? __ldg(m.prefix_lens + b) : 0;
    if (kt * 128 >= prefix) first = max(first, kt * 128 - causal_off);
  }
  lo = hi = 0;
  if (end > first) {
    lo = first / kRows;
    hi = (end + kRows - 1) / kRows;
  }
}

// Bit-reproducible dq: how many key tiles above `kt` take part in query tile `qt` (kRows rows), by the step rule of
// the main kernels (key_tile_range). Their launch order is descending, so a block waits for earlier blocks alone.
template <int kRows>
__device__ __forceinline__ int key_tiles_above(const ScoreModDev& m, int b, int qt, int kt, int n_kvblk, int Sq,
                                               int causal_off) {
  int count = 0;
  for (int n = kt + 1; n < n_kvblk; ++n) {
    int lo, hi;
    key_tile_range<kRows>(m, b, n, Sq, causal_off, lo, hi);
    if (qt >= lo && qt < hi) ++count;
  }
  return count;
}

// tanh(z) of N values of a row, z = ln2 / 2 * arg2 * x (that is, e^(2z) = 2^(arg2 x)), in place. All 32 lanes call it.
//
// Where every |z| of the warp's values is at most 3/4 (scores well below the cap, which is what a cap is chosen for), it is an
// odd polynomial, z times a polynomial of degree 4 in z^2 that is best in the maximum norm (found by weighted least squares
// repeated until the error levels out): |error| <= 2e-7, fused multiply-adds of pairs alone, with the scale of x in the
// coefficients. Otherwise 1 - 2 r with r = 1 / (1 + 2^(arg2 x)): an exponential and a reciprocal, |error| <= 2^-22. A cap of
// 50 turns either into at most 2^-15 in the exponent of a weight, far below the 2^-9 of the rounding of P; the hardware's
// tanh (2^-11 relative) would move the weights by percents. The special functions are what a capped kernel would be bound by
// otherwise: 16 lanes per cycle and SM, three per score. Measured (2 x 8192 causal, 32/8 heads, D = 128, cap 50): forward
// 1.96 ms with the second form alone, 2.00 with a polynomial in 2^-|arg2 x| instead of the reciprocal, 1.68 with the first
// form up to |z| = 1 (one degree more), 1.55 ms as it is; backward 3.61, 3.84, 3.50, 3.25 ms (3.19 since its tiles are taken
// 32 queries at a time).
constexpr float kSmallTanh = 2.1640425613334453f;   // 1.5 log2(e): |arg2 x| at |z| = 3/4
constexpr float kT0 = 0.9999972283219466f, kT1 = -0.333230764880115f, kT2 = 0.1322609166463934f,
                kT3 = -0.04928044841513475f, kT4 = 0.012318832984223586f;
template <int N>
__device__ __forceinline__ void tanh_row(float (&x)[N], float arg2) {
  float a0 = 0.f, a1 = 0.f;
#pragma unroll
  for (int c = 0; c < N; c += 4) {
    a0 = max3(a0, fabsf(x[c]), fabsf(x[c + 1]));
    a1 = max3(a1, fabsf(x[c + 2]), fabsf(x[c + 3]));
  }
  const float z1 = arg2 * 0.34657359027997264f, z2 = z1 * z1;       // z = z1 x
  // (beyond z1 = 2^13 the last coefficient would leave the range of float32)
  if (z1 < 8192.f && !__any_sync(0xffffffffu, fmaxf(a0, a1) * arg2 > kSmallTanh)) {
    const float c0 = kT0 * z1, c1 = kT1 * (z1 * z2), c2 = kT2 * (z1 * z2 * z2), c3 = kT3 * (z1 * z2 * z2 * z2),
                c4 = kT4 * (z1 * z2 * z2 * (z2 * z2));
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      float u0, u1, t0, t1;
      fma2(u0, u1, x[c], x[c + 1], x[c], x[c + 1], 0.f, 0.f);
      fma2(t0, t1, u0, u1, c4, c4, c3, c3);
      fma2(t0, t1, t0, t1, u0, u1, c2, c2);
      fma2(t0, t1, t0, t1, u0, u1, c1, c1);
      fma2(t0, t1, t0, t1, u0, u1, c0, c0);
      fma2(x[c], x[c + 1], t0, t1, x[c], x[c + 1], 0.f, 0.f);
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      fma2(x[c], x[c + 1], x[c], x[c + 1], arg2, arg2, 0.f, 0.f);
      const float r0 = rcp_approx(1.f + ex2_approx(x[c])), r1 = rcp_approx(1.f + ex2_approx(x[c + 1]));
      fma2(x[c], x[c + 1], r0, r1, -2.f, -2.f, 1.f, 1.f);
    }
  }
}

// The forward's score change of one query row and 128 keys from kv0: x holds the dot products and becomes the scores,
// which the softmax multiplies by `sc` to get units of log2: tanh(s / cap) with sc = cap * log2(e), with slopes alone the
// scores in units of log2 with sc = 1, without either the dot products with sc = softmax_scale * log2(e).
template <int kMod>
struct ModTerms {
  float scale_log2, arg2;
  float slope;      // slope_h * log2(e) / sc
  int qpos;         // position of the query among the keys: i + Sk - Sq
  __device__ __forceinline__ ModTerms(float scale_log2_, float arg2_, float cap2, float slope_h, int qpos_)
      : scale_log2(scale_log2_), arg2(arg2_), slope(slope_h * kLog2eMod), qpos(qpos_) {
    if constexpr (has_cap(kMod)) slope *= 1.f / cap2;
  }
  static __device__ __forceinline__ float sc(float scale_log2, float cap2) {
    return has_cap(kMod) ? cap2 : has_slope(kMod) ? 1.f : scale_log2;
  }
  template <int N>
  __device__ __forceinline__ void operator()(float (&x)[N], int kv0) const {
    if constexpr (has_cap(kMod)) tanh_row(x, arg2);
    if constexpr (has_slope(kMod)) {
      const float mul = has_cap(kMod) ? 1.f : scale_log2;
      const float base = static_cast<float>(kv0 - qpos);
      if (kv0 + N - 1 <= qpos || kv0 >= qpos) {
        // all keys on one side of the query: the bias is linear in the key
        const float s = kv0 >= qpos ? -slope : slope;
        float b0 = base, b1 = base + 1.f;
#pragma unroll
        for (int c = 0; c < N; c += 2) {
          float t0, t1;
          if constexpr (!has_cap(kMod)) fma2(x[c], x[c + 1], x[c], x[c + 1], mul, mul, 0.f, 0.f);
          add2(t0, t1, b0, b1, static_cast<float>(c), static_cast<float>(c));
          fma2(x[c], x[c + 1], t0, t1, s, s, x[c], x[c + 1]);
        }
      } else {
#pragma unroll
        for (int c = 0; c < N; ++c)
          x[c] = fmaf(fabsf(base + static_cast<float>(c)), -slope, x[c] * mul);
      }
    }
  }
};

// The backward's score change of two entries of a key row: s0 and s1 hold the dot products (or, where the row
// statistics are folded into them, the dot products minus lse / scale; with a cap tanh_row's results) and become the
// exponents of P in units of log2, up to the statistics n0 and n1 (-lse * log2(e)); g0 and g1 receive
// d score / d (scale * dot product). d0: position of the first entry's query minus the key's.
template <int kMod>
__device__ __forceinline__ void mod_exponents(float& s0, float& s1, float n0, float n1, float scale_log2, float cap2,
                                              float slope2, float d0, float& g0, float& g1) {
  if constexpr (has_cap(kMod)) {
    fma2(g0, g1, s0, s1, -s0, -s1, 1.f, 1.f);
    fma2(s0, s1, s0, s1, cap2, cap2, n0, n1);
  } else {
    fma2(s0, s1, s0, s1, scale_log2, scale_log2, n0, n1);
  }
  if constexpr (has_slope(kMod)) {
    s0 = fmaf(fabsf(d0), -slope2, s0);
    s1 = fmaf(fabsf(d0 + 1.f), -slope2, s1);
  }
}

}  // namespace fa2
