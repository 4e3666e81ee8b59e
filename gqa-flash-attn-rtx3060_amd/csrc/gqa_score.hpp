// gqa_score.hpp — changed scores (ScoreMod): what the attention kernels' second
// instances, built with FwdModParams or SplitModParams, do between the product
// of queries and keys and the softmax.
//
//   s <- cap tanh(s / cap),  s <- s - slope |p - j|,  visible keys by causal
//   order, a prefix and documents,
//
// p the query's position in key coordinates (row + Skv - Sq), j the key's, all
// in units of the raw product s = q . k: the softmax applies the score scale
// as it does without changes.  A row that sees no key gives zeros and LSE
// -inf here (without changes it gives the reference's 0 / 0 = NaN).
//
// What bounds them is the vector ALU: a plain tile costs a score one exp2 and
// about four further instructions, next to the matrix product it hides.
#pragma once

#include <type_traits>

#include "gqa_common.hpp"
#include "gqa_lds.hpp"
#include "gqa_params.hpp"

namespace gqa {

// Instances with changed scores carry their parameters in a type of their own.
template <typename P> constexpr bool kHasMod = std::is_same<P, FwdModParams>::value || std::is_same<P, SplitModParams>::value;

// The reference point stored with the partial of a row that saw no key: below
// every score (so a real partial of the row outweighs it), finite (so the
// combine of empty partials alone, l = 0, gives zeros).
constexpr float kEmptyRef = -1e30f;

// The scores of one tile in W-wide register vectors.
//
// s <- cap tanh(s / cap) = cap - 2 cap / (1 + 2^(s cap_exp)); the ends follow
// from 1 / (1 + inf) = 0 and 1 / (1 + 0) = 1.
template <int W, typename V, int N>
__device__ __forceinline__ void cap_scores(V (&s)[N], const ScoreMod& m) {
#pragma unroll
  for (int e = 0; e < N * W; ++e) {
    const float x = fast_exp2(s[e / W][e % W] * m.cap_exp);
    s[e / W][e % W] = __builtin_fmaf(-2.f * m.cap, __builtin_amdgcn_rcpf(1.f + x), m.cap);
  }
}

// s <- s - slope |p - j|, slope in raw units; rel: (this lane's first key) - p,
// off(e): the key of value e counted from the lane's first.  `past`
// (wave-uniform): no key of the tile lies behind any row's own position.
template <int W, typename V, int N, typename F>
__device__ __forceinline__ void bias_scores(V (&s)[N], float slope, int rel, bool past, F off) {
  const float r = (float)rel;
  if (past) {
#pragma unroll
    for (int e = 0; e < N * W; ++e) s[e / W][e % W] = __builtin_fmaf(slope, r + (float)off(e), s[e / W][e % W]);
  } else {
#pragma unroll
    for (int e = 0; e < N * W; ++e)
      s[e / W][e % W] = __builtin_fmaf(-slope, __builtin_fabsf(r + (float)off(e)), s[e / W][e % W]);
  }
}

// mask_tile with a first visible key: `lim` and `low` counted from the tile's
// first key, both less 8 for the upper lane half.
__device__ __forceinline__ void mask_tile_span(f32x16 (&s)[2], int lim, int low) {
  const uint32_t n = (uint32_t)max(lim - low, 0);
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int v = 0; v < 16; ++v)
      s[mb][v] = (uint32_t)(32 * mb + key_of(v, 0) - low) >= n ? -__builtin_inff() : s[mb][v];
}

// A query row's slope in raw units (0 without a distance bias), a sequence's
// prefix among its skv keys (0 without one; any value of the caller's comes to
// one in [0, skv], so that sums with it stay in range).
__device__ __forceinline__ float row_slope(const ScoreMod& m, int head) {
  return m.slopes != nullptr ? m.slopes[head] * m.inv_scale : 0.f;
}
__device__ __forceinline__ int seq_prefix(const ScoreMod& m, int b, int skv) {
  return m.prefix != nullptr ? min(max(load_uniform(m.prefix + b), 0), skv) : 0;
}

// Smallest and largest over the wave.
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = min(x, __shfl_xor(x, o, 64));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x = max(x, __shfl_xor(x, o, 64));
  return __builtin_amdgcn_readfirstlane(x);
}

// What a query block of the single pass sees under changed scores: keys [beg,
// end) over its rows (none: beg = end = 0); every row of the wave sees [full_lo,
// full_hi); the lane's own row [lo, vis), both less 8 hh as mask_tile counts
// them; rel0: (8 hh) - its position.
struct RowSpan {
  int beg, end, full_lo, full_hi, lo, vis, rel0;
  int chunk;  // key chunks: the item's
};
// The block's rows are positions [pos_lo, pos_hi] of sequence b (pos_hi at most
// sq - 1, at least pos_lo); the lane's row is `pos`, if `valid`.
__device__ __forceinline__ RowSpan row_span(const ScoreMod& m, const Dims& dm, int b, int skv, int sq, int pos_lo,
                                            int pos_hi, int pos, bool valid, int lane, int hh) {
  RowSpan x;
  const int off = skv - sq, prefix = seq_prefix(m, b, skv);
  const auto end_of = [&](int ps) { return dm.causal ? min(skv, max(ps + off + 1, prefix)) : skv; };
  x.rel0 = 8 * hh - (pos + off);
  x.beg = x.full_lo = 0;
  x.end = max(end_of(pos_hi), 0);
  x.full_hi = end_of(pos_lo);
  x.lo = 0;
  x.vis = end_of(pos);
  if (m.span_lo != nullptr) {  // (sq <= skv)
    const int* ql = m.span_lo + (int64_t)b * dm.Skv + off;
    const int* qh = m.span_hi + (int64_t)b * dm.Skv + off;
    const int row = valid ? pos : pos_lo;
    x.lo = min(max(ql[row], 0), skv);
    x.vis = min(x.vis, valid ? max(qh[row], 0) : 0);
    int first = 0x7fffffff, last = 0;
    for (int ps = pos_lo + lane; ps <= pos_hi; ps += 64) {
      const int l = max(ql[ps], 0), h = min(qh[ps], end_of(ps));
      if (l < h) {
        first = min(first, l);
        last = max(last, h);
      }
    }
    x.end = wave_max(last);
    x.beg = x.end > 0 ? wave_min(first) : 0;
    x.full_lo = wave_max(valid ? x.lo : 0);
    x.full_hi = wave_min(valid ? x.vis : 0x7fffffff);
  }
  x.lo -= 8 * hh;
  x.vis -= 8 * hh;
  return x;
}

}  // namespace gqa
