// gqa_score.hpp — changed scores (ScoreMod): what gqa_scored.hip, and the other
// attention kernels' second instances, built with FwdModParams or
// SplitModParams, do between the product of queries and keys and the softmax.
//
//   s <- cap tanh(s / cap),  s <- s - slope |p - j|,  visible keys by causal
//   order, a prefix and documents,
//
// p the query's position in key coordinates (row + Skv - Sq), j the key's.  A
// row that sees no key gives zeros and LSE -inf here (without changes it gives
// the reference's 0 / 0 = NaN).
//
// What bounds them is the number of vector instructions a score: three and a
// half without changes (fma, exp2, sum, half a conversion), beside the matrix
// products that they hide.  An instruction more costs 8192 causal tokens (G = 4,
// head_dim 128) about 35 us of 460, exp2 and reciprocals like any other: five
// instructions of a cap in place of the raw score 646 us, a polynomial tanh of
// five and a half 663, the four below 594 (gqa_scored.hip: 925 TFLOP/s, the
// vector unit 67 % busy, the matrix unit 43 %).
//
// So a usual cap takes four, by changing the unit:
//   cap tanh(s / cap) = cap - 2 cap / (1 + exp(2 s / cap))
// is 2 cap times s' = -1 / (1 + 2^(cap_exp s)) plus a constant, which the softmax
// does not see (the log-sum-exp gets it back: shift2); Dims::c is 2 softcap
// log2(e).  A distance bias of keys that no row precedes is one: the row's own
// part, slope (first key - p), goes into the exponent's offset.
#pragma once

#include <type_traits>

#include "gqa_common.hpp"
#include "gqa_lds.hpp"
#include "gqa_params.hpp"

namespace gqa {

// Instances with changed scores carry their parameters in a type of their own.
template <typename P>
constexpr bool kHasMod = std::is_same<P, FwdModParams>::value || std::is_same<P, SplitModParams>::value;

// The reference point stored with the partial of a row that saw no key: below
// every score (so a real partial of the row outweighs it), finite (so the
// combine of empty partials alone, l = 0, gives zeros).
constexpr float kEmptyRef = -1e30f;

// v_max3_f32 of a and the sizes of b and c.
__device__ __forceinline__ float vmax3_abs(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The scores of one tile are in W-wide register vectors (N * W a multiple of 8).
//
// s <- cap tanh(s / cap) for wide caps, where a rounding of the other form, 2^-22
// of the cap, would be lost to scores far below it: s (1 + u P(u)), u = s^2, with the
// cap's powers in P, if all of the wave's tile are within lim3; else score by
// score that polynomial of s / cap up to its end, and cap - 2 cap / (1 + exp(2 s /
// cap)) past it, where 2^-22 of the cap is 2^-20 of the value.  (By the tile's
// largest score alone the second form would take that error to the ordinary rows
// beside a row of large scores: 0.2 at softcap 8e6.)
template <int W, typename V, int N>
__device__ __forceinline__ void wide_cap_scores(V (&s)[N], const ScoreMod& m) {
  constexpr int E = N * W;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < E; e += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      t[k] = vmax3_abs(t[k], s[(e + 2 * k) / W][(e + 2 * k) % W], s[(e + 2 * k + 1) / W][(e + 2 * k + 1) % W]);
  const float mx = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
  if (__builtin_amdgcn_ballot_w64(!(mx <= m.lim3)) == 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x = s[e / W][e % W], u = x * x;
      s[e / W][e % W] = __builtin_fmaf(x * u, __builtin_fmaf(__builtin_fmaf(m.p3[2], u, m.p3[1]), u, m.p3[0]), x);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float x = s[e / W][e % W], y = x * m.inv_cap, u = y * y;
      const float in = __builtin_fmaf(x * u, __builtin_fmaf(__builtin_fmaf(kTanhP[2], u, kTanhP[1]), u, kTanhP[0]), x);
      const float ex = fast_exp2(y * (2.f * kLog2e));
      const float out = __builtin_fmaf(-2.f * m.cap, __builtin_amdgcn_rcpf(1.f + ex), m.cap);
      s[e / W][e % W] = __builtin_fabsf(y) <= kTanhEnd ? in : out;
    }
  }
}

// The cap (the ends of the usual form follow from 1 / (1 + inf) = 0 and 1 / (1 +
// 0) = 1; NaN stays NaN).
template <int W, typename V, int N>
__device__ __forceinline__ void cap_scores(V (&s)[N], const ScoreMod& m) {
  if (m.cap_exp > 0.f) {
#pragma unroll
    for (int e = 0; e < N * W; ++e)
      s[e / W][e % W] = __builtin_amdgcn_rcpf(-1.f - fast_exp2(s[e / W][e % W] * m.cap_exp));
  } else if (m.cap > 0.f) {
    wide_cap_scores<W>(s, m);
  }
}

// score - slope |p - j|; rel: (this lane's first key) - p, off(e): the key of value
// e counted from the lane's first.  Returns what is left to be added to every
// score of the lane: slope rel, if (`past`, wave-uniform) no key of the tile lies
// behind any row's own position, else 0.
template <int W, typename V, int N, typename F>
__device__ __forceinline__ float bias_scores(V (&s)[N], float slope, int rel, bool past, F off) {
  const float r = (float)rel;
  if (past) {
#pragma unroll
    for (int e = 0; e < N * W; ++e) s[e / W][e % W] = __builtin_fmaf(slope, (float)off(e), s[e / W][e % W]);
    return slope * r;
  }
#pragma unroll
  for (int e = 0; e < N * W; ++e)
    s[e / W][e % W] = __builtin_fmaf(-slope, __builtin_fabsf(r + (float)off(e)), s[e / W][e % W]);
  return 0.f;
}

// softmax_rebase (gqa_fwd_parts.hpp) for scores s + t, t the lane's own.
// Returns (t - m_ref) c, the offset of the exponent.
template <int NACC>
__device__ __forceinline__ float softmax_rebase_at(const f32x16 (&s)[2], float t, float& m_ref, float& l_run,
                                                   f32x16 (&acc)[NACC], float c) {
  float a[4] = {s[0][0], s[0][1], s[1][0], s[1][1]};
#pragma unroll
  for (int v = 2; v < 16; v += 4)
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      a[2 * mb] = vmax3(a[2 * mb], s[mb][v], s[mb][v + 1]);
      if (v + 2 < 16) a[2 * mb + 1] = vmax3(a[2 * mb + 1], s[mb][v + 2], s[mb][v + 3]);
    }
  const float mx = xhalf_max(vmax3(vmax3(a[0], a[1], a[2]), a[3], a[3]) + t);
  const float m_new = fmaxf(m_ref, mx);
  const float m_use = (m_new == -__builtin_inff()) ? 0.f : m_new;
  const float alpha = fast_exp2((m_ref - m_use) * c);
  l_run *= alpha;
#pragma unroll
  for (int db = 0; db < NACC; ++db)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[db][v] *= alpha;
  m_ref = m_new;
  return (t - m_use) * c;
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

// Tile order: with a distance bias in causal order the last keys weigh most, so
// the tiles are taken from the last one back and a row's reference point is
// settled by its first tiles, where ascending tiles raise it again and again
// (head slopes 2^-1/4 to 2^-8, 8192 tokens, head_dim 128, in the single pass of
// gqa_fwd.hip's shape: 677 us -> 493).  Place it of n tiles
// from tb on (places past the end stay there: their loads read zeros).
__device__ __forceinline__ int tile_at(int tb, int n, int it, bool back) {
  return tb + (back && it < n ? n - 1 - it : it);
}

// Dealt items (item_of): the pair that takes the place of `bh` among
// the XCD's idx-th items.  An XCD hands its workgroups to its four shader engines
// in turn, whichever of them is free, so a sequence whose place has a period of
// two or four stays on one engine, or two, and the long ones' engines run on while
// the others idle; turned by one place a round it comes to all four.  4 x 256
// tokens over 2000-9000 keys with a cap, in 3 chunks: 184 us -> 128, in 8 180 -> 144;
// documents in 2 x 8192 173 -> 169.5, 4 x 777 with prefixes 42.5 -> 42.
__device__ __forceinline__ int turned_pair(const FwdParams& p, int bh, int idx) {
  if (p.xcd_heads & 1) return bh;  // (it comes to all of them by itself)
  const int x = bh & 7, at = (bh >> 3) + (p.xcd_heads & 2 ? idx >> 1 : idx);
  return (at - fast_div(at, p.div_heads.mul, p.div_heads.shift) * p.xcd_heads) * 8 + x;
}

// A query row's slope in kernel units (0 without a distance bias), a sequence's
// prefix among its skv keys (0 without one; any value of the caller's comes to
// one in [0, skv], so that sums with it stay in range).
__device__ __forceinline__ float row_slope(const ScoreMod& m, int head) {
  return m.slopes != nullptr ? m.slopes[head] * m.unit : 0.f;
}
__device__ __forceinline__ int seq_prefix(const ScoreMod& m, int b, int skv) {
  return m.prefix != nullptr ? min(max(load_uniform(m.prefix + b), 0), skv) : 0;
}

// A row's reference point in log2 units, as partials and the log-sum-exp take it.
template <typename P> __device__ __forceinline__ float log2_ref(const P& p, float m, float c) {
  if constexpr (kHasMod<P>) return __builtin_fmaf(m, c, p.mod.shift2);
  else return m * c;
}

// Smallest and largest over the wave (row shifts, then row broadcasts, into
// lane 63; a lane without a source keeps its own).
__device__ __forceinline__ int wave_min(int x) {
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xF, 0xF, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xF, 0xF, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xF, 0xF, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xF, 0xF, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xA, 0xF, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ int wave_max(int x) { return -wave_min(-x); }

// What a query block of the single pass sees under changed scores: keys [beg,
// end) over its rows (none: beg = end = 0); every row of the wave sees [full_lo,
// full_hi); the lane's own row [lo, vis), both less 8 hh as mask_tile counts
// them; rel0: (8 hh) - its position.
struct RowSpan {
  int beg, end, full_lo, full_hi, lo, vis, rel0;
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
    const int lo = ql[row], hi = qh[row];
    int first = skv, last = 0;
    for (int ps = pos_lo + lane; ps <= pos_hi; ps += 64) {
      const int l = max(ql[ps], 0), h = min(qh[ps], end_of(ps));
      if (l < h) {
        first = min(first, l);
        last = max(last, h);
      }
    }
    x.lo = min(max(lo, 0), skv);
    x.vis = min(x.vis, valid ? max(hi, 0) : 0);
    x.end = wave_max(last);
    x.beg = min(wave_min(first), x.end);
    x.full_lo = wave_max(valid ? x.lo : 0);
    x.full_hi = wave_min(valid ? x.vis : skv);
  }
  x.lo -= 8 * hh;
  x.vis -= 8 * hh;
  return x;
}

}  // namespace gqa
