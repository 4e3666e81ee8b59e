// gqa_rope.hip — per-head norms of queries and keys and the rotation of their
// positions, in one pass between the projection and the attention; optionally
// with K and V stored at their slots of a paged cache in the same pass.
//
//   y = x rsqrt(mean(x^2) + eps) w            (fp32; without weights y = x)
//   (y_a, y_b) <- (y_a cos t - y_b sin t, y_b cos t + y_a sin t),
//   t = position[axis(i)] inv_freq(i) for pair i = (a, b) < R / 2, pairs (i, i +
//   R / 2) or (2 i, 2 i + 1); dimensions from R on are not rotated
//
// all in fp32 and rounded once.  cos and sin come from a table computed in
// fp64 (an angle of position 131072 has no fraction left in fp32).
//
// Bound by memory: q, k (and v) are read once and written once.  D / 16 lanes
// hold a (token, head) row, 16 values each, as the two 8-value chunks whose
// pairs they rotate: no exchange but the sum of squares.  A wave takes rows of
// one token, so its cos and sin stay in registers over the heads.  Measured, bf16,
// head_dim 128, 32/8 heads: 16384 tokens 72.4 us, 4.64 TB/s (a large copy reaches
// 4.9-5.0); 5003 tokens of three axes into a paged cache 27.2 us, 4.53 TB/s; 64
// tokens into it 3.2 us, bound by two dependent reads (position, table row), with
// a token's rows over as many waves as 4096 allow.  A wave a token with its loads
// where they are used: 87.5 and 9.3 us for the first and the last.
#include <algorithm>
#include <type_traits>

#include "gqa_common.hpp"
#include "gqa_params.hpp"
#include "gqa_rope_rows.hpp"

namespace gqa {

// Wave: token, and units part, part + parts, ... of its rows; a unit is RPW
// heads of q, of k or of v.  The next unit's rows are loaded while one is worked
// on.
template <int DT, int D>
__global__ __launch_bounds__(256) void gqa_rope_kernel(RopeParams p) {
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 16, RPW = 64 / LPR;
  const int lane = threadIdx.x & 63;
  const int wid = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tok = fast_div(wid, p.div_parts.mul, p.div_parts.shift);
  if (tok >= p.n_tokens) return;
  const int part = wid - tok * p.parts;
  const int b = fast_div(tok, p.div_s.mul, p.div_s.shift), s = tok - b * p.S;
  const int j = lane % LPR, row = lane / LPR;
  const RowLane at = row_lane(p, j);
  const int ca = at.ca, cb = at.cb;

  const int nq = (p.Hq + RPW - 1) / RPW, nk = p.k.ptr != nullptr ? (p.Hkv + RPW - 1) / RPW : 0;
  const int units = nq + nk + (p.kc.ptr != nullptr ? nk : 0);
  const T* qr = static_cast<const T*>(p.q.ptr) + b * p.q.sb + s * p.q.ss;
  const T* kr = static_cast<const T*>(p.k.ptr) + b * p.k.sb + s * p.k.ss;
  const T* vr = static_cast<const T*>(p.v.ptr) + b * p.v.sb + s * p.v.ss;
  u32x4 xa, xb;
  const auto fetch = [&](int u) {
    const int kind = u < nq ? 0 : u < nq + nk ? 1 : 2;
    const int h = (kind == 0 ? u : kind == 1 ? u - nq : u - nq - nk) * RPW + row;
    const T* r = kind == 0 ? qr + h * p.q.sh : kind == 1 ? kr + h * p.k.sh : vr + h * p.v.sh;
    xa = xb = u32x4{0u, 0u, 0u, 0u};
    if (u < units && h < (kind == 0 ? p.Hq : p.Hkv)) {
      xa = *reinterpret_cast<const u32x4*>(r + 8 * ca);
      xb = *reinterpret_cast<const u32x4*>(r + 8 * cb);
    }
  };
  fetch(part);

  float cs[8], sn[8];
  int64_t slot = -1;
  if (p.kc.ptr != nullptr) slot = p.slots[tok];
  if (at.rl > 0) row_angles(p, at, tok, cs, sn);
  const int64_t blk = slot >> p.block_shift, off = slot & ((1 << p.block_shift) - 1);

  for (int u = part; u < units; u += p.parts) {
    const int kind = u < nq ? 0 : u < nq + nk ? 1 : 2;
    const int h = (kind == 0 ? u : kind == 1 ? u - nq : u - nq - nk) * RPW + row;
    u32x4 oa = xa, ob = xb;
    fetch(u + p.parts);
    if (kind != 2) {
      float ya[8], yb[8];
      unpack8<DT>(oa, ya);
      unpack8<DT>(ob, yb);
      row_norm_rotate<DT, D>(p, at, kind == 0 ? p.wq : p.wk, cs, sn, ya, yb);
      oa = pack8<DT>(ya);
      ob = pack8<DT>(yb);
    }
    const bool cached = kind != 0 && p.kc.ptr != nullptr;
    if (h >= (kind == 0 ? p.Hq : p.Hkv) || (cached && slot < 0)) continue;
    T* o;
    if (cached) {
      const TensorRef& dst = kind == 1 ? p.kc : p.vc;
      o = static_cast<T*>(const_cast<void*>(dst.ptr)) + blk * dst.sb + off * dst.ss + (int64_t)h * dst.sh;
    } else {
      const TensorRef& dst = kind == 0 ? p.qo : p.ko;
      o = static_cast<T*>(const_cast<void*>(dst.ptr)) + b * dst.sb + s * dst.ss + (int64_t)h * dst.sh;
    }
    *reinterpret_cast<u32x4*>(o + 8 * ca) = oa;
    *reinterpret_cast<u32x4*>(o + 8 * cb) = ob;
  }
}

hipError_t launch_rope(const RopeParams& in, int dtype, hipStream_t stream) {
  RopeParams p = in;
  if (p.n_tokens <= 0) return hipSuccess;
  // Few tokens: their rows over more waves, up to kRopeWaves in all.
  const int rpw = 1024 / p.D, nk = p.k.ptr != nullptr ? (p.Hkv + rpw - 1) / rpw : 0;
  const int units = (p.Hq + rpw - 1) / rpw + nk + (p.kc.ptr != nullptr ? nk : 0);
  constexpr int kRopeWaves = 4096;
  p.parts = std::min(units, std::max(1, kRopeWaves / p.n_tokens));
  p.div_parts = make_fast_div((uint32_t)p.parts);
  p.div_s = make_fast_div((uint32_t)p.S);
  const int64_t waves = (int64_t)p.n_tokens * p.parts;
  const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
  if (dtype == 0) {
    if (p.D == 128) hipLaunchKernelGGL((gqa_rope_kernel<0, 128>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((gqa_rope_kernel<0, 64>), grid, block, 0, stream, p);
  } else {
    if (p.D == 128) hipLaunchKernelGGL((gqa_rope_kernel<1, 128>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((gqa_rope_kernel<1, 64>), grid, block, 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace gqa
