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

namespace gqa {

namespace {

template <int DT> __device__ inline void unpack8(u32x4 x, float (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = x[i];  // (a value: the builtin reads a vector's element from the vector's start)
    if constexpr (DT == 0) {
      y[2 * i] = __uint_as_float(w << 16);
      y[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
    } else {
      typedef _Float16 f16x2 __attribute__((__vector_size__(2 * sizeof(_Float16))));
      const f16x2 h = __builtin_bit_cast(f16x2, w);
      y[2 * i] = (float)h[0];
      y[2 * i + 1] = (float)h[1];
    }
  }
}
template <int DT> __device__ inline u32x4 pack8(const float (&y)[8]) {
  u32x4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = Elem<DT>::pack2(y[2 * i], y[2 * i + 1]);
  return x;
}

// Sum over the LPR lanes (4 or 8, aligned) that hold a row.
template <int LPR> __device__ inline float row_sum(float x) {
  x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0xB1, 0xF, 0xF, true));  // lane ^ 1
  x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x4E, 0xF, 0xF, true));  // lane ^ 2
  if constexpr (LPR == 8)
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x141, 0xF, 0xF, true));  // 7 - lane
  return x;
}

// Norm weights of this lane's two chunks.
template <int DT>
__device__ inline void load_weights(const void* w, int w32, int ca, int cb, float (&wa)[8], float (&wb)[8]) {
  if (w32) {
    const float* f = static_cast<const float*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      wa[i] = f[8 * ca + i];
      wb[i] = f[8 * cb + i];
    }
  } else {
    const u32x4* x = static_cast<const u32x4*>(w);
    unpack8<DT>(x[ca], wa);
    unpack8<DT>(x[cb], wb);
  }
}

}  // namespace

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
  // This lane's chunks (8 values each): a rotated pair of them, or two behind
  // the rotated dimensions.
  const int rl = p.table != nullptr ? p.R / 16 : 0;  // lanes with rotated chunks
  const bool rot = j < rl;
  const bool apart = rot && !p.interleaved;
  const int ca = apart ? j : 2 * j, cb = apart ? p.R / 16 + j : 2 * j + 1;

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

  // cos and sin of this lane's 8 pairs: of the half form, or 4 of each chunk
  // (interleaved chunks 2 j and 2 j + 1 hold pairs 8 j .. 8 j + 7).
  float cs[8], sn[8];
  int64_t slot = -1;
  if (p.kc.ptr != nullptr) slot = p.slots[tok];
  const auto position = [&](int axis) -> int64_t {
    const int64_t at = (int64_t)axis * p.n_tokens + tok;
    return p.pos64 ? static_cast<const int64_t*>(p.pos)[at] : (int64_t)static_cast<const int*>(p.pos)[at];
  };
  const auto line = [&](int64_t ps) {  // the table's row of a position, in it
    return p.table + (ps < 0 ? 0 : ps < p.max_pos ? ps : p.max_pos - 1) * p.R;
  };
  if (rl > 0) {
    if (p.axes == 1) {
      const int64_t ps = position(0);
      const f32x4* e = reinterpret_cast<const f32x4*>(line(ps)) + 4 * (rot ? j : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 x = e[i];
        cs[2 * i] = x[0], sn[2 * i] = x[1], cs[2 * i + 1] = x[2], sn[2 * i + 1] = x[3];
      }
      if (ps >= p.max_pos)
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = sn[i] = __builtin_nanf("");
    } else {
      const int64_t p0 = position(0), p1 = position(1), p2 = p.axes > 2 ? position(2) : 0,
                    p3 = p.axes > 3 ? position(3) : 0;
      typedef float f32x2 __attribute__((__vector_size__(8)));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = 8 * (rot ? j : 0) + i;
        const int w = pair >> 4;
        const uint32_t word = w == 0   ? p.pair_axis[0]
                              : w == 1 ? p.pair_axis[1]
                              : w == 2 ? p.pair_axis[2]
                                       : p.pair_axis[3];
        const uint32_t axis = (word >> (2 * (pair & 15))) & 3;
        const int64_t ps = axis == 0 ? p0 : axis == 1 ? p1 : axis == 2 ? p2 : p3;
        const f32x2 x = reinterpret_cast<const f32x2*>(line(ps))[pair];
        cs[i] = ps < p.max_pos ? x[0] : __builtin_nanf("");
        sn[i] = ps < p.max_pos ? x[1] : __builtin_nanf("");
      }
    }
  }
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
      const void* w = kind == 0 ? p.wq : p.wk;
      if (w != nullptr) {
        float wa[8], wb[8], ss = 0.f;
        load_weights<DT>(w, p.w32, ca, cb, wa, wb);
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(ya[i], ya[i], __builtin_fmaf(yb[i], yb[i], ss));
        const float inv = 1.0f / __builtin_sqrtf(row_sum<LPR>(ss) * (1.0f / D) + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ya[i] = ya[i] * inv * wa[i];
          yb[i] = yb[i] * inv * wb[i];
        }
      }
      if (rot) {
        if (!p.interleaved) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = ya[i], c = yb[i];
            ya[i] = a * cs[i] - c * sn[i];
            yb[i] = c * cs[i] + a * sn[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = ya[2 * i], c = ya[2 * i + 1];
            ya[2 * i] = a * cs[i] - c * sn[i];
            ya[2 * i + 1] = c * cs[i] + a * sn[i];
            const float d = yb[2 * i], e = yb[2 * i + 1];
            yb[2 * i] = d * cs[4 + i] - e * sn[4 + i];
            yb[2 * i + 1] = e * cs[4 + i] + d * sn[4 + i];
          }
        }
      }
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
