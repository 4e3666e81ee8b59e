// gqa_rope_rows.hpp — a (token, head) row of queries or keys as gqa_rope.hip and the
// 8-bit cache's writes (gqa_cache8.hip) hold it: D / 16 lanes, 16 values each, as the
// two 8-value chunks whose pairs they rotate; norm and rotation in fp32.
#pragma once

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

// What lane j of a row holds: chunks ca and cb, a rotated pair of them (`rot`), or
// two behind the rotated dimensions.  rl: lanes with rotated chunks.
struct RowLane {
  int j, ca, cb, rl;
  bool rot;
};
__device__ __forceinline__ RowLane row_lane(const RopeParams& p, int j) {
  RowLane x;
  x.j = j;
  x.rl = p.table != nullptr ? p.R / 16 : 0;
  x.rot = j < x.rl;
  const bool apart = x.rot && !p.interleaved;
  x.ca = apart ? j : 2 * j;
  x.cb = apart ? p.R / 16 + j : 2 * j + 1;
  return x;
}

// cos and sin of the lane's 8 pairs at a token's position: of the half form, or 4 of
// each chunk (interleaved chunks 2 j and 2 j + 1 hold pairs 8 j .. 8 j + 7).
__device__ __forceinline__ void row_angles(const RopeParams& p, const RowLane& at, int tok, float (&cs)[8],
                                           float (&sn)[8]) {
  const auto position = [&](int axis) -> int64_t {
    const int64_t at = (int64_t)axis * p.n_tokens + tok;
    return p.pos64 ? static_cast<const int64_t*>(p.pos)[at] : (int64_t)static_cast<const int*>(p.pos)[at];
  };
  const auto line = [&](int64_t ps) {  // the table's row of a position, in it
    return p.table + (ps < 0 ? 0 : ps < p.max_pos ? ps : p.max_pos - 1) * p.R;
  };
  const int first = at.rot ? at.j : 0;
  if (p.axes == 1) {
    const int64_t ps = position(0);
    const f32x4* e = reinterpret_cast<const f32x4*>(line(ps)) + 4 * first;
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
      const int pair = 8 * first + i;
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

// The row's norm (with weights w, or none) and rotation of the lane's two chunks.
// (Which product of a rotation is rounded before the sum is written out, so that every
// kernel gives a row the same bits.)
template <int DT, int D>
__device__ __forceinline__ void row_norm_rotate(const RopeParams& p, const RowLane& at, const void* w,
                                                const float (&cs)[8], const float (&sn)[8], float (&ya)[8],
                                                float (&yb)[8]) {
  if (w != nullptr) {
    float wa[8], wb[8], ss = 0.f;
    load_weights<DT>(w, p.w32, at.ca, at.cb, wa, wb);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(ya[i], ya[i], __builtin_fmaf(yb[i], yb[i], ss));
    const float inv = 1.0f / __builtin_sqrtf(row_sum<D / 16>(ss) * (1.0f / D) + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ya[i] = ya[i] * inv * wa[i];
      yb[i] = yb[i] * inv * wb[i];
    }
  }
  if (at.rot) {
    if (!p.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = ya[i], c = yb[i];
        ya[i] = __builtin_fmaf(a, cs[i], -(c * sn[i]));
        yb[i] = __builtin_fmaf(c, cs[i], a * sn[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = ya[2 * i], c = ya[2 * i + 1];
        ya[2 * i] = __builtin_fmaf(a, cs[i], -(c * sn[i]));
        ya[2 * i + 1] = __builtin_fmaf(a, sn[i], c * cs[i]);
        const float d = yb[2 * i], e = yb[2 * i + 1];
        yb[2 * i] = __builtin_fmaf(d, cs[4 + i], -(e * sn[4 + i]));
        yb[2 * i + 1] = __builtin_fmaf(d, sn[4 + i], e * cs[4 + i]);
      }
    }
  }
}

// The same for a row that becomes e4m3 codes, closer to its exact value than fp32's
// roundings one after another: a value that they move across the middle of two codes is
// off by a whole step, an eighth of it.  1 / rms in 64 bits, as two floats; weighted
// values of 16-bit types are exact; the product that a rotation subtracts keeps its
// rounding error (p + e = c sin).
template <int LPR> __device__ inline double row_sum(double x) {
  const auto from = [&](auto ctrl) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)b, decltype(ctrl)::value, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(b >> 32), decltype(ctrl)::value, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  x += from(std::integral_constant<int, 0xB1>{});
  x += from(std::integral_constant<int, 0x4E>{});
  if constexpr (LPR == 8) x += from(std::integral_constant<int, 0x141>{});
  return x;
}
template <int DT, int D>
__device__ __forceinline__ void row_norm_rotate_closely(const RopeParams& p, const RowLane& at, const void* w,
                                                        const float (&cs)[8], const float (&sn)[8], float (&ya)[8],
                                                        float (&yb)[8]) {
  float hi = 1.f, lo = 0.f;
  if (w != nullptr) {
    float wa[8], wb[8];
    double ss = 0.0;
    load_weights<DT>(w, p.w32, at.ca, at.cb, wa, wb);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      ss = __builtin_fma((double)ya[i], (double)ya[i], __builtin_fma((double)yb[i], (double)yb[i], ss));
    // Rows are brought to a size about 1 by 2^-h before the weights, whose products then
    // stay within fp32 whatever the row's size (64 tokens 4.62 -> 4.67 us, 8192 as they were).
    const double x = row_sum<D / 16>(ss) * (1.0 / D) + (double)p.eps, r = __builtin_amdgcn_rsq(x);
    const int h = max(min((__builtin_amdgcn_frexp_exp(x) + 1) >> 1, 126), -126);
    // (The instruction's 2^-23, then a step of Newton's; infinite rows: 0.)
    const double inv = __builtin_ldexp(x < __builtin_inf() ? r * (1.5 - 0.5 * x * r * r) : r, h);
    hi = (float)inv;
    lo = (float)(inv - (double)hi);
    const float less = __builtin_ldexpf(1.f, -h);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ya[i] = ya[i] * less * wa[i];
      yb[i] = yb[i] * less * wb[i];
    }
  }
  const auto minus = [](float a, float co, float c, float si) __attribute__((always_inline)) {  // a co - c si
    const float q = c * si, e = __builtin_fmaf(c, si, -q);
    return __builtin_fmaf(a, co, -q) - (e == e ? e : 0.f);  // (infinite products have no error term)
  };
  const auto turn = [&](float& a, float& c, float co, float si) __attribute__((always_inline)) {
    const float x = minus(a, co, c, si);
    c = minus(c, co, a, -si);
    a = x;
  };
  if (at.rot) {
    if (!p.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) turn(ya[i], yb[i], cs[i], sn[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        turn(ya[2 * i], ya[2 * i + 1], cs[i], sn[i]);
        turn(yb[2 * i], yb[2 * i + 1], cs[4 + i], sn[4 + i]);
      }
    }
  }
  if (w != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ya[i] = __builtin_fmaf(ya[i], hi, ya[i] * lo);
      yb[i] = __builtin_fmaf(yb[i], hi, yb[i] * lo);
    }
  }
}

}  // namespace

}  // namespace gqa
