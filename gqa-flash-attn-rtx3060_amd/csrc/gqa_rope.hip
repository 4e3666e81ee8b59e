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
// one token, so its cos and sin stay in registers over the heads.
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
// heads of q, of k or of v.
template <int DT, int D>
__global__ __launch_bounds__(256) void gqa_rope_kernel(RopeParams p) {
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 16, RPW = 64 / LPR;
  const int lane = threadIdx.x & 63;
  const int64_t wid = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wid >= p.n_tokens * p.parts) return;
  const int64_t tok = wid / p.parts;
  const int part = (int)(wid - tok * p.parts);
  const int64_t b = tok / p.S, s = tok - b * p.S;
  const int j = lane % LPR, row = lane / LPR;
  // This lane's chunks (8 values each): a rotated pair of them, or two behind
  // the rotated dimensions.
  const int rl = p.table != nullptr ? p.R / 16 : 0;  // lanes with rotated chunks
  const bool rot = j < rl;
  int ca, cb;
  if (rot && !p.interleaved) {
    ca = j;
    cb = p.R / 16 + j;
  } else {
    ca = 2 * j;
    cb = 2 * j + 1;
  }
  // cos and sin of its pairs: 8 of the half form, or 4 of each chunk.
  float cs[8], sn[8];
  if (rot) {
    const int first = 8 * j;  // (interleaved: chunks 2 j and 2 j + 1 hold pairs 8 j .. 8 j + 7)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int pair = first + i;
      const int axis = p.axes > 1 ? (p.pair_axis[pair >> 4] >> (2 * (pair & 15))) & 3 : 0;
      const int64_t at = (int64_t)axis * p.n_tokens + tok;
      const int64_t ps = p.pos64 ? static_cast<const int64_t*>(p.pos)[at] : (int64_t)static_cast<const int*>(p.pos)[at];
      const int64_t in = ps < 0 ? 0 : (ps < p.max_pos ? ps : p.max_pos - 1);
      const float* e = p.table + (in * (p.R / 2) + pair) * 2;
      cs[i] = ps < p.max_pos ? e[0] : __builtin_nanf("");
      sn[i] = ps < p.max_pos ? e[1] : __builtin_nanf("");
    }
  }
  const int64_t slot = p.kc.ptr != nullptr ? p.slots[tok] : -1;
  const int64_t blk = slot >> p.block_shift, off = slot & ((1 << p.block_shift) - 1);

  const int nq = (p.Hq + RPW - 1) / RPW, nk = p.k.ptr != nullptr ? (p.Hkv + RPW - 1) / RPW : 0;
  const int nv = p.kc.ptr != nullptr ? nk : 0;
  for (int u = part; u < nq + nk + nv; u += p.parts) {
    const int kind = u < nq ? 0 : u < nq + nk ? 1 : 2;
    const int h = (kind == 0 ? u : kind == 1 ? u - nq : u - nq - nk) * RPW + row;
    const bool in = h < (kind == 0 ? p.Hq : p.Hkv);
    const TensorRef& src = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    u32x4 xa = {0u, 0u, 0u, 0u}, xb = xa;
    if (in) {
      const T* r = static_cast<const T*>(src.ptr) + b * src.sb + s * src.ss + (int64_t)h * src.sh;
      xa = *reinterpret_cast<const u32x4*>(r + 8 * ca);
      xb = *reinterpret_cast<const u32x4*>(r + 8 * cb);
    }
    if (kind != 2) {
      float ya[8], yb[8];
      unpack8<DT>(xa, ya);
      unpack8<DT>(xb, yb);
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
      xa = pack8<DT>(ya);
      xb = pack8<DT>(yb);
    }
    if (!in) continue;
    T* o;
    if (kind == 0 || p.kc.ptr == nullptr) {
      const TensorRef& dst = kind == 0 ? p.qo : p.ko;
      o = static_cast<T*>(const_cast<void*>(dst.ptr)) + b * dst.sb + s * dst.ss + (int64_t)h * dst.sh;
    } else {
      if (slot < 0) continue;
      const TensorRef& dst = kind == 1 ? p.kc : p.vc;
      o = static_cast<T*>(const_cast<void*>(dst.ptr)) + blk * dst.sb + off * dst.ss + (int64_t)h * dst.sh;
    }
    *reinterpret_cast<u32x4*>(o + 8 * ca) = xa;
    *reinterpret_cast<u32x4*>(o + 8 * cb) = xb;
  }
}

hipError_t launch_rope(const RopeParams& in, int dtype, hipStream_t stream) {
  RopeParams p = in;
  if (p.n_tokens <= 0) return hipSuccess;
  p.parts = 1;
  const int64_t blocks = (p.n_tokens * p.parts + 3) / 4;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks), block(256);
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
