// gqa_cache8.hip — writes and reads of a paged K/V cache in 8 bits (gqa_cache8.hpp).
//
// Store: new tokens' K and V rows, K normed and rotated on the way (gqa_rope_rows.hpp)
// or as it comes, and with it the queries, as gqa_rope.hip stores 16-bit ones.  A
// page takes one exponent a kv head, the least for its tokens:
//
//   e' = max(e, least e_n with |y| <= 448 2^e_n over the page's new values y),
//
// e counting only if tokens stand in front of the new ones (a page fills from its
// first slot on, so a call that stores that one begins the page anew).  The new
// values become codes of y 2^-e', to the nearest, and where e' > e the tokens in
// front are brought to it: code 2^(e - e'), to the nearest, which is exact but for
// those that fall below 2^-6 2^e'.
//
// A page's new tokens follow one another in the call (sequence-major, as batches
// are), so the workgroup that meets the first of them does the page: a task is (run
// of tokens of one page, K or V, 2^head_shift heads).  Two passes over the run, one
// for the largest value and one for the codes; the second reads from L2.  Nothing is
// ordered by chance: results do not depend on the schedule.
//
// Bound by memory where tokens are many (rows read once from HBM, codes written),
// by the chain of dependent reads (slot, position, table row, exponent) where few.
#include <algorithm>

#include "gqa_cache8.hpp"
#include "gqa_rope_rows.hpp"
#include "gqa_score.hpp"

namespace gqa {

namespace {

// y within +-limit (what a 16-bit value of the rows' type can stand for when
// rounded to a code); NaN stays.
__device__ inline float within(float y, float limit) {
  return __builtin_fabsf(y) > limit ? __builtin_copysignf(limit, y) : y;
}

// Largest over the LPR lanes (4 or 8, aligned) that hold a row.
template <int LPR> __device__ inline float row_max(float x) {
  x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0xB1, 0xF, 0xF, true)));
  x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x4E, 0xF, 0xF, true)));
  if constexpr (LPR == 8)
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x141, 0xF, 0xF, true)));
  return x;
}

__device__ inline int64_t load_uniform64(const int64_t* p) {
  typedef const __attribute__((address_space(4))) int64_t ConstLong;
  return *(ConstLong*)(uintptr_t)p;
}

}  // namespace

// Workgroups [0, n_kv): keys and values; the others: queries, a wave for part of a
// token's heads, as gqa_rope_kernel.
template <int DT, int D> __global__ __launch_bounds__(256) void gqa_store8_kernel(Store8Params p) {
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 16, RPW = 64 / LPR;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const RowLane at = row_lane(p, lane % LPR);

  if ((int)blockIdx.x >= p.n_kv) {
    const int wid = ((int)blockIdx.x - p.n_kv) * 4 + wave;
    const int tok = fast_div(wid, p.div_parts.mul, p.div_parts.shift);
    if (tok >= p.n_tokens) return;
    float cs[8], sn[8];
    if (at.rl > 0) row_angles(p, at, tok, cs, sn);
    const T* qr = static_cast<const T*>(p.q.ptr) + tok * p.q.ss;
    T* qo = static_cast<T*>(const_cast<void*>(p.qo.ptr)) + tok * p.qo.ss;
    for (int h = (wid - tok * p.parts) * RPW + lane / LPR; h - lane / LPR < p.Hq; h += p.parts * RPW) {
      float ya[8] = {}, yb[8] = {};
      if (h < p.Hq) {
        unpack8<DT>(*reinterpret_cast<const u32x4*>(qr + h * p.q.sh + 8 * at.ca), ya);
        unpack8<DT>(*reinterpret_cast<const u32x4*>(qr + h * p.q.sh + 8 * at.cb), yb);
      }
      row_norm_rotate<DT, D>(p, at, p.wq, cs, sn, ya, yb);
      if (h < p.Hq) {
        *reinterpret_cast<u32x4*>(qo + h * p.qo.sh + 8 * at.ca) = pack8<DT>(ya);
        *reinterpret_cast<u32x4*>(qo + h * p.qo.sh + 8 * at.cb) = pack8<DT>(yb);
      }
    }
    return;
  }

  __shared__ int most[64];  // largest |y| of each head, by its bits
  int rest = blockIdx.x;
  const bool is_k = (rest & 1) == 0;
  rest >>= 1;
  const int group = rest % p.n_groups;
  const int t0 = (rest / p.n_groups) * p.chunk, t1 = min(t0 + p.chunk, p.n_tokens);
  const int hg = 1 << p.head_shift, step = (4 * RPW) >> p.head_shift;  // heads; tokens a step
  const int row = wave * RPW + lane / LPR;
  const int h = group * hg + (row & (hg - 1)), first = row >> p.head_shift;
  const bool mine = h < p.Hkv;
  const TensorRef& src = is_k ? p.k : p.v;
  const TensorRef& dst = is_k ? p.kc : p.vc;
  const Exponents& ex = is_k ? p.ke : p.ve;
  const T* rows = static_cast<const T*>(src.ptr) + (mine ? h : 0) * src.sh;

  for (int tok = t0; tok < t1; ++tok) {
    const int64_t slot = load_uniform64(p.slots + tok);
    if (slot < 0) continue;
    const int64_t page = slot >> p.block_shift;
    if (tok > 0) {
      const int64_t before = load_uniform64(p.slots + tok - 1);
      if (before >= 0 && before >> p.block_shift == page) continue;  // not the page's first token
    }
    // The page's tokens from here on, at most a page of them, and their first slot.
    const int bs = 1 << p.block_shift, end = min(p.n_tokens - tok, bs);
    int n = 0, low = bs;
    for (int at0 = 0; at0 < end; at0 += 64) {
      const int64_t s = at0 + lane < end ? p.slots[tok + at0 + lane] : -1;
      const uint64_t other = __builtin_amdgcn_ballot_w64(s < 0 || s >> p.block_shift != page);
      const int here = other == 0 ? 64 : __builtin_ctzll(other);
      low = min(low, wave_min(lane < here ? (int)(s & (bs - 1)) : bs));
      n = at0 + here;
      if (here < 64) break;
    }

    // y of the lane's two chunks of the run's token i.
    const auto values = [&](int i, float (&ya)[8], float (&yb)[8]) __attribute__((always_inline)) {
      const T* x = rows + (int64_t)(tok + i) * src.ss;
      u32x4 xa = {0u, 0u, 0u, 0u}, xb = {0u, 0u, 0u, 0u};
      const bool on = mine && i < n;
      if (on) {
        xa = *reinterpret_cast<const u32x4*>(x + 8 * at.ca);
        xb = *reinterpret_cast<const u32x4*>(x + 8 * at.cb);
      }
      unpack8<DT>(xa, ya);
      unpack8<DT>(xb, yb);
      if (is_k) {
        float cs[8] = {}, sn[8] = {};
        if (at.rl > 0) row_angles(p, at, tok + min(i, n - 1), cs, sn);
        row_norm_rotate<DT, D>(p, at, p.wk, cs, sn, ya, yb);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ya[e] = within(ya[e], p.limit);
        yb[e] = within(yb[e], p.limit);
      }
    };

    __syncthreads();  // (most is free)
    if (threadIdx.x < 64) most[threadIdx.x] = 0;
    __syncthreads();
    float big = 0.f;
    for (int i0 = 0; i0 < n; i0 += step) {
      float ya[8], yb[8];
      values(i0 + first, ya, yb);
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fmaxf(__builtin_fabsf(ya[e]), __builtin_fabsf(yb[e])));
    }
    big = row_max<LPR>(big);
    if (lane % LPR == 0) atomicMax(&most[row & (hg - 1)], __float_as_int(big));
    __syncthreads();

    char* base = static_cast<char*>(const_cast<void*>(dst.ptr)) + page * dst.sb + (mine ? h : 0) * dst.sh;
    int* ep = ex.e + page * ex.sb + (mine ? h : 0) * ex.sh;
    const int was = clamp_exp(*ep);
    int e = exponent_of(__int_as_float(most[row & (hg - 1)]));
    if (low > 0) e = max(e, was);
    __syncthreads();  // (all have read the exponent)
    if (mine && first == 0 && lane % LPR == 0) *ep = e;
    if (mine && low > 0 && e > was) {
      // The tokens in front, brought to the new exponent: 16 codes a lane.
      const float less = exp_scale(max(was - e, kExpMin));
      for (int o = first; o < low; o += step) {
        u32x4* c = reinterpret_cast<u32x4*>(base + (int64_t)o * dst.ss + 16 * (lane % LPR));
        u32x4 x = *c;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w = x[k];
          const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
          const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
          x[k] = codes4(lo[0] * less, lo[1] * less, hi[0] * less, hi[1] * less);
        }
        *c = x;
      }
    }
    const float scale = exp_scale(-e);
    for (int i0 = 0; i0 < n; i0 += step) {
      const int i = i0 + first;
      float ya[8], yb[8];
      values(i, ya, yb);
      if (!mine || i >= n) continue;
      const int64_t o = p.slots[tok + i] & (bs - 1);
      char* c = base + o * dst.ss;
      u32x2 a, b;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        a[k] = codes4(ya[4 * k] * scale, ya[4 * k + 1] * scale, ya[4 * k + 2] * scale, ya[4 * k + 3] * scale);
        b[k] = codes4(yb[4 * k] * scale, yb[4 * k + 1] * scale, yb[4 * k + 2] * scale, yb[4 * k + 3] * scale);
      }
      *reinterpret_cast<u32x2*>(c + 8 * at.ca) = a;
      *reinterpret_cast<u32x2*>(c + 8 * at.cb) = b;
    }
    tok += n - 1;
  }
}

hipError_t launch_store8(const Store8Params& in, int dtype, hipStream_t stream) {
  Store8Params p = in;
  if (p.n_tokens <= 0) return hipSuccess;
  const int rpw = 1024 / p.D;
  // Keys and values.
  p.head_shift = 0;
  while ((1 << p.head_shift) < p.Hkv && (1 << p.head_shift) < rpw) ++p.head_shift;
  p.n_groups = (p.Hkv + (1 << p.head_shift) - 1) >> p.head_shift;
  p.chunk = 1;
  p.n_chunks = (p.n_tokens + p.chunk - 1) / p.chunk;
  const int64_t n_kv = 2ll * p.n_groups * p.n_chunks;
  // Queries: as launch_rope.
  const int units = p.q.ptr != nullptr ? (p.Hq + rpw - 1) / rpw : 0;
  constexpr int kRopeWaves = 4096;
  p.parts = std::max(1, std::min(units, std::max(1, kRopeWaves / p.n_tokens)));
  p.div_parts = make_fast_div((uint32_t)p.parts);
  const int64_t waves = units > 0 ? (int64_t)p.n_tokens * p.parts : 0;
  const int64_t total = n_kv + (waves + 3) / 4;
  if (total >= (int64_t)1 << 31) return hipErrorInvalidValue;
  p.n_kv = (int)n_kv;
  const dim3 grid((unsigned)total), block(256);
  if (dtype == 0) {
    if (p.D == 128) hipLaunchKernelGGL((gqa_store8_kernel<0, 128>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((gqa_store8_kernel<0, 64>), grid, block, 0, stream, p);
  } else {
    if (p.D == 128) hipLaunchKernelGGL((gqa_store8_kernel<1, 128>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((gqa_store8_kernel<1, 64>), grid, block, 0, stream, p);
  }
  return hipGetLastError();
}

// Rows at `slots` as 16-bit values: a thread widens 16 codes of K and the same of V.
// Negative slots give zeros.
template <int DT> __global__ __launch_bounds__(256) void gqa_read8_kernel(Read8Params p) {
  using T = typename Elem<DT>::T;
  const int cpr = p.D / 16;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= (int64_t)p.n_tokens * p.Hkv * cpr) return;
  const int c = (int)(idx % cpr);
  const int64_t th = idx / cpr;
  const int h = (int)(th % p.Hkv);
  const int64_t tok = th / p.Hkv;
  const int64_t slot = p.slots[tok];
  u32x4 k = {0u, 0u, 0u, 0u}, v = {0u, 0u, 0u, 0u};
  float sk = 1.f, sv = 1.f;
  if (slot >= 0) {
    const int64_t page = slot >> p.block_shift, o = slot & ((1 << p.block_shift) - 1);
    k = *reinterpret_cast<const u32x4*>(static_cast<const char*>(p.kc.ptr) + page * p.kc.sb + o * p.kc.ss + h * p.kc.sh + 16 * c);
    v = *reinterpret_cast<const u32x4*>(static_cast<const char*>(p.vc.ptr) + page * p.vc.sb + o * p.vc.ss + h * p.vc.sh + 16 * c);
    sk = exp_scale(clamp_exp(p.ke.e[page * p.ke.sb + h * p.ke.sh]));
    sv = exp_scale(clamp_exp(p.ve.e[page * p.ve.sb + h * p.ve.sh]));
  }
  u32x4* ko = reinterpret_cast<u32x4*>(static_cast<T*>(const_cast<void*>(p.k.ptr)) + tok * p.k.ss + h * p.k.sh + 16 * c);
  u32x4* vo = reinterpret_cast<u32x4*>(static_cast<T*>(const_cast<void*>(p.v.ptr)) + tok * p.v.ss + h * p.v.sh + 16 * c);
  ko[0] = widen8<DT>(k[0], sk, k[1], sk);
  ko[1] = widen8<DT>(k[2], sk, k[3], sk);
  vo[0] = widen8<DT>(v[0], sv, v[1], sv);
  vo[1] = widen8<DT>(v[2], sv, v[3], sv);
}

hipError_t launch_read8(const Read8Params& p, int dtype, hipStream_t stream) {
  const int64_t total = (int64_t)p.n_tokens * p.Hkv * (p.D / 16);
  if (total <= 0) return hipSuccess;
  const int64_t blocks = (total + 255) / 256;
  if (blocks >= (int64_t)1 << 31) return hipErrorInvalidValue;
  if (dtype == 0) hipLaunchKernelGGL(gqa_read8_kernel<0>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(gqa_read8_kernel<1>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace gqa
