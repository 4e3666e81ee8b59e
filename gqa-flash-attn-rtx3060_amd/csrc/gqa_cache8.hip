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
// of tokens of one page, K or V, 2^head_shift heads).  One pass over the run finds its
// largest value, one makes the codes: of values still in registers if the run is one
// step (32 (token, head) rows at head_dim 128, 64 at 64), else from L2.
// Nothing is ordered by chance: results do not depend on the schedule.
//
// Measured, bf16, 32/8 heads of 128, 16-token pages: norms, rotation and store of 8192
// tokens 52 us, 189 MB at 3.6 TB/s (a large copy 5.1; registers for four waves a
// SIMD are what keeps it from more: the rotation of 16-bit caches alone, at six, 49.5
// us for 206 MB); K and V alone 14.0 us, 51 MB.  64 tokens, one a page: 4.7 and 3.7
// us, a chain of dependent reads (slot; exponent, table row) after a launch of 2.6.
// Rows and angles of a small call's tokens are loaded before their slots are known.
#include <algorithm>

#include "gqa_cache8.hpp"
#include "gqa_lds.hpp"
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
// token's heads, as gqa_rope_kernel.  ROPE: keys are normed or rotated, and there may
// be queries; without, half the registers.
template <int DT, int D, bool ROPE> __global__ __launch_bounds__(256) void gqa_store8_kernel(Store8Params p) {
  using T = typename Elem<DT>::T;
  constexpr int LPR = D / 16, RPW = 64 / LPR;
  const int lane = threadIdx.x & 63;
  constexpr int waves = 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const RowLane at = row_lane(p, lane % LPR);

  if (ROPE && (int)blockIdx.x >= p.n_kv) {
    const int wid = ((int)blockIdx.x - p.n_kv) * waves + wave;
    const int tok = fast_div(wid, p.div_parts.mul, p.div_parts.shift);
    if (tok >= p.n_tokens) return;
    const T* qr = static_cast<const T*>(p.q.ptr) + tok * p.q.ss;
    T* qo = static_cast<T*>(const_cast<void*>(p.qo.ptr)) + tok * p.qo.ss;
    // The next heads' rows are loaded while these are worked on.
    const int turn = p.parts * RPW, h0 = (wid - tok * p.parts) * RPW, row = lane / LPR;
    u32x4 xa, xb;
    const auto fetch = [&](int h) {
      xa = xb = u32x4{0u, 0u, 0u, 0u};
      if (h < p.Hq) {
        xa = *reinterpret_cast<const u32x4*>(qr + h * p.q.sh + 8 * at.ca);
        xb = *reinterpret_cast<const u32x4*>(qr + h * p.q.sh + 8 * at.cb);
      }
    };
    fetch(h0 + row);
    float cs[8], sn[8];
    if (at.rl > 0) row_angles(p, at, tok, cs, sn);
    for (int hw = h0; hw < p.Hq; hw += turn) {
      const int h = hw + row;
      float ya[8], yb[8];
      unpack8<DT>(xa, ya);
      unpack8<DT>(xb, yb);
      fetch(h + turn);
      row_norm_rotate<DT, D>(p, at, p.wq, cs, sn, ya, yb);
      if (h < p.Hq) {
        *reinterpret_cast<u32x4*>(qo + h * p.qo.sh + 8 * at.ca) = pack8<DT>(ya);
        *reinterpret_cast<u32x4*>(qo + h * p.qo.sh + 8 * at.cb) = pack8<DT>(yb);
      }
    }
    return;
  }

  __shared__ int most[64];  // largest |y| of each head, by its bits
  // (Tasks with work may be every block_size-th of them: dealt as the hardware deals
  // workgroups, they would all be on one or two XCDs.)
  int rest = xcd_remap(blockIdx.x, p.n_kv);
  const bool is_k = (rest & 1) == 0;
  rest >>= 1;
  const int group = rest % p.n_groups;
  const int t0 = (rest / p.n_groups) * p.chunk, t1 = min(t0 + p.chunk, p.n_tokens);
  const int hg = 1 << p.head_shift, step = (waves * RPW) >> p.head_shift;  // heads; tokens a step
  const int row = wave * RPW + lane / LPR;
  const int h = group * hg + (row & (hg - 1)), first = row >> p.head_shift;
  const bool mine = h < p.Hkv;
  const TensorRef& src = is_k ? p.k : p.v;
  const TensorRef& dst = is_k ? p.kc : p.vc;
  const Exponents& ex = is_k ? p.ke : p.ve;
  const T* rows = static_cast<const T*>(src.ptr) + (mine ? h : 0) * src.sh;
  const int bs = 1 << p.block_shift;

  // y of the lane's two chunks of token tok (`on`: it has one).
  const auto fetch = [&](int tok, bool on, u32x4& xa, u32x4& xb) __attribute__((always_inline)) {
    xa = xb = u32x4{0u, 0u, 0u, 0u};
    if (on) {
      const T* x = rows + (int64_t)tok * src.ss;
      xa = *reinterpret_cast<const u32x4*>(x + 8 * at.ca);
      xb = *reinterpret_cast<const u32x4*>(x + 8 * at.cb);
    }
  };
  const auto angles = [&](int tok, float (&cs)[8], float (&sn)[8]) __attribute__((always_inline)) {
    if constexpr (ROPE) {
      if (is_k && at.rl > 0) row_angles(p, at, tok, cs, sn);
    }
  };
  const auto finish = [&](const u32x4& xa, const u32x4& xb, const float (&cs)[8], const float (&sn)[8], float (&ya)[8],
                          float (&yb)[8]) __attribute__((always_inline)) {
    unpack8<DT>(xa, ya);
    unpack8<DT>(xb, yb);
    if constexpr (ROPE) {
      if (is_k) row_norm_rotate_closely<DT, D>(p, at, p.wk, cs, sn, ya, yb);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ya[e] = within(ya[e], p.limit);
      yb[e] = within(yb[e], p.limit);
    }
  };

  // Lane l: token t0 + l, its page (none: -1) and the slot in it.
  const int left = min(64, p.n_tokens - t0);
  const int64_t slot = lane < left ? p.slots[t0 + lane] : -1;
  const int64_t before = t0 > 0 ? load_uniform64(p.slots + t0 - 1) : -1;
  // (The first token's rows and angles, which a decode step's task is about, with
  // them.)
  u32x4 xa, xb;
  float cs[8] = {}, sn[8] = {};
  if (p.chunk == 1) {
    fetch(t0 + first, mine && first < left, xa, xb);
    angles(t0 + min(first, left - 1), cs, sn);
  }
  if (threadIdx.x < 64) most[threadIdx.x] = 0;
  const int page_of = slot < 0 ? -1 : (int)(slot >> p.block_shift), off_of = (int)(slot & (bs - 1));
  const int front = __shfl_up(page_of, 1);
  const int prev = lane > 0 ? front : before < 0 ? -1 : (int)(before >> p.block_shift);
  uint64_t owners = __builtin_amdgcn_ballot_w64(lane < t1 - t0 && page_of >= 0 && page_of != prev);
  while (owners != 0) {
    const int j = __builtin_ctzll(owners), tok = t0 + j;
    owners &= owners - 1;
    const int page = __builtin_amdgcn_readlane(page_of, j);
    // The page's tokens from here on, n of them, and their first slot.
    const uint64_t same = __builtin_amdgcn_ballot_w64(page_of == page) >> j;
    int n = same == ~0ull ? 64 : __builtin_ctzll(~same);
    int low = wave_min(lane >= j && lane < j + n ? off_of : bs);
    for (int more = 64; j + n == more && t0 + more < p.n_tokens; more += 64) {
      const int64_t s = t0 + more + lane < p.n_tokens ? p.slots[t0 + more + lane] : -1;
      const uint64_t other = __builtin_amdgcn_ballot_w64(s < 0 || (int)(s >> p.block_shift) != page);
      const int here = other == 0 ? 64 : __builtin_ctzll(other);
      low = min(low, wave_min(lane < here ? (int)(s & (bs - 1)) : bs));
      n += here;
      if (here < 64) break;
    }
    n = min(n, bs);

    char* base = static_cast<char*>(const_cast<void*>(dst.ptr)) + page * dst.sb + (mine ? h : 0) * dst.sh;
    int* ep = ex.e + page * ex.sb + (mine ? h : 0) * ex.sh;
    int was = clamp_exp(*ep);
    float big = 0.f, ya[8], yb[8];
    for (int i0 = 0; i0 < n; i0 += step) {
      if (p.chunk > 1 || i0 > 0) {
        const int i = i0 + first;
        fetch(tok + i, mine && i < n, xa, xb);
        angles(tok + min(i, n - 1), cs, sn);
      } else if (first >= n) {
        xa = xb = u32x4{0u, 0u, 0u, 0u};
      }
      finish(xa, xb, cs, sn, ya, yb);
#pragma unroll
      for (int e = 0; e < 8; ++e) big = fmaxf(big, fmaxf(__builtin_fabsf(ya[e]), __builtin_fabsf(yb[e])));
    }
    big = row_max<LPR>(big);
    pin(was);
    // (Barriers of LDS alone: loads and stores stay in flight.)
    phase_barrier();  // most is zero, and all have read the exponent
    if (lane % LPR == 0) atomicMax(&most[row & (hg - 1)], __float_as_int(big));
    phase_barrier();
    int e = exponent_of(__int_as_float(most[row & (hg - 1)]));
    if (owners != 0) {  // (for the next page)
      phase_barrier();
      if (threadIdx.x < 64) most[threadIdx.x] = 0;
    }
    if (low > 0) e = max(e, was);
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
      if (n > step) {  // (else y is there)
        fetch(tok + i, mine && i < n, xa, xb);
        angles(tok + min(i, n - 1), cs, sn);
        finish(xa, xb, cs, sn, ya, yb);
      }
      int o = __shfl(off_of, (j + i) & 63);
      if (!mine || i >= n) continue;
      if (j + i >= 64) o = (int)(p.slots[tok + i] & (bs - 1));
      char* c = base + (int64_t)o * dst.ss;
      u32x2 a, b;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        a[k] = codes4(ya[4 * k] * scale, ya[4 * k + 1] * scale, ya[4 * k + 2] * scale, ya[4 * k + 3] * scale);
        b[k] = codes4(yb[4 * k] * scale, yb[4 * k + 1] * scale, yb[4 * k + 2] * scale, yb[4 * k + 3] * scale);
      }
      *reinterpret_cast<u32x2*>(c + 8 * at.ca) = a;
      *reinterpret_cast<u32x2*>(c + 8 * at.cb) = b;
    }
  }
}

template <int DT, int D> static void launch_store8_t(const Store8Params& p, int64_t total, hipStream_t stream) {
  const dim3 grid((unsigned)total), block(256);
  if (p.q.ptr != nullptr || p.table != nullptr || p.wk != nullptr)
    hipLaunchKernelGGL((gqa_store8_kernel<DT, D, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((gqa_store8_kernel<DT, D, false>), grid, block, 0, stream, p);
}

hipError_t launch_store8(const Store8Params& in, int dtype, hipStream_t stream) {
  Store8Params p = in;
  if (p.n_tokens <= 0) return hipSuccess;
  const int rpw = 1024 / p.D;
  // Keys and values.
  p.head_shift = 0;
  while ((1 << p.head_shift) < p.Hkv && (1 << p.head_shift) < rpw) ++p.head_shift;
  // A wave's worth of heads a workgroup, fewer where a page's tokens then go in one
  // step: a prompt's pages (us, K and V alone, 8 kv heads of 128, a wave's heads / fewer,
  // pages of 16, 64, 256: 400 tokens 10.8 / 4.0, 18 / 5.4, 65 / 12; 8192 tokens 15.4 /
  // 13.8, 38 / 15.5, 141 / 25).  Not in small calls of more than a few tokens, which
  // may be a token of each of many pages: more workgroups for the same rows (64 with
  // norms and queries 4.4 / 5.0, 256 in pages of 64 4.0 / 7.5; a prompt of 100 pays
  // 6.8 for 4.9).
  const int bs = 1 << p.block_shift;
  const auto groups = [&] { return (p.Hkv + (1 << p.head_shift) - 1) >> p.head_shift; };
  while (p.head_shift > 0 && ((4 * rpw) >> p.head_shift) < bs &&
         (p.n_tokens > 256 || p.n_tokens * groups() <= 32))
    --p.head_shift;
  p.n_groups = groups();
  // Tokens that a workgroup looks at, up to a page of 16-64: a workgroup that finds no
  // page's first token costs as much as one that does (8192 tokens in pages of 16, 4 a
  // workgroup 20 us, 16 15), while 512 still fill the device.
  p.chunk = std::max(1, std::min(std::min(std::max(bs, 16), 64), (int)(2ll * p.n_groups * p.n_tokens / 512)));
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
  if (dtype == 0) {
    if (p.D == 128) launch_store8_t<0, 128>(p, total, stream);
    else launch_store8_t<0, 64>(p, total, stream);
  } else {
    if (p.D == 128) launch_store8_t<1, 128>(p, total, stream);
    else launch_store8_t<1, 64>(p, total, stream);
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
    const auto codes = [&](const TensorRef& t) {
      return static_cast<const char*>(t.ptr) + page * t.sb + o * t.ss + h * t.sh + 16 * c;
    };
    k = *reinterpret_cast<const u32x4*>(codes(p.kc));
    v = *reinterpret_cast<const u32x4*>(codes(p.vc));
    sk = exp_scale(clamp_exp(p.ke.e[page * p.ke.sb + h * p.ke.sh]));
    sv = exp_scale(clamp_exp(p.ve.e[page * p.ve.sb + h * p.ve.sh]));
  }
  const auto row = [&](const TensorRef& t) {
    return reinterpret_cast<u32x4*>(static_cast<T*>(const_cast<void*>(t.ptr)) + tok * t.ss + h * t.sh + 16 * c);
  };
  u32x4 *ko = row(p.k), *vo = row(p.v);
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
