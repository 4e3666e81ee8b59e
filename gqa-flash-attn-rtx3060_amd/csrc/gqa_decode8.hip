// gqa_decode8.hip — attention over a paged cache in 8 bits (gqa_cache8.hpp) for few
// query rows: single tokens, and as many as give 16 packed rows per kv head (row r ->
// position r / G, head r % G).
//
//   s_j = scale q . (kc_j 2^ke(page of j)),  o = sum_j p_j (vc_j 2^ve(page of j)) / l
//
// with the online softmax, changed scores and partials of the 16-bit passes
// (gqa_decode_kernel.hpp, gqa_score.hpp).  Codes are widened to the queries' type
// with their page's power of two on the way into the matrix instructions (exact),
// scores, sums and accumulators are fp32, P is rounded to the queries' type.
//
// What bounds it is the read of the cache, half the bytes of 16 bits, so each byte
// has twice the arithmetic of the 16-bit pass.  There the four waves of a workgroup
// share a tile, wait for each other twice a tile, and each computes all scores of it;
// here a wave is on its own: it takes every fourth tile of TW keys (4 KiB of K and
// of V), all of its scores and all head dimensions, loads tiles into LDS of its own
// two ahead, and meets the others once a piece, in LDS.  No barrier within the
// stream, no score computed twice.
//
// The keys of all sequences are cut into equal ranges, one a workgroup, on the
// device (gqa_flat.hpp), in units of four tiles.
#include <algorithm>

#include "gqa_cache8.hpp"
#include "gqa_decode_kernel.hpp"
#include "gqa_lds.hpp"

namespace gqa {

namespace {

// This wave's memory operations: all but n of its loads into LDS done, and its LDS
// reads; nothing moves across.
template <int IMM> __device__ inline void wave_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(IMM);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

typedef int v2i32 __attribute__((__vector_size__(2 * sizeof(int))));
typedef __attribute__((address_space(3))) v2i32 lds_v2i32;
// In each 16-lane group lane j addresses 8 bytes of row j / 2 (bytes 8 (j % 2) ..)
// and receives byte j of the 8 rows.
__device__ inline u32x2 ld_tr8(const char* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i32*)(p)));
}

}  // namespace

// Lane (i16 = l % 16, lg = l / 16).  S^T of a 16-key block: A = its K rows, lane
// (i16, lg) holds dims (D / 4) lg + 8 ks + 0..7 of row i16 for k-step ks, so that its
// codes are consecutive (Q^T in the same order).  Register v of block kb holds key
// 16 kb + 4 lg + v of query row i16.  O^T += V^T P^T over 32 keys: k-slots 8 lg + e are
// keys 4 lg + e and 16 + 4 lg + (e - 4), the lane's own probabilities; V^T is read
// transposed, 8 rows of one dim a read.  The chunks of a row are swizzled so that the
// 16 lanes of a K read, and the 32 of a V read, cover all banks once: fk, fv below.
template <int DT, int D, bool MOD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void gqa_decode8_kernel(Split8Params p) {
  using E = Elem<DT>;
  constexpr int TW = 4096 / D;     // keys of a wave's tile
  constexpr int NB = TW / 16;      // 16-key blocks
  constexpr int CPR = D / 16;      // 16-byte chunks per row
  constexpr int RPI = 64 / CPR;    // rows per load instruction: 8 or 16, within a block
  constexpr int IPB = 16 / RPI;    // load instructions per block
  constexpr int NKS = D / 32;      // k-steps of S^T
  constexpr int NDB = D / 16;      // 16-dim blocks of O^T
  constexpr int NLD = 2 * NB * IPB;  // loads of a tile
  constexpr int UNIT = 4 * TW;
  static_assert(UNIT == decode8_unit(D), "unit of the flat split");
  // An array a stage, so that the compiler can tell the load's target from the stage
  // being read; a wave's 8 KiB of each: K, then V.
  __shared__ __attribute__((aligned(1024))) char lds_a[4 * 8192];
  __shared__ __attribute__((aligned(1024))) char lds_b[4 * 8192];
  // Where the waves' states meet: kMeet rows of each (two workgroups a CU have 80 KiB
  // each).
  constexpr int kMeet = 768 / D;
  __shared__ __attribute__((aligned(16))) float meet[4 * kMeet * D];
  __shared__ float st_m[4][16], st_l[4][16];

  const Dims& dm = p.dm;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6) & 3;
  const int i16 = lane & 15, lg = lane >> 4;
  const int total = dm.Hkv * p.slots;
  const FlatWave<UNIT> flat_wave(p, lane);
  if (blockIdx.x == (unsigned)total) {  // one workgroup past the slots writes the combine's plan
    if (wave == 0) write_plan(p, flat_wave);
    return;
  }
  const int w = xcd_remap(blockIdx.x, total);
  const int kvh = fast_div(w, p.div_splits.mul, p.div_splits.shift), s = w - kvh * p.slots;
  const bool varlen = p.q_len != nullptr;
  const int pos = fast_div(i16, p.div_g.mul, p.div_g.shift), g = i16 - pos * dm.G;
  const int head = kvh * dm.G + min(g, dm.G - 1);
  [[maybe_unused]] const float slope = MOD ? row_slope(p.mod, head) : 0.f;
  const float c = dm.c;

  const uint32_t kss = (uint32_t)p.k.ss, vss = (uint32_t)p.v.ss;
  const char* kbase = static_cast<const char*>(p.k.ptr) + (int64_t)kvh * p.k.sh;
  const char* vbase = static_cast<const char*>(p.v.ptr) + (int64_t)kvh * p.v.sh;
  const int* keb = p.ke.e + kvh * p.ke.sh;
  const int* veb = p.ve.e + kvh * p.ve.sh;

  // Load offsets: row lrow of an instruction, chunk lane % CPR of LDS, which holds
  // chunk (lane % CPR) ^ f of the row.  Rows of instruction i of block bl: 16 bl + RPI
  // i + lrow.
  //   D = 128: fk = (row >> 1) & 7,  fv = ((row >> 1) & 3) | (row >> 4 & 1) << 2
  //   D = 64:  fk = (row >> 2) & 3,  fv = ((row >> 2) & 1) | (row >> 4 & 1) << 1
  const auto fk = [](int row) { return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
  const auto fv = [](int row) {
    return D == 128 ? ((row >> 1) & 3) | (((row >> 4) & 1) << 2) : ((row >> 2) & 1) | (((row >> 4) & 1) << 1);
  };
  const int lrow = lane / CPR, lch = lane % CPR;
  char* const la = lds_a + wave * 8192;
  char* const lb = lds_b + wave * 8192;
  // LDS read offsets.  K: row i16 of a block (fk does not depend on the block).  V:
  // rows 4 lg + 0..3 and 16 + 4 lg + 0..3 of 32 (fv does not depend on which 32).
  uint32_t ka[NKS / 2];
#pragma unroll
  for (int x = 0; x < NKS / 2; ++x) ka[x] = (uint32_t)(i16 * D + 16 * (((NKS / 2) * lg + x) ^ fk(i16)));
  const int j16 = lane & 15, vrow = 4 * lg + ((j16 >> 1) & 3) + 16 * (j16 >> 3);
  const uint32_t va = (uint32_t)(vrow * D + 16 * fv(vrow) + 8 * (j16 & 1));

  const auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  // The piece at hand: keys [c0, c1) of sequence b; and the one after it.
  struct Piece {
    int b, skv, c0, c1;
    bool some;
  };
  Piece cur, nxt;
  int n = 0;  // this wave's tiles: wave, wave + 4, ...
  int qpos = 0, qpos_lo = 0, seen = 0, seen_lo = 0;
  bool valid = false;
  u32x4 qreg[NKS];
  // Pages and scales of this wave's 64 16-key blocks from its tile `base` on, a block a
  // lane (page -1: behind the piece): read together, handed out by lane, so that the
  // stream of tiles waits for no scalar load.
  constexpr int W = 64 / NB;
  int base = 0, page_l = -1, page_n = -1;
  float sk_l = 1.f, sv_l = 1.f;

  const auto pages_of = [&](const Piece& x, int it) __attribute__((always_inline)) {
    const int key = x.c0 + (4 * (it + lane / NB) + wave) * TW + 16 * (lane % NB);
    return x.some && key < x.c1 ? p.block_table[(int64_t)x.b * p.table_stride + (key >> p.block_shift)] : -1;
  };
  const auto scales = [&]() __attribute__((always_inline)) {  // of page_l: exponents, loaded
    const int64_t id = max(page_l, 0);
    sk_l = __int_as_float(page_l >= 0 ? keb[id * p.ke.sb] : 0);
    sv_l = __int_as_float(page_l >= 0 ? veb[id * p.ve.sb] : 0);
  };
  const auto finish_scales = [&]() __attribute__((always_inline)) {
    sk_l = exp_scale(clamp_exp(__float_as_int(sk_l)));
    sv_l = exp_scale(clamp_exp(__float_as_int(sv_l)));
    pin(sk_l);
    pin(sv_l);
  };
  const auto scale_at = [&](float x, int it, int bl) __attribute__((always_inline)) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), (it - base) * NB + bl));
  };
  const auto issue = [&](int it, char* stage) __attribute__((always_inline)) {
    typedef __attribute__((address_space(3))) void lds_void;
#pragma unroll
    for (int bl = 0; bl < NB; ++bl) {
      const int key = cur.c0 + (4 * it + wave) * TW + 16 * bl, rows = cur.c1 - key;
      const int page = __builtin_amdgcn_readlane(page_l, (it - base) * NB + bl);
      __amdgpu_buffer_rsrc_t tk = make_rsrc(kbase, 0u), tv = make_rsrc(vbase, 0u);
      if (rows > 0) {
        const int64_t slot = key & ((1 << p.block_shift) - 1);
        const uint32_t last = (uint32_t)(min(rows, 16) - 1);
        tk = make_rsrc(kbase + (int64_t)page * p.k.sb + slot * p.k.ss, last * kss + D);
        tv = make_rsrc(vbase + (int64_t)page * p.v.sb + slot * p.v.ss, last * vss + D);
      }
#pragma unroll
      for (int i = 0; i < IPB; ++i) {
        const int row = 16 * bl + RPI * i + lrow;
        const uint32_t ko = (uint32_t)lrow * kss + 16u * (uint32_t)(lch ^ fk(row));
        const uint32_t vo = (uint32_t)lrow * vss + 16u * (uint32_t)(lch ^ fv(row));
        const int at = (bl * IPB + i) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(tk, (lds_void*)(stage + at), 16, ko, (uint32_t)(i * RPI) * kss, 0,
                                                 kDmaStream);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(tv, (lds_void*)(stage + 4096 + at), 16, vo, (uint32_t)(i * RPI) * vss,
                                                 0, kDmaStream);
      }
    }
  };

  FlatWalk<FlatWave<UNIT>, true> walk;
  walk.start(flat_wave, s);
  // nxt: the piece after the one at hand, its pages on their way.
  const auto look = [&]() __attribute__((always_inline)) {
    int from, cnt;
    nxt.some = walk.next(flat_wave, from, cnt);
    nxt.b = nxt.skv = nxt.c0 = nxt.c1 = 0;
    if (nxt.some) {
      nxt.b = uniform(walk.b);
      nxt.skv = uniform(walk.skv);
      nxt.c0 = uniform(from * UNIT);
      nxt.c1 = min(nxt.c0 + uniform(cnt) * UNIT, nxt.skv);
    }
    page_n = pages_of(nxt, 0);
  };
  // nxt becomes the piece at hand: its scales, queries and first two tiles are on
  // their way.
  const auto begin = [&]() __attribute__((always_inline)) {
    cur = nxt;
    page_l = page_n;
    base = 0;
    scales();
    const int sq = varlen ? min(max(load_uniform(p.q_len + cur.b), 0), dm.Sq) : dm.Sq;
    const int64_t tok0 = varlen ? (int64_t)load_uniform(p.q_start + cur.b) : 0;
    const int prefix = MOD ? seq_prefix(p.mod, cur.b, cur.skv) : 0;
    valid = pos < sq;
    qpos = pos + (cur.skv - sq);
    qpos_lo = cur.skv - sq;
    seen = max(qpos, prefix - 1);
    seen_lo = max(qpos_lo, prefix - 1);
    n = ((cur.c1 - cur.c0 + TW - 1) / TW - wave + 3) >> 2;
    const char* qrow = static_cast<const char*>(p.q.ptr) +
                       2 * ((varlen ? (tok0 + pos) * p.q.ss : (int64_t)cur.b * p.q.sb + (int64_t)pos * p.q.ss) +
                            (int64_t)head * p.q.sh + (D / 4) * lg);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
      qreg[ks] = valid ? *reinterpret_cast<const u32x4*>(qrow + 16 * ks) : u32x4{0u, 0u, 0u, 0u};
    look();
    // (Always both, so that the compiler counts on them and waits for the first alone:
    // tiles behind the piece load nothing.)
    issue(0, la);
    issue(1, lb);
  };

  f32x4 acc[NDB];
  float m_run, l_run;
  // Tile `it` out of its stage, then its stage's next one.
  const auto step = [&](auto issue_c, auto last_c, int it, char* stage) __attribute__((always_inline)) {
    constexpr bool ISSUE = decltype(issue_c)::value;
    wave_wait<vmcnt_imm(decltype(last_c)::value ? 0 : NLD)>();
    float sk[NB], sv[NB];
#pragma unroll
    for (int bl = 0; bl < NB; ++bl) {
      sk[bl] = scale_at(sk_l, it, bl);
      sv[bl] = scale_at(sv_l, it, bl);
    }
    const char* ck = stage;
    const char* cv = stage + 4096;
    f32x4 sx[NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      sx[kb] = f32x4{};
#pragma unroll
      for (int x = 0; x < NKS / 2; ++x) {
        const u32x4 raw = *reinterpret_cast<const u32x4*>(ck + kb * 16 * D + ka[x]);
        sx[kb] = E::mfma16(widen8<DT>(raw[0], sk[kb], raw[1], sk[kb]), qreg[2 * x], sx[kb]);
        sx[kb] = E::mfma16(widen8<DT>(raw[2], sk[kb], raw[3], sk[kb]), qreg[2 * x + 1], sx[kb]);
      }
    }
    const int key0 = cur.c0 + (4 * it + wave) * TW;
    float row_t = 0.f;  // added to every score of the lane
    if constexpr (MOD) {
      cap_scores<4>(sx, p.mod);
      if (p.mod.slopes != nullptr)
        row_t = bias_scores<4>(sx, slope, key0 + 4 * lg - qpos, key0 + TW - 1 <= qpos_lo,
                               [](int e) { return 16 * (e >> 2) + (e & 3); });
    }
    if (key0 + TW > cur.c1 || (dm.causal && key0 + TW - 1 > seen_lo)) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int key = key0 + 16 * kb + 4 * lg + v;
          const bool off = key >= cur.c1 || (dm.causal && key > seen);
          sx[kb][v] = off ? -__builtin_inff() : sx[kb][v];
        }
    }
    float mx = fmaxf(fmaxf(sx[0][0], sx[0][1]), fmaxf(sx[0][2], sx[0][3]));
#pragma unroll
    for (int kb = 1; kb < NB; ++kb) mx = fmaxf(vmax3(mx, sx[kb][0], sx[kb][1]), fmaxf(sx[kb][2], sx[kb][3]));
    mx = xhalf_max(xquad_max(mx + row_t));
    const float m_new = fmaxf(m_run, mx);
    const float m_use = (m_new == -__builtin_inff()) ? 0.f : m_new;
    const float alpha = fast_exp2((m_run - m_use) * c), nmc = (row_t - m_use) * c;
    float pv[NB][4], rs = 0.f;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int v = 0; v < 4; ++v) pv[kb][v] = fast_exp2(__builtin_fmaf(sx[kb][v], c, nmc));
      rs += (pv[kb][0] + pv[kb][1]) + (pv[kb][2] + pv[kb][3]);
    }
    l_run = l_run * alpha + rs;
    m_run = m_new;
#pragma unroll
    for (int db = 0; db < NDB; ++db) acc[db] *= alpha;
#pragma unroll
    for (int jj = 0; jj < NB / 2; ++jj) {
      const u32x4 pk =
          u32x4{E::pack2(pv[2 * jj][0], pv[2 * jj][1]), E::pack2(pv[2 * jj][2], pv[2 * jj][3]),
                E::pack2(pv[2 * jj + 1][0], pv[2 * jj + 1][1]), E::pack2(pv[2 * jj + 1][2], pv[2 * jj + 1][3])};
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const u32x2 raw = ld_tr8(cv + 32 * jj * D + (va ^ (uint32_t)(16 * db)));
        acc[db] = E::mfma16(widen8<DT>(raw[0], sv[2 * jj], raw[1], sv[2 * jj + 1]), pk, acc[db]);
      }
    }
    if constexpr (ISSUE) {
      wave_wait<kLgkm0>();  // (the stage has been read)
      if (it + 2 - base >= W) {
        base = it + 1;
        page_l = pages_of(cur, base);
        pin(page_l);
        scales();
        finish_scales();
      }
      issue(it + 2, stage);
    }
  };

  const int rows = dm.G * dm.Sq;
  int done_b = -1;  // the piece whose state the waves hold
  bool done_valid = false;
  look();
  if (!nxt.some) return;
  for (;;) {
    const bool more = nxt.some;
    if (more) begin();
    if (done_b >= 0) {
      // With the next piece's loads on their way the four waves' states meet, kMeet query
      // rows at a time.
      const float l_tot = xhalf_sum(xquad_sum(l_run));
      if (lg == 0) {
        st_m[wave][i16] = m_run;
        st_l[wave][i16] = done_valid ? l_tot : -1.f;
      }
      for (int r0 = 0; r0 < rows; r0 += kMeet) {
        if (i16 >= r0 && i16 < r0 + kMeet) {
          float* to = meet + ((wave * kMeet + i16 - r0) * D + 4 * lg);
#pragma unroll
          for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4*>(to + 16 * db) = acc[db];
        }
        phase_barrier();
#pragma unroll
        for (int f = t; f < kMeet * (D / 4); f += 256) {
          const int rl = f / (D / 4), d4 = f - rl * (D / 4), r = r0 + rl;
          if (r >= rows || st_l[0][r] < 0.f) continue;
          float ms = st_m[0][r];
#pragma unroll
          for (int x = 1; x < 4; ++x) ms = fmaxf(ms, st_m[x][r]);
          const float mu = ms == -__builtin_inff() ? 0.f : ms;
          f32x4 o = {0.f, 0.f, 0.f, 0.f};
          float l = 0.f;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float a = fast_exp2((st_m[x][r] - mu) * c);
            l += a * st_l[x][r];
            o += a * *reinterpret_cast<const f32x4*>(meet + (x * kMeet + rl) * D + 4 * d4);
          }
          const int ps = fast_div(r, p.div_g.mul, p.div_g.shift);
          const int64_t row = partial_row(p, true, done_b, kvh * dm.G + r - ps * dm.G, ps, s);
          *reinterpret_cast<f32x4*>(p.ws_acc + row * D + 4 * d4) = o;
          if (d4 == 0) {
            p.ws_m[row] = ms == -__builtin_inff() ? kEmptyRef : __builtin_fmaf(ms, c, MOD ? p.mod.shift2 : 0.f);
            p.ws_l[row] = l;
          }
        }
        phase_barrier();
      }
    }
    if (!more) break;
#pragma unroll
    for (int db = 0; db < NDB; ++db) acc[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run = -__builtin_inff();
    l_run = 0.f;
    done_b = cur.b;
    done_valid = valid;
    wave_wait<vmcnt_imm(2 * NLD)>();  // what came before the first tile's loads
    finish_scales();
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) pin(qreg[ks]);
    // Tiles in pairs; the last one or two refill nothing.
    using BT = std::true_type;
    using BF = std::false_type;
    int it = 0;
    for (; it + 4 <= ((n + 1) & ~1); it += 2) {
      step(BT{}, BF{}, it, la);
      step(BT{}, BF{}, it + 1, lb);
    }
    if (it + 1 == n) {
      step(BF{}, BT{}, it, la);
    } else if (it < n) {
      step(BF{}, BF{}, it, la);
      step(BF{}, BT{}, it + 1, lb);
    }
  }
  wave_wait<vmcnt_imm(0)>();  // (no load may be on its way into LDS when the workgroup ends)
}

template <int DT, int D> static hipError_t launch_decode8_t(Split8Params p, hipStream_t stream) {
  const int64_t total = (int64_t)p.dm.Hkv * p.slots;
  const int64_t units = (p.dm.Skv + decode8_unit(D) - 1) / decode8_unit(D);
  // (32-bit products of units and slots in the walk.)
  if (total <= 0 || total >= (int64_t)1 << 30 || (units * p.dm.B + 1) * (p.slots + 1) >= (int64_t)1 << 31)
    return hipErrorInvalidValue;
  p.div_splits = make_fast_div((uint32_t)p.slots);
  p.div_g = make_fast_div((uint32_t)p.dm.G);
  p.div_units = make_fast_div((uint32_t)std::max<int64_t>(units, 1));
  const ScoreMod& m = p.mod;
  const bool changed = m.cap_exp != 0.f || m.cap != 0.f || m.slopes != nullptr || m.prefix != nullptr;
  const dim3 grid((unsigned)(total + 1)), block(256);
  if (changed) hipLaunchKernelGGL((gqa_decode8_kernel<DT, D, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((gqa_decode8_kernel<DT, D, false>), grid, block, 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_decode8(const Split8Params& p, int dtype, hipStream_t stream) {
  if (p.dm.G * p.dm.Sq > kDecode8Rows || p.block_shift < 4) return hipErrorInvalidValue;
  if (dtype == 0) return p.dm.D == 128 ? launch_decode8_t<0, 128>(p, stream) : launch_decode8_t<0, 64>(p, stream);
  return p.dm.D == 128 ? launch_decode8_t<1, 128>(p, stream) : launch_decode8_t<1, 64>(p, stream);
}

}  // namespace gqa
