// gqa_decode8.hip — attention over a paged cache in 8 bits (gqa_cache8.hpp) for few
// query rows: single tokens, and as many as give 32 packed rows per kv head (row r ->
// position r / G, head r % G), NR blocks of 16: codes are widened once for both.
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
// here a wave is on its own: it takes every fourth tile of 32 keys (4 KiB of K and of V, 2
// at head_dim 64), all of its scores and all head dimensions, loads tiles into LDS of its
// own two ahead, and meets the others once a piece, in LDS.  No barrier within the stream,
// no score computed twice.
//
// The keys of all sequences are cut into equal ranges, one a workgroup, on the
// device (gqa_flat.hpp), in units of four tiles.
#include <algorithm>

#include "gqa_cache8.hpp"
#include "gqa_decode_kernel.hpp"
#include "gqa_lds.hpp"

namespace gqa {

namespace {

// This wave's memory operations, as far as the immediate says (vmcnt_imm(n): all but n of
// its loads, into LDS among them; kLgkm0: its LDS reads); nothing moves across.
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
template <int DT, int D, int NR, bool MOD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void gqa_decode8_kernel(Split8Params p) {
  using E = Elem<DT>;
  // Keys of a wave's tile.  (64 at head_dim 64, as many bytes: 24 tokens of 200-6000 keys
  // 17.1 us, this 16.0; 256 of up to 300 28.6 / 25.8; 8 queries of 8000 11.0 / 12.7, of
  // 131072 41.6 / 39.4.)
  constexpr int TW = 32;
  constexpr int TBY = TW * D;      // its bytes of K, and of V
  constexpr int NB = TW / 16;      // 16-key blocks
  constexpr int CPR = D / 16;      // 16-byte chunks per row
  constexpr int RPI = 64 / CPR;    // rows per load instruction: 8 or 16, within a block
  constexpr int IPB = 16 / RPI;    // load instructions per block
  constexpr int NKS = D / 32;      // k-steps of S^T
  constexpr int NDB = D / 16;      // 16-dim blocks of O^T
  constexpr int NLD = 2 * NB * IPB;  // loads of a tile
  constexpr int UNIT = 4 * TW;
  // The running reference follows a row's maximum only once it lags by 2^kLag: until then
  // probabilities exceed 1, which no type here minds (fp16 holds 2^15), and the
  // accumulators need no scaling (16 x 8 queries of 8000 keys 71.0 -> 69.7 us).
  constexpr float kLag = 8.f;
  static_assert(UNIT == kDecode8Unit, "unit of the flat split");
  // An array a stage, so that the compiler can tell the load's target from the stage
  // being read; a wave's part of each: K, then V.
  __shared__ __attribute__((aligned(1024))) char lds_a[4 * 2 * TBY];
  __shared__ __attribute__((aligned(1024))) char lds_b[4 * 2 * TBY];
  constexpr int kJoin = (int)sizeof(lds_b) / (16 * D);  // query rows whose four states a stage holds
  __shared__ float st_m[4][16 * NR], st_l[4][16 * NR];

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
  // Heads whose rows share a 128-byte line of the cache, PAIR of them, are neighbours in
  // the launch, so that the line comes to an XCD's L2 once (head_dim 64, 16 x 8 queries of
  // 8000 keys 51.0 -> 40.2 us).
  constexpr int PAIR = 128 / D;
  const int wp = dm.Hkv % PAIR == 0 ? w / PAIR : w;
  const int kp = fast_div(wp, p.div_splits.mul, p.div_splits.shift), s = wp - kp * p.slots;
  const int kvh = dm.Hkv % PAIR == 0 ? kp * PAIR + w % PAIR : kp;
  const bool varlen = p.q_len != nullptr;
  // This lane's query rows, i16 of each 16-row block.
  int pos[NR], head[NR];
  [[maybe_unused]] float slope[NR];
#pragma unroll
  for (int rb = 0; rb < NR; ++rb) {
    const int r = 16 * rb + i16;
    pos[rb] = fast_div(r, p.div_g.mul, p.div_g.shift);
    head[rb] = kvh * dm.G + r - pos[rb] * dm.G;
    slope[rb] = MOD ? row_slope(p.mod, head[rb]) : 0.f;
  }
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
  char* const la = lds_a + wave * 2 * TBY;
  char* const lb = lds_b + wave * 2 * TBY;
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
  int qpos[NR], seen[NR], qpos_lo = 0, seen_lo = 0;
  bool valid[NR];
  u32x4 qreg[NR][NKS];
  // Addresses and scales of this wave's 64 16-key blocks from its tile `base` on, a block a
  // lane (page -1: behind the piece): read together, handed out by lane, so that the
  // stream of tiles waits for no scalar load and multiplies no strides (from L2, 16 x 4
  // queries of 8000 keys 26.3 -> 24.5 us).
  constexpr int W = 64 / NB;
  int base = 0, page_l = -1, page_n = -1;
  uint32_t klo = 0, khi = 0, vlo = 0, vhi = 0;
  float sk_l = 1.f, sv_l = 1.f;

  const auto pages_of = [&](const Piece& x, int it) __attribute__((always_inline)) {
    const int key = x.c0 + (4 * (it + lane / NB) + wave) * TW + 16 * (lane % NB);
    return x.some && key < x.c1 ? p.block_table[(int64_t)x.b * p.table_stride + (key >> p.block_shift)] : -1;
  };
  const auto scales = [&]() __attribute__((always_inline)) {  // of page_l: addresses; exponents, loaded
    const int64_t id = max(page_l, 0);
    const int key = cur.c0 + (4 * (base + lane / NB) + wave) * TW + 16 * (lane % NB);
    const int64_t slot = key & ((1 << p.block_shift) - 1);
    const uint64_t ko = (uint64_t)kbase + id * p.k.sb + slot * p.k.ss;
    const uint64_t vo = (uint64_t)vbase + id * p.v.sb + slot * p.v.ss;
    klo = (uint32_t)ko, khi = (uint32_t)(ko >> 32), vlo = (uint32_t)vo, vhi = (uint32_t)(vo >> 32);
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
      const int from = (it - base) * NB + bl;
      const auto at = [&](uint32_t lo, uint32_t hi) {
        return reinterpret_cast<const char*>((uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, from) << 32 |
                                             (uint32_t)__builtin_amdgcn_readlane(lo, from));
      };
      const uint32_t last = (uint32_t)(min(rows, 16) - 1);
      const __amdgpu_buffer_rsrc_t tk = make_rsrc(at(klo, khi), rows > 0 ? last * kss + D : 0u);
      const __amdgpu_buffer_rsrc_t tv = make_rsrc(at(vlo, vhi), rows > 0 ? last * vss + D : 0u);
#pragma unroll
      for (int i = 0; i < IPB; ++i) {
        const int row = 16 * bl + RPI * i + lrow;
        const uint32_t ko = (uint32_t)lrow * kss + 16u * (uint32_t)(lch ^ fk(row));
        const uint32_t vo = (uint32_t)lrow * vss + 16u * (uint32_t)(lch ^ fv(row));
        const int at = (bl * IPB + i) * 1024;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(tk, (lds_void*)(stage + at), 16, ko, (uint32_t)(i * RPI) * kss, 0,
                                                 kDmaStream);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(tv, (lds_void*)(stage + TBY + at), 16, vo, (uint32_t)(i * RPI) * vss,
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
    qpos_lo = cur.skv - sq;
    seen_lo = max(qpos_lo, prefix - 1);
    n = ((cur.c1 - cur.c0 + TW - 1) / TW - wave + 3) >> 2;
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      valid[rb] = pos[rb] < sq;
      qpos[rb] = pos[rb] + (cur.skv - sq);
      seen[rb] = max(qpos[rb], prefix - 1);
      const int64_t at = varlen ? (tok0 + pos[rb]) * p.q.ss : (int64_t)cur.b * p.q.sb + (int64_t)pos[rb] * p.q.ss;
      const char* qrow = static_cast<const char*>(p.q.ptr) + 2 * (at + (int64_t)head[rb] * p.q.sh + (D / 4) * lg);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        qreg[rb][ks] = valid[rb] ? *reinterpret_cast<const u32x4*>(qrow + 16 * ks) : u32x4{0u, 0u, 0u, 0u};
    }
    look();
    issue(0, la);
  };

  f32x4 acc[NR][NDB];
  float m_run[NR], l_run[NR];
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
    const char* cv = stage + TBY;
    // One row block: all reads of the tile first (32 sequences of up to 8000 keys 34.1 ->
    // 33.0 us).  Two: where they are used (all first, for the registers they hold, 42.7 ->
    // 44.1 us in 16 x 8 queries of up to 8000 keys).
    u32x4 rawk[NB][NKS / 2];
    u32x2 rawv[NB / 2][NDB];
    if constexpr (NR == 1) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int x = 0; x < NKS / 2; ++x) rawk[kb][x] = *reinterpret_cast<const u32x4*>(ck + kb * 16 * D + ka[x]);
#pragma unroll
      for (int jj = 0; jj < NB / 2; ++jj)
#pragma unroll
        for (int db = 0; db < NDB; ++db) rawv[jj][db] = ld_tr8(cv + 32 * jj * D + (va ^ (uint32_t)(16 * db)));
      __builtin_amdgcn_sched_barrier(0);
    }
    f32x4 sx[NR][NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) sx[rb][kb] = f32x4{};
#pragma unroll
      for (int x = 0; x < NKS / 2; ++x) {
        const u32x4 raw = NR == 1 ? rawk[kb][x] : *reinterpret_cast<const u32x4*>(ck + kb * 16 * D + ka[x]);
        const u32x4 lo = widen8<DT>(raw[0], sk[kb], raw[1], sk[kb]), hi = widen8<DT>(raw[2], sk[kb], raw[3], sk[kb]);
#pragma unroll
        for (int rb = 0; rb < NR; ++rb) {
          sx[rb][kb] = E::mfma16(lo, qreg[rb][2 * x], sx[rb][kb]);
          sx[rb][kb] = E::mfma16(hi, qreg[rb][2 * x + 1], sx[rb][kb]);
        }
      }
    }
    const int key0 = cur.c0 + (4 * it + wave) * TW;
    u32x4 pk[NR][NB / 2];
    float row_t[NR], mx[NR], nmc[NR], pv[NR][NB][4];
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      row_t[rb] = 0.f;  // added to every score of the lane
      if constexpr (MOD) {
        cap_scores<4>(sx[rb], p.mod);
        if (p.mod.slopes != nullptr)
          row_t[rb] = bias_scores<4>(sx[rb], slope[rb], key0 + 4 * lg - qpos[rb], key0 + TW - 1 <= qpos_lo,
                                     [](int e) { return 16 * (e >> 2) + (e & 3); });
      }
    }
    if (key0 + TW > cur.c1 || (dm.causal && key0 + TW - 1 > seen_lo)) {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb)
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int key = key0 + 16 * kb + 4 * lg + v;
            const bool off = key >= cur.c1 || (dm.causal && key > seen[rb]);
            sx[rb][kb][v] = off ? -__builtin_inff() : sx[rb][kb][v];
          }
    }
    bool lags = false;
#pragma unroll
    for (int rb = 0; rb < NR; ++rb)
      mx[rb] = fmaxf(fmaxf(sx[rb][0][0], sx[rb][0][1]), fmaxf(sx[rb][0][2], sx[rb][0][3]));
#pragma unroll
    for (int kb = 1; kb < NB; ++kb)
#pragma unroll
      for (int rb = 0; rb < NR; ++rb)
        mx[rb] = fmaxf(vmax3(mx[rb], sx[rb][kb][0], sx[rb][kb][1]), fmaxf(sx[rb][kb][2], sx[rb][kb][3]));
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) mx[rb] = xquad_max(mx[rb] + row_t[rb]);
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) mx[rb] = xhalf_max(mx[rb]);
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) lags |= (mx[rb] - m_run[rb]) * c > kLag || m_run[rb] == -__builtin_inff();
    if (__any(lags)) {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        const float m_new = fmaxf(m_run[rb], mx[rb]);
        const float alpha = m_new == -__builtin_inff() ? 1.f : fast_exp2((m_run[rb] - m_new) * c);
        m_run[rb] = m_new;
        l_run[rb] *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db) acc[rb][db] *= alpha;
      }
    }
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) nmc[rb] = (row_t[rb] - (m_run[rb] == -__builtin_inff() ? 0.f : m_run[rb])) * c;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
#pragma unroll
        for (int v = 0; v < 4; ++v) pv[rb][kb][v] = fast_exp2(__builtin_fmaf(sx[rb][kb][v], c, nmc[rb]));
      }
#pragma unroll
    for (int jj = 0; jj < NB / 2; ++jj)
#pragma unroll
      for (int rb = 0; rb < NR; ++rb)
        pk[rb][jj] = u32x4{E::pack2(pv[rb][2 * jj][0], pv[rb][2 * jj][1]),
                           E::pack2(pv[rb][2 * jj][2], pv[rb][2 * jj][3]),
                           E::pack2(pv[rb][2 * jj + 1][0], pv[rb][2 * jj + 1][1]),
                           E::pack2(pv[rb][2 * jj + 1][2], pv[rb][2 * jj + 1][3])};
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      float rs = 0.f;
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) rs += (pv[rb][kb][0] + pv[rb][kb][1]) + (pv[rb][kb][2] + pv[rb][kb][3]);
      l_run[rb] += rs;
    }
#pragma unroll
    for (int jj = 0; jj < NB / 2; ++jj) {
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const u32x2 raw = NR == 1 ? rawv[jj][db] : ld_tr8(cv + 32 * jj * D + (va ^ (uint32_t)(16 * db)));
        const u32x4 w = widen8<DT>(raw[0], sv[2 * jj], raw[1], sv[2 * jj + 1]);
#pragma unroll
        for (int rb = 0; rb < NR; ++rb) acc[rb][db] = E::mfma16(w, pk[rb][jj], acc[rb][db]);
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
  bool done_valid[NR] = {};
  // The four waves' states meet and leave as the slot's partials, kJoin query rows at a
  // time, in the second stage (the next piece's first tile is on its way into the first; a
  // place of its own, and both tiles on their way, took three times the rounds: 16 x 8
  // queries of up to 8000 keys 43.3 us, this 40.2, 32 tokens of up to 8000 33.5 / 32.4).
  // 16-byte chunks of a row are swizzled, so that the lanes of a write cover the banks.
  const auto join = [&]() __attribute__((always_inline)) {
    const auto at = [&](int wv, int rl, int chunk) {
      return reinterpret_cast<float*>(lds_b) + (wv * kJoin + rl) * D + 4 * (chunk ^ (rl & 15));
    };
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      const float l_tot = xhalf_sum(xquad_sum(l_run[rb]));
      if (lg == 0) {
        st_m[wave][16 * rb + i16] = m_run[rb];
        st_l[wave][16 * rb + i16] = done_valid[rb] ? l_tot : -1.f;
      }
    }
    phase_barrier();  // (the stage has been read)
    for (int r0 = 0; r0 < rows; r0 += kJoin) {
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        const int rl = 16 * rb + i16 - r0;
        if (rl >= 0 && rl < kJoin) {
#pragma unroll
          for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4*>(at(wave, rl, 4 * db + lg)) = acc[rb][db];
        }
      }
      phase_barrier();
      for (int f = t; f < min(kJoin, rows - r0) * (D / 4); f += 256) {
        const int rl = f / (D / 4), d4 = f - rl * (D / 4), r = r0 + rl;
        if (st_l[0][r] < 0.f) continue;
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
          o += a * *reinterpret_cast<const f32x4*>(at(x, rl, d4));
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
  };
  using BT = std::true_type;
  using BF = std::false_type;
  look();
  if (!nxt.some) return;
  for (;;) {
    if (done_b >= 0) wave_wait<vmcnt_imm(0)>();  // (loads of tiles behind the last piece)
    const bool more = nxt.some;
    if (more) begin();
    if (done_b >= 0) join();
    if (!more) return;
    // (Always both tiles, so that the compiler counts on them and waits for the first
    // alone: tiles behind the piece load nothing.)
    issue(1, lb);
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
#pragma unroll
      for (int db = 0; db < NDB; ++db) acc[rb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run[rb] = -__builtin_inff();
      l_run[rb] = 0.f;
      done_valid[rb] = valid[rb];
    }
    done_b = cur.b;
    wave_wait<vmcnt_imm(2 * NLD)>();  // what came before the first tile's loads
    finish_scales();
#pragma unroll
    for (int rb = 0; rb < NR; ++rb)
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) pin(qreg[rb][ks]);
    // Tiles in pairs; the last one or two refill nothing.
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
}

// Joins the slots' partials of each row, as gqa_split_reduce_kernel does with a workgroup
// a row, for sequences that lie in few slots: a row's D / 4 lanes take all of its
// partials, 1024 / D rows a workgroup.  Rows in the order of the slots' walk, (kv head,
// sequence, head, query), so that a row is joined on the XCD that wrote its partials.
template <int DT, int D>
__global__ __launch_bounds__(256) void gqa_decode8_join_kernel(ReduceParams p, FastDiv div_g, int G) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int ND4 = D / 4, R = 256 / ND4, BATCH = 4;
  const int t = threadIdx.x, d4 = t % ND4, bg = p.B * G;
  const int x = xcd_remap(blockIdx.x, gridDim.x) * R + t / ND4;
  const int xh = fast_div(x, p.div_sq.mul, p.div_sq.shift), pos = x - xh * p.Sq;
  const int kvh = fast_div(xh, p.div_total.mul, p.div_total.shift), xb = xh - kvh * bg;
  const int b = fast_div(xb, div_g.mul, div_g.shift), h = kvh * G + xb - b * G;
  if (h >= p.Hq) return;
  const bool varlen = p.q_len != nullptr;
  if (varlen && pos >= p.q_len[b]) return;
  const int64_t step = (int64_t)p.Hq * p.Sq;
  const int S = p.plan[2 * b + 1];
  const int64_t row0 = p.plan[2 * b] * step + (int64_t)h * p.Sq + pos;
  const float *wm = p.ws_m + row0, *wl = p.ws_l + row0, *wa = p.ws_acc + row0 * D + 4 * d4;
  float m = kEmptyRef, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < S; s0 += BATCH) {
    float mv[BATCH], lv[BATCH];
    f32x4 av[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int s = s0 + k;
      mv[k] = kEmptyRef;
      lv[k] = 0.f;
      av[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (s < S) {
        mv[k] = wm[s * step];
        lv[k] = wl[s * step];
        av[k] = *reinterpret_cast<const f32x4*>(wa + s * step * D);
      }
    }
    const float mb = fmaxf(fmaxf(fmaxf(mv[0], mv[1]), fmaxf(mv[2], mv[3])), m);
    const float keep = fast_exp2(m - mb);
    l *= keep;
    o *= keep;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const float a = fast_exp2(mv[k] - mb);
      l += a * lv[k];
      o += a * av[k];
    }
    m = mb;
  }
  const int64_t tok = varlen ? (int64_t)p.q_start[b] + pos : 0;
  if (p.lse != nullptr && d4 == 0)
    p.lse[varlen ? tok * p.Hq + h : ((int64_t)b * p.Hq + h) * p.Sq + pos] = (m + __log2f(l)) * kLn2;
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // (a row that sees no key: zeros)
  T* orow = static_cast<T*>(const_cast<void*>(p.o.ptr)) + (int64_t)h * p.o.sh +
            (varlen ? tok * p.o.ss : (int64_t)b * p.o.sb + (int64_t)pos * p.o.ss);
  u32x2 y;
  y[0] = E::pack2(o[0] * inv, o[1] * inv);
  y[1] = E::pack2(o[2] * inv, o[3] * inv);
  *reinterpret_cast<u32x2*>(orow + 4 * d4) = y;
}

template <int DT, int D> static hipError_t launch_decode8_t(Split8Params p, hipStream_t stream) {
  const int64_t total = (int64_t)p.dm.Hkv * p.slots;
  const int64_t units = (p.dm.Skv + kDecode8Unit - 1) / kDecode8Unit;
  // (32-bit products of units and slots in the walk.)
  if (total <= 0 || total >= (int64_t)1 << 30 || (units * p.dm.B + 1) * (p.slots + 1) >= (int64_t)1 << 31)
    return hipErrorInvalidValue;
  p.div_splits = make_fast_div((uint32_t)p.slots);
  p.div_g = make_fast_div((uint32_t)p.dm.G);
  p.div_units = make_fast_div((uint32_t)std::max<int64_t>(units, 1));
  const ScoreMod& m = p.mod;
  const bool changed = m.cap_exp != 0.f || m.cap != 0.f || m.slopes != nullptr || m.prefix != nullptr;
  const dim3 grid((unsigned)(total + 1)), block(256);
  if (p.dm.G * p.dm.Sq <= 16) {
    if (changed) hipLaunchKernelGGL((gqa_decode8_kernel<DT, D, 1, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((gqa_decode8_kernel<DT, D, 1, false>), grid, block, 0, stream, p);
  } else {
    if (changed) hipLaunchKernelGGL((gqa_decode8_kernel<DT, D, 2, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((gqa_decode8_kernel<DT, D, 2, false>), grid, block, 0, stream, p);
  }
  return hipGetLastError();
}

hipError_t launch_decode8(const Split8Params& p, int dtype, hipStream_t stream) {
  if (p.dm.G * p.dm.Sq > kDecode8Rows || p.block_shift < 4) return hipErrorInvalidValue;
  if (dtype == 0) return p.dm.D == 128 ? launch_decode8_t<0, 128>(p, stream) : launch_decode8_t<0, 64>(p, stream);
  return p.dm.D == 128 ? launch_decode8_t<1, 128>(p, stream) : launch_decode8_t<1, 64>(p, stream);
}

template <int DT, int D> static hipError_t launch_join_t(ReduceParams p, int G, hipStream_t stream) {
  const int64_t rows = (int64_t)p.B * p.Hq * p.Sq, wgs = (rows * (D / 4) + 255) / 256;
  if (rows <= 0 || rows >= (int64_t)1 << 30) return hipErrorInvalidValue;
  p.div_sq = make_fast_div((uint32_t)p.Sq);
  p.div_total = make_fast_div((uint32_t)(p.B * G));
  hipLaunchKernelGGL((gqa_decode8_join_kernel<DT, D>), dim3((unsigned)wgs), dim3(256), 0, stream, p,
                     make_fast_div((uint32_t)G), G);
  return hipGetLastError();
}

// Slots a sequence, on average, up to which its rows share a workgroup.  A workgroup a row
// / this, us a call, head_dim 128 of 32 heads over 8: 256 sequences of up to 300 keys (0.25
// slots each) 48.6 / 37.6, 64 of 1000 (1) 29.1 / 26.5, 16 of 4000 (4) 26.6 / 25.8, with 8
// queries each 48.5 / 43.0; 8 of 4000 (8) 18.0 / 18.0 and 33.1 / 30.3; 4 of 8000 (16) 17.1
// / 18.6; 2 of 16000 (32) 17.9 / 22.5.
// (A slot that writes the sequences that lie in it alone itself, us: 500 of 1000 keys 161.6
// -> 154.6, 64 of 1500 33.5 -> 34.3, one token of 700 8.1 -> 8.7: left.)
constexpr int kFewSlots = 8;

hipError_t launch_decode8_join(const ReduceParams& p, int G, int dtype, hipStream_t stream) {
  if (p.slots > kFewSlots * p.B) return launch_split_reduce(p, dtype, stream);
  if (dtype == 0) return p.D == 128 ? launch_join_t<0, 128>(p, G, stream) : launch_join_t<0, 64>(p, G, stream);
  return p.D == 128 ? launch_join_t<1, 128>(p, G, stream) : launch_join_t<1, 64>(p, G, stream);
}

}  // namespace gqa
