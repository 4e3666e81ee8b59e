// gqa_chunk8.hip — attention over a paged cache in 8 bits (gqa_cache8.hpp) for more
// query rows than gqa_decode8.hip takes: verification of drafts, chunks of prompts,
// whole prompts.
//
// Rows, products, softmax and changed scores are those of gqa_scored.hip: 128 packed
// rows in four waves, S^T = K Q^T and O^T += V^T P^T by 32x32x16 MFMAs over 64-key
// tiles, lazily rescaled online softmax.  What differs is the way of a tile into LDS:
// its codes are loaded into registers a phase ahead, widened there to the queries' type
// with their page's power of two (exact), and stored in the swizzled layout of the
// 16-bit tiles.  A workgroup widens a code once, for all of its waves: an instruction
// per two codes.  (Each wave widening what it reads from LDS would take as many times
// that as there are waves.)
//
// One group of four waves, tile j: MFMA phase (P V of the tile before, S of this one),
// which first loads the codes of K(j + 1) and V(j), barrier, softmax phase, which ends by
// storing them where K(j) and V(j - 1) were; barrier.  K and V have one stage each.
//
// Two groups, for more rows of long sequences (chunk8_rows): group 1 is a phase behind
// group 0, so that one's MFMAs run beside the other's softmax on each SIMD; group 0 fills
// K's stages, group 1 V's, two of each, in their MFMA phases, from what their softmax
// phases load: group 0 K(j + 1) in the phase of its S(j), group 1 V(j) in that of its,
// before group 0's next phase takes it; what they write over was read a phase before or
// earlier.  That halves what a row pays for loads, widening and LDS writes, which are most
// of what the cache in 8 bits costs over one in 16: 2048 queries over 16384 keys, 32 heads
// over 8, 550 us for one group and 486 for two (470 the kernel over a cache in 16 bits;
// 390 without loads and stores).  Widening in the softmax phase, whose instructions then
// outlast the other group's MFMAs, took 2.5 % more, pages and exponents by scalar loads
// instead of by lane 1 %.  At head_dim 64 the softmax takes twice as long as the matrix
// instructions, so that three workgroups of one group a CU, each for itself, do more than
// groups in step (8192 tokens over themselves 330 us / 375, 4 x 256 queries over 2000-9000
// keys 79 / 86, but 2048 queries over 16384 keys, two workgroups a CU, 339 / 318), and more
// than two (8 x 512 queries over 512-4096 keys 118 / 128).
#include <algorithm>
#include <type_traits>

#include "gqa_cache8.hpp"
#include "gqa_decode_kernel.hpp"
#include "gqa_fwd_parts.hpp"
#include "gqa_lds.hpp"
#include "gqa_score.hpp"

namespace gqa {

namespace {

constexpr int kTileKeys = FwdStage<64>::kKeys;
static_assert(kTileKeys == FwdStage<128>::kKeys, "tiles of both head dimensions");

// How a call over key pieces (p.kv_splits of them, at least one a sequence) cuts its
// sequences: into pieces of `tiles` tiles, the fewest of which there are not more than
// p.kv_splits, counted from the lengths by every wave for itself (gqa_flat.hpp cuts at
// equal shares, through the middle of what many query blocks read).  The shares of equal
// chunks of the longest sequence, most of them empty or short, cost 4 x 256 queries over
// 2000-9000 keys 143 us for 2 chunks, 120 for 3 and 154 for 4, and these pieces 111.
struct Pieces {
  const Fwd8Params& p;
  int lane, tiles;

  // Tiles of sequence g0 + lane (none without queries).
  __device__ int tiles_of(int g0) const {
    const int s = g0 + lane;
    if (s >= p.dm.B || (p.q_len != nullptr && p.q_len[s] <= 0)) return 0;
    return (min(max(p.seq_lens[s], 0), p.dm.Skv) + kTileKeys - 1) / kTileKeys;
  }
  __device__ static int last(int x) { return __builtin_amdgcn_readlane(x, 63); }

  __device__ Pieces(const Fwd8Params& p, int lane) : p(p), lane(lane) {
    int total = 0, longest = 1;
    for (int g0 = 0; g0 < p.dm.B; g0 += 64) {
      const int t = tiles_of(g0);
      total += last(wave_scan(t));
      longest = max(longest, wave_max(t));
    }
    // A candidate a lane, from the equal share up in steps of a sixteenth; the last one
    // always does.
    const int share = max((total + p.kv_splits - 1) / p.kv_splits, 1);
    const int mine = lane == 63 ? longest : share + lane * ((share + 15) / 16);
    const float inv = 1.0f / (float)mine;
    int count = 0;
    for (int g0 = 0; g0 < p.dm.B; g0 += 64) {
      const int t = tiles_of(g0), n = min(p.dm.B - g0, 64);
      for (int l = 0; l < n; ++l) {
        const int x = __builtin_amdgcn_readlane(t, l), q = (int)((float)x * inv), r = x - q * mine;
        count += q + (r > 0) + (r > mine) - (r <= -mine);  // ceil(x / mine): q is off by at most one
      }
    }
    const uint64_t fits = __builtin_amdgcn_ballot_w64(count <= p.kv_splits || lane == 63);
    tiles = __builtin_amdgcn_readlane(mine, __builtin_ffsll((long long)fits) - 1);
  }

  // f(sequence of the lane, its first piece, its pieces), by 64 sequences, until it
  // returns true.
  template <class F> __device__ void each(F f) const {
    int before = 0;
    for (int g0 = 0; g0 < p.dm.B; g0 += 64) {
      const int n = (tiles_of(g0) + tiles - 1) / tiles, upto = wave_scan(n);
      if (f(g0, before + upto - n, n)) return;
      before += last(upto);
    }
  }
};

}  // namespace

// NG: groups of four waves, 128 rows each.  KC: over key pieces, whose partials
// launch_decode8_join joins by the plan that one workgroup past the others writes.
template <int DT, int D, int NG, bool KC>
__global__ __launch_bounds__(256 * NG)
__attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2))) void gqa_chunk8_kernel(Fwd8Params p) {
  using E = Elem<DT>;
  using T = typename E::T;
  using ST = FwdStage<D>;
  constexpr int NDB = D / 32;   // 32-wide d blocks of O^T
  constexpr int NKS = D / 16;   // k-steps of S^T
  constexpr int PF = 4;         // MFMA slots of LDS-read lookahead
  constexpr int TB = ST::kTileBytes;
  constexpr int CPR8 = D / 8;   // 8-code chunks per row, 16 bytes of the widened tile
  constexpr int RPL = 64 / CPR8;  // rows per load of a wave: 4 or 8
  constexpr int NL = 16 / RPL;    // loads of a wave's 16 rows
  __shared__ __attribute__((aligned(1024))) char lds[2 * NG * TB];  // NG stages of K, then of V

  const Dims& dm = p.dm;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6) & (4 * NG - 1);
  const int group = NG == 2 ? wave >> 2 : 0, gw = wave & 3;
  const int i = lane & 31, hh = lane >> 5;
  const bool varlen = p.q_len != nullptr;

  // Work item: as gqa_scored.hip, or (kv head, piece, query block), so that the blocks
  // that read a piece are neighbours on an XCD.
  int b, kvh, mrank, piece = 0, tb = 0, piece_tiles = 0;
  if constexpr (KC) {
    const int total = dm.Hkv * p.kv_splits * p.n_mblk;
    const Pieces pieces(p, lane);
    if (blockIdx.x == (unsigned)total) {
      if (wave == 0) {
        pieces.each([&](int g0, int first, int n) {
          if (g0 + lane < dm.B) {  // (within the partials whatever the lengths did meanwhile)
            p.plan[2 * (g0 + lane)] = min(first, p.kv_splits);
            p.plan[2 * (g0 + lane) + 1] = min(n, p.kv_splits - min(first, p.kv_splits));
          }
          return false;
        });
      }
      return;
    }
    const int w = xcd_remap(blockIdx.x, total);
    const int rest = fast_div(w, p.div_mblk.mul, p.div_mblk.shift);
    mrank = w - rest * p.n_mblk;
    kvh = fast_div(rest, p.div_items.mul, p.div_items.shift);
    piece = rest - kvh * p.kv_splits;
    b = -1;
    pieces.each([&](int g0, int first, int n) {
      const uint64_t at = __builtin_amdgcn_ballot_w64(first <= piece && piece < first + n);
      if (at == 0) return false;
      const int l = __builtin_ffsll((long long)at) - 1;
      b = g0 + l;
      tb = (piece - __builtin_amdgcn_readlane(first, l)) * pieces.tiles;
      return true;
    });
    if (b < 0) return;  // (fewer pieces)
    piece_tiles = pieces.tiles;
  } else {
    const int w = xcd_remap(blockIdx.x, p.n_mblk * dm.Hkv * dm.B);
    int bh;
    item_of(p, w, p.n_mblk, bh, mrank);
    if (p.xcd_heads > 1) bh = turned_pair(p, bh, mrank);
    b = fast_div(bh, p.div_hkv.mul, p.div_hkv.shift);
    kvh = bh - b * dm.Hkv;
  }
  const int pid_m = dm.causal ? p.n_mblk - 1 - mrank : mrank;
  const int skv = min(max(load_uniform(p.seq_lens + b), 0), dm.Skv);
  const int sq = varlen ? min(max(load_uniform(p.q_len + b), 0), dm.Sq) : dm.Sq;
  const int64_t tok0 = varlen ? (int64_t)load_uniform(p.q_start + b) : 0;
  const int pos_lo = pid_m * p.block_m;
  if (pos_lo >= sq) return;  // a block past this sequence's queries

  // This lane's query row.
  const int r = wave * 32 + i;
  const int g = (int)(__umul24(r, p.bm_mul) >> 16);
  const int pos = pos_lo + r - g * p.block_m;
  const bool valid = g < dm.G && pos < sq;
  const int head = kvh * dm.G + (g < dm.G ? g : 0);
  const int qpos_lo = pos_lo + (skv - sq);
  const int pos_hi = min(pos_lo + p.block_m, sq) - 1;
  const RowSpan span = row_span(p.mod, dm, b, skv, sq, pos_lo, pos_hi, pos, valid, lane, hh);
  float slope = row_slope(p.mod, head);
  // Tiles [tb, tb + n) of this item.
  int n = (span.end + ST::kKeys - 1) / ST::kKeys;
  if constexpr (KC) n = max(min(n - tb, piece_tiles), 0);
  // The piece's partial of this lane's row, in the flat split's layout.
  const int64_t part = ((int64_t)piece * dm.Hq + head) * dm.Sq + pos;
  if (KC && n == 0) {  // (behind the last key that the block sees)
    if (valid) {
      for (int d = 4 * hh; d < D; d += 8)
        *reinterpret_cast<f32x4*>(p.ws_acc + part * D + d) = f32x4{0.f, 0.f, 0.f, 0.f};
      if (hh == 0) {
        p.ws_m[part] = kEmptyRef;
        p.ws_l[part] = 0.f;
      }
    }
    return;
  }
  const bool back = p.mod.slopes != nullptr && dm.causal;
  const auto tile_of = [&](int j) __attribute__((always_inline)) { return tile_at(tb, n, j, back); };

  // This wave's rows of a tile: 16 gw + 0..15, which lie in one page.  Rows past the
  // item's last key, or the last that the block sees, load as zeros.  One group: of K
  // and of V; two: group 0's are K's, group 1's V's.
  constexpr int NOP = NG == 1 ? 2 : 1;
  const int rows_ld = KC ? min(span.end, (tb + n) * ST::kKeys) : span.end;
  const bool of_v = NG == 2 && group == 1;
  const char* kbh = static_cast<const char*>(p.k.ptr) + (int64_t)kvh * p.k.sh;
  const char* vbh = static_cast<const char*>(p.v.ptr) + (int64_t)kvh * p.v.sh;
  const int* keb = p.ke.e + kvh * p.ke.sh;
  const int* veb = p.ve.e + kvh * p.ve.sh;
  const char* const op_base[2] = {of_v ? vbh : kbh, vbh};
  const int64_t op_sb[2] = {of_v ? p.v.sb : p.k.sb, p.v.sb};
  const uint32_t op_ss[2] = {(uint32_t)(of_v ? p.v.ss : p.k.ss), (uint32_t)p.v.ss};
  const int* const op_e[2] = {of_v ? veb : keb, veb};
  const int64_t op_eb[2] = {of_v ? p.ve.sb : p.ke.sb, p.ve.sb};
  const int* table_row = p.block_table + (int64_t)b * p.table_stride;
  // Pages (-1: no rows) and scales of this wave's rows of tiles base .. base + 63, a tile
  // a lane.
  int base = 0, page_l;
  float scale_l[NOP];
  const auto look = [&](int from) __attribute__((always_inline)) {
    base = from;
    const int key = tile_of(from + lane) * ST::kKeys + 16 * gw;
    page_l = key < rows_ld ? table_row[key >> p.block_shift] : -1;
#pragma unroll
    for (int o = 0; o < NOP; ++o)
      scale_l[o] = exp_scale(clamp_exp(page_l >= 0 ? op_e[o][(int64_t)page_l * op_eb[o]] : 0));
    pin(page_l);
#pragma unroll
    for (int o = 0; o < NOP; ++o) pin(scale_l[o]);
  };
  const auto page_of = [&](int j) __attribute__((always_inline)) {
    return __builtin_amdgcn_readlane(page_l, j - base);
  };
  const auto scale_of = [&](int o, int j) __attribute__((always_inline)) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(scale_l[o]), j - base));
  };
  const int lrow = lane / CPR8, lch = lane % CPR8;
  u32x2 rx[NOP][NL];
  float rs[NOP];
  uint32_t off[NOP];
#pragma unroll
  for (int o = 0; o < NOP; ++o) off[o] = (uint32_t)lrow * op_ss[o] + 8u * lch;
  // Operand o's rows of tile j from `page`.
  const auto load = [&](int o, int j, int page) __attribute__((always_inline)) {
    const int key = tile_of(j) * ST::kKeys + 16 * gw, rows = rows_ld - key;
    __amdgpu_buffer_rsrc_t rt = make_rsrc(op_base[o], 0u);
    if (rows > 0) {
      const int64_t slot = key & ((1 << p.block_shift) - 1);
      rt = make_rsrc(op_base[o] + (int64_t)page * op_sb[o] + slot * op_ss[o],
                     (uint32_t)(min(rows, 16) - 1) * op_ss[o] + D);
    }
#pragma unroll
    for (int u = 0; u < NL; ++u)
      rx[o][u] = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_raw_buffer_load_b64(rt, off[o], (uint32_t)(u * RPL) * op_ss[o], 0));
  };
  // Eight codes a lane and load into 16 bytes of the widened tile: 16 lanes write a whole
  // row, or two (sixteen codes a lane would put the lanes of a V write on half the banks).
  uint32_t so[NOP][NL];
#pragma unroll
  for (int o = 0; o < NOP; ++o)
#pragma unroll
    for (int u = 0; u < NL; ++u) {
      const int row = 16 * gw + RPL * u + lrow;
      const int sw = of_v || o == 1 ? ST::sv(row) : ST::gk(row & 15);
      so[o][u] = (uint32_t)(row * (2 * D) + 16 * (lch ^ sw)) + (of_v || o == 1 ? (uint32_t)(NG * TB) : 0u);
    }
  const auto store = [&](int o, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NL; ++u) {
      char* to = lds + stage * TB;
      *reinterpret_cast<u32x4*>(to + so[o][u]) = widen8<DT>(rx[o][u][0], rs[o], rx[o][u][1], rs[o]);
    }
  };

  // The stages of tile 0: K's, and with two groups V's.
  look(0);
  int page_v = page_of(0);  // one group: the tile at hand's, for V
  float scale_v = NG == 1 ? scale_of(NOP - 1, 0) : 1.f;
  if (NG == 1 || group == 0) {
    load(0, 0, page_v);
    rs[0] = scale_of(0, 0);
  }
  u32x4 qreg[NKS];
  {
    const int ps = valid ? pos : pos_lo;  // (an invalid row's are zeroed)
    const T* qrow = static_cast<const T*>(p.q.ptr) + (int64_t)head * p.q.sh +
                    (varlen ? (tok0 + ps) * p.q.ss : (int64_t)b * p.q.sb + (int64_t)ps * p.q.ss);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qreg[ks] = *reinterpret_cast<const u32x4*>(qrow + 16 * ks + 8 * hh);
  }
  if (NG == 1 || group == 0) store(0, 0);
  const int lead = NG == 2 ? 1 - group : 0;
  if constexpr (NG == 2) {
    load(0, lead, page_of(lead));
    rs[0] = scale_of(0, lead);
#pragma unroll
    for (int u = 0; u < NL; ++u) so[0][u] += lead * TB;
  }
  if (!valid) {
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qreg[ks] = u32x4{0u, 0u, 0u, 0u};
  }

  // LDS read offsets (the masks are no-ops on the values; they give the compiler
  // known bounds).
  uint32_t ka[NKS];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks)
    ka[ks] = (uint32_t)(pi_key(i) * (2 * D) + 16 * ((2 * ks + hh) ^ ST::gk(pi_key(i)))) & ((TB / 2 - 1) & ~15u);
  uint32_t vb[NDB];
  {
    const int q = lane >> 4, ii = lane & 15;
    const int rowl = 8 * (q >> 1) + (ii >> 2);
    const int f = (ST::CPR == 16) ? (ii >> 2) : ((ii >> 3) & 1);  // sv(rowl) / 4
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      vb[db] = (uint32_t)(rowl * (2 * D) + 16 * (4 * (db ^ f) + 2 * (q & 1) + ((ii & 3) >> 1)) + 8 * (ii & 1)) &
               ((TB - 1) & ~7u);
  }

  f32x16 acc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) acc[db] = f32x16{};
  float m_run = -__builtin_inff(), l_run = 0.f;
  const float c = dm.c;
  f32x16 sc[2];    // S^T of the current tile (MFMA phase -> softmax phase)
  u32x4 pk[2][2];  // P^T operands (softmax phase -> next MFMA phase)

  using BT = std::true_type;
  using BF = std::false_type;

  // MFMA phase of tile j: P*V of the tile before and S^T of this one.  par: j's parity.
  const auto mphase = [&](int mj, auto pvc, auto sc_, auto par) __attribute__((always_inline)) {
    constexpr bool DO_PV = decltype(pvc)::value;
    constexpr bool DO_S = decltype(sc_)::value;
    constexpr int NPV = DO_PV ? 4 * NDB : 0;
    constexpr int NS = DO_S ? 2 * NKS : 0;
    constexpr int PAR = decltype(par)::value ? 1 : 0;
    if constexpr (NG == 1 && DO_S) {  // the codes that the softmax phase stores
      if (mj + 1 - base >= 64) look(mj + 1);
      load(1, mj, page_v);
      rs[1] = scale_v;
      page_v = page_of(mj + 1);
      scale_v = scale_of(1, mj + 1);
      load(0, mj + 1, page_v);
      rs[0] = scale_of(0, mj + 1);
    }
    const char* ck = lds + (NG == 2 ? PAR * TB : 0);
    const char* cv = lds + NG * TB + (NG == 2 ? (1 - PAR) * TB : 0);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(3);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 opv[NPV > 0 ? NPV : 1];
    u32x4 opk[NS > 0 ? NS : 1];
    if constexpr (DO_PV) {
#pragma unroll
      for (int j = 0; j < NPV; ++j) {
        const int mb = j / (2 * NDB), kk = (j / NDB) & 1, db = j % NDB;
        const int ro = (32 * mb + 16 * kk) * (2 * D);
        const u32x2 lo = ld_tr(cv + vb[db] + ro);
        const u32x2 hi = ld_tr(cv + vb[db] + ro + 4 * (2 * D));
        opv[j] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    }
    if constexpr (DO_S) {
#pragma unroll
      for (int j = 0; j < NS; ++j) opk[j] = *reinterpret_cast<const u32x4*>(ck + (j & 1) * 32 * (2 * D) + ka[j >> 1]);
    }
    if constexpr (DO_PV) {
#pragma unroll
      for (int j = 0; j < NPV; ++j) {
        const int mb = j / (2 * NDB), kk = (j / NDB) & 1, db = j % NDB;
        acc[db] = E::mfma(opv[j], pk[mb][kk], acc[db]);
      }
    }
    if constexpr (DO_S) {
      sc[0] = f32x16{};
      sc[1] = f32x16{};
#pragma unroll
      for (int j = 0; j < NS; ++j) sc[j & 1] = E::mfma(opk[j], qreg[j >> 1], sc[j & 1]);
    }
    if constexpr (NG == 2 && DO_S) {
#pragma unroll
      for (int u = 0; u < NL; ++u)
        *reinterpret_cast<u32x4*>(lds + (so[0][u] ^ (uint32_t)(PAR * TB))) =
            widen8<DT>(rx[0][u][0], rs[0], rx[0][u][1], rs[0]);
    }
    mphase_prefetch<NPV, NPV + NS, PF, 0>();
    mphase_pipe<NPV, NPV + NS, PF, 0>();
    if constexpr (DO_S) {
      pin(sc[0]);
      pin(sc[1]);
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) pin(acc[db]);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(0);
    phase_barrier();
  };

  // Softmax phase of tile j, which stores the next tile's codes and loads ahead.
  const auto vphase = [&](int j, auto first_c, auto par) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(first_c)::value;
    if constexpr (NG == 2) {
      if (j + 1 + lead - base >= 64) look(j + 1 + lead);
      load(0, j + 1 + lead, page_of(j + 1 + lead));
      rs[0] = scale_of(0, j + 1 + lead);
    }
    const int key0 = tile_of(j) * ST::kKeys;
    float row_t = 0.f;  // added to every score of the lane
    cap_scores<16>(sc, p.mod);
    if (p.mod.slopes != nullptr)
      row_t = bias_scores<16>(sc, slope, key0 + span.rel0, key0 + ST::kKeys - 1 <= qpos_lo,
                              [](int e) { return 32 * (e >> 4) + key_of(e & 15, 0); });
    if (key0 + ST::kKeys > span.full_hi) mask_tile(sc, span.vis - key0);
    float rs0 = 0.f, rs1 = 0.f;
    bool keep = false;
    if constexpr (!FIRST) keep = __builtin_amdgcn_ballot_w64(m_run == -__builtin_inff()) == 0;
    if (keep) {
      const float nmc = (row_t - m_run) * c;
      rs0 = softmax_exp<DT>(sc[0], nmc, c, pk[0]);
      rs1 = softmax_exp<DT>(sc[1], nmc, c, pk[1]);
      keep = __builtin_amdgcn_ballot_w64(!(rs0 + rs1 <= kRescaleSum)) == 0;
    }
    if (!keep) {
      float nmc;
      if constexpr (FIRST) {  // (nothing to rescale yet)
        f32x16 none[1] = {f32x16{}};
        nmc = softmax_rebase_at<1>(sc, row_t, m_run, l_run, none, c);
      } else {
        nmc = softmax_rebase_at<NDB>(sc, row_t, m_run, l_run, acc, c);
      }
      rs0 = softmax_exp<DT>(sc[0], nmc, c, pk[0]);
      rs1 = softmax_exp<DT>(sc[1], nmc, c, pk[1]);
    }
    if constexpr (NG == 1) {
      store(0, 0);
      store(1, 0);
    }
    l_run += rs0 + rs1;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) pin(pk[mb][kk]);
    phase_barrier();
  };

  phase_barrier();
  if (group == 1) phase_barrier();  // (a phase behind group 0)
  if (n > 0) {
    mphase(0, BF{}, BT{}, BF{});
    vphase(0, BT{}, BF{});
    int j = 1;
    for (; j + 1 < n; j += 2) {
      mphase(j, BT{}, BT{}, BT{});
      vphase(j, BF{}, BT{});
      mphase(j + 1, BT{}, BT{}, BF{});
      vphase(j + 1, BF{}, BF{});
    }
    if (j < n) {
      mphase(j, BT{}, BT{}, BT{});
      vphase(j, BF{}, BT{});
      mphase(n, BT{}, BF{}, BF{});
    } else {
      mphase(n, BT{}, BF{}, BT{});
    }
  }
  if (NG == 2 && group == 0) phase_barrier();
  __syncthreads();

  const float l_tot = xhalf_sum(l_run);
  if constexpr (KC) {
    // Lane (i, hh) holds dims 32 db + 8 j + 4 hh + 0..3 of its row in acc[db][4 j ..].
    if (!valid) return;
    float* wa = p.ws_acc + part * D + 4 * hh;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(wa + 32 * db + 8 * j) =
            f32x4{acc[db][4 * j], acc[db][4 * j + 1], acc[db][4 * j + 2], acc[db][4 * j + 3]};
    if (hh == 0) {
      p.ws_m[part] = m_run == -__builtin_inff() ? kEmptyRef : __builtin_fmaf(m_run, c, p.mod.shift2);
      p.ws_l[part] = l_tot;
    }
    return;
  }
  const float inv = l_tot == 0.f ? 0.f : 1.0f / l_tot;  // (a row that sees no key: zeros)
  if (p.lse != nullptr && valid && hh == 0) {
    const int64_t li = varlen ? (tok0 + pos) * dm.Hq + head : ((int64_t)b * dm.Hq + head) * dm.Sq + pos;
    p.lse[li] = (__builtin_fmaf(m_run, c, p.mod.shift2) + __log2f(l_tot)) * kLn2;
  }
  // The wave's 32 x D output goes through LDS (row-major, 16-byte chunks
  // XOR-swizzled by row; in the former stages), so that it leaves as whole
  // rows.
  constexpr int CPR16 = 2 * D / 16, RPI = 64 / CPR16;
  char* ot = lds + wave * (32 * 2 * D);
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x2 x;
      x[0] = E::pack2(acc[db][4 * j] * inv, acc[db][4 * j + 1] * inv);
      x[1] = E::pack2(acc[db][4 * j + 2] * inv, acc[db][4 * j + 3] * inv);
      const int ch = (4 * db + j) ^ (i & (CPR16 - 1));
      *reinterpret_cast<u32x2*>(ot + i * (2 * D) + ch * 16 + 8 * hh) = x;
    }
  __builtin_amdgcn_s_waitcnt(kLgkm0);  // this wave's LDS writes before its reads
  const int cc = lane % CPR16;
#pragma unroll
  for (int ri = 0; ri < 32 / RPI; ++ri) {
    const int rr = RPI * ri + lane / CPR16;
    const u32x4 x = *reinterpret_cast<const u32x4*>(ot + rr * (2 * D) + ((cc ^ (rr & (CPR16 - 1))) * 16));
    const int r2 = wave * 32 + rr, g2 = (int)(__umul24(r2, p.bm_mul) >> 16), pos2 = pos_lo + r2 - g2 * p.block_m;
    if (g2 < dm.G && pos2 < sq) {
      T* orow = static_cast<T*>(const_cast<void*>(p.o.ptr)) + (int64_t)(kvh * dm.G + g2) * p.o.sh +
                (varlen ? (tok0 + pos2) * p.o.ss : (int64_t)b * p.o.sb + (int64_t)pos2 * p.o.ss);
      *reinterpret_cast<u32x4*>(orow + 8 * cc) = x;
    }
  }
}

template <int DT, int D> static hipError_t launch_chunk8_t(Fwd8Params p, hipStream_t stream) {
  const int64_t total = (int64_t)p.n_mblk * p.dm.Hkv * (p.kv_splits > 0 ? p.kv_splits : p.dm.B);
  if (total <= 0) return hipSuccess;
  if (total >= ((int64_t)1 << 31) - 1) return hipErrorInvalidValue;
  set_item_order(p, p.n_mblk, true, kDealPairs(D));
  if (p.kv_splits > 0) p.div_items = make_fast_div((uint32_t)p.kv_splits);
  p.div_mblk = make_fast_div((uint32_t)p.n_mblk);
  p.div_hkv = make_fast_div((uint32_t)p.dm.Hkv);
  p.bm_mul = (65536u + (uint32_t)p.block_m - 1) / (uint32_t)p.block_m;
  const dim3 grid((unsigned)(total + (p.kv_splits > 0 ? 1 : 0)));
  if constexpr (D == 128) {
    if (p.block_m * p.dm.G > kShortRows) {
      if (p.kv_splits > 0) hipLaunchKernelGGL((gqa_chunk8_kernel<DT, D, 2, true>), grid, dim3(512), 0, stream, p);
      else hipLaunchKernelGGL((gqa_chunk8_kernel<DT, D, 2, false>), grid, dim3(512), 0, stream, p);
      return hipGetLastError();
    }
  }
  if (p.kv_splits > 0) hipLaunchKernelGGL((gqa_chunk8_kernel<DT, D, 1, true>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((gqa_chunk8_kernel<DT, D, 1, false>), grid, dim3(256), 0, stream, p);
  return hipGetLastError();
}

// p.block_m = chunk8_rows(..) / G, p.n_mblk accordingly.
hipError_t launch_chunk8(const Fwd8Params& p, int dtype, hipStream_t stream) {
  if (p.block_shift < 4 || (p.block_table == nullptr && p.dm.Skv > 0)) return hipErrorInvalidValue;
  if (dtype == 0) return p.dm.D == 128 ? launch_chunk8_t<0, 128>(p, stream) : launch_chunk8_t<0, 64>(p, stream);
  return p.dm.D == 128 ? launch_chunk8_t<1, 128>(p, stream) : launch_chunk8_t<1, 64>(p, stream);
}

}  // namespace gqa
