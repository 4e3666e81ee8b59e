// gqa_chunk8.hip — attention over a paged cache in 8 bits (gqa_cache8.hpp) for more
// query rows than gqa_decode8.hip takes: verification of drafts, chunks of prompts,
// whole prompts.
//
// Rows, products, softmax, changed scores and the key chunks' partials are those of
// gqa_scored.hip: 128 packed rows in four waves, S^T = K Q^T and O^T += V^T P^T by
// 32x32x16 MFMAs over 64-key tiles, lazily rescaled online softmax.  What differs is
// the way of a tile into LDS: its codes are loaded into registers a phase ahead,
// widened there to the queries' type with their page's power of two (exact), and
// stored in the swizzled layout of the 16-bit tiles.  A workgroup widens a code once,
// for all four waves: an instruction per two codes, 32 a lane and tile beside the
// softmax of 32 scores.  (Each wave widening what it reads from LDS would take four
// times as many.)  Registers are the second stage, so K and V have one each in LDS.
//
// Tile j: MFMA phase (P V of the tile before, S of this one), barrier, softmax
// phase, which first stores K(j + 1) and V(j) where K(j) and V(j - 1) were, then
// loads K(j + 2) and V(j + 1); barrier.
#include <algorithm>
#include <type_traits>

#include "gqa_cache8.hpp"
#include "gqa_fwd_parts.hpp"
#include "gqa_lds.hpp"
#include "gqa_score.hpp"

namespace gqa {

// KC: key chunks (p.kv_splits > 0), whose partials launch_scored_combine joins.
template <int DT, int D, bool KC>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void gqa_chunk8_kernel(Fwd8Params p) {
  using E = Elem<DT>;
  using T = typename E::T;
  using ST = FwdStage<D>;
  constexpr int NDB = D / 32;   // 32-wide d blocks of O^T
  constexpr int NKS = D / 16;   // k-steps of S^T
  constexpr int PF = 6;         // MFMA slots of LDS-read lookahead
  constexpr int TB = ST::kTileBytes;
  constexpr int CPR8 = D / 16;  // 16-code chunks per row
  constexpr int RPL = 64 / CPR8;  // rows per load of a wave: 8 or 16
  constexpr int NL = 16 / RPL;    // loads of a wave's 16 rows
  __shared__ __attribute__((aligned(1024))) char lds0_v[TB];
  __shared__ __attribute__((aligned(1024))) char lds1_k[TB];

  const Dims& dm = p.dm;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6) & 3;
  const int i = lane & 31, hh = lane >> 5;
  const bool varlen = p.q_len != nullptr;

  // Work item: as gqa_scored.hip.
  const int n_items = KC ? p.n_mblk * p.kv_splits : p.n_mblk;
  const int w = xcd_remap(blockIdx.x, n_items * dm.Hkv * dm.B);
  int bh, mrank, chunk = 0;
  item_of(p, w, n_items, bh, mrank);
  if (p.xcd_heads > 1) bh = turned_pair(p, bh, mrank);
  if constexpr (KC) {
    chunk = fast_div(mrank, p.div_mblk.mul, p.div_mblk.shift);
    mrank -= chunk * p.n_mblk;
  }
  const int pid_m = dm.causal ? p.n_mblk - 1 - mrank : mrank;
  const int b = fast_div(bh, p.div_hkv.mul, p.div_hkv.shift), kvh = bh - b * dm.Hkv;
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
  int tb = 0, n = (span.end + ST::kKeys - 1) / ST::kKeys;
  if constexpr (KC) {
    tb = chunk * p.kv_chunk_tiles;
    n = max(min(n - tb, p.kv_chunk_tiles), 0);
  }
  // The chunk's partial of this lane's row, in the split workspace's layout.
  const int64_t part = (((int64_t)b * dm.Hq + head) * dm.Sq + pos) * p.kv_splits + chunk;
  if (KC && n == 0) {  // (no sum: the combine reads nothing else of it)
    if (valid && hh == 0) {
      p.ws_m[part] = kEmptyRef;
      p.ws_l[part] = 0.f;
    }
    return;
  }
  const bool back = p.mod.slopes != nullptr && dm.causal;
  const auto tile_of = [&](int j) __attribute__((always_inline)) { return tile_at(tb, n, j, back); };

  // This wave's rows of a tile: 16 wave + 0..15, which lie in one page.  Rows past the
  // item's last key, or the last that the block sees, load as zeros.
  const int rows_ld = KC ? min(span.end, (tb + n) * ST::kKeys) : span.end;
  const uint32_t kss = (uint32_t)p.k.ss, vss = (uint32_t)p.v.ss;
  const char* kbh = static_cast<const char*>(p.k.ptr) + (int64_t)kvh * p.k.sh;
  const char* vbh = static_cast<const char*>(p.v.ptr) + (int64_t)kvh * p.v.sh;
  const int* keb = p.ke.e + kvh * p.ke.sh;
  const int* veb = p.ve.e + kvh * p.ve.sh;
  const int* table_row = p.block_table + (int64_t)b * p.table_stride;
  const auto page_of = [&](int j) __attribute__((always_inline)) {  // (-1: no rows)
    const int key = tile_of(j) * ST::kKeys + 16 * wave;
    return key < rows_ld ? load_uniform(table_row + (key >> p.block_shift)) : -1;
  };
  const auto scale_of = [&](const int* e, int64_t sb, int page) __attribute__((always_inline)) {
    return page < 0 ? 1.f : exp_scale(clamp_exp(load_uniform(e + (int64_t)page * sb)));
  };
  const int lrow = lane / CPR8, lch = lane % CPR8;
  const auto load = [&](u32x4 (&x)[NL], const char* head_ptr, int64_t sb, uint32_t ss, int j, int page)
                        __attribute__((always_inline)) {
    const int key = tile_of(j) * ST::kKeys + 16 * wave, rows = rows_ld - key;
    __amdgpu_buffer_rsrc_t rt = make_rsrc(head_ptr, 0u);
    if (rows > 0) {
      const int64_t slot = key & ((1 << p.block_shift) - 1);
      rt = make_rsrc(head_ptr + (int64_t)page * sb + slot * ss, (uint32_t)(min(rows, 16) - 1) * ss + D);
    }
    const uint32_t off = (uint32_t)lrow * ss + 16u * lch;
#pragma unroll
    for (int u = 0; u < NL; ++u)
      x[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rt, off, (uint32_t)(u * RPL) * ss, 0));
  };
  // Sixteen codes a lane and load into two 16-byte chunks of the 16-bit tile.
  const auto store = [&](char* tile, const u32x4 (&x)[NL], float scale, bool is_k) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NL; ++u) {
      const int row = 16 * wave + RPL * u + lrow;
      const int sw = is_k ? ST::gk(row & 15) : ST::sv(row);
      char* to = tile + row * (2 * D);
      *reinterpret_cast<u32x4*>(to + 16 * ((2 * lch) ^ sw)) = widen8<DT>(x[u][0], scale, x[u][1], scale);
      *reinterpret_cast<u32x4*>(to + 16 * ((2 * lch + 1) ^ sw)) = widen8<DT>(x[u][2], scale, x[u][3], scale);
    }
  };

  u32x4 rk[NL], rv[NL];
  int id_v = page_of(0), id_k = page_of(1);
  load(rk, kbh, p.k.sb, kss, 0, id_v);
  float sk = scale_of(keb, p.ke.sb, id_v), sv = scale_of(veb, p.ve.sb, id_v);
  u32x4 qreg[NKS];
  {
    const int ps = valid ? pos : pos_lo;  // (an invalid row's are zeroed)
    const T* qrow = static_cast<const T*>(p.q.ptr) + (int64_t)head * p.q.sh +
                    (varlen ? (tok0 + ps) * p.q.ss : (int64_t)b * p.q.sb + (int64_t)ps * p.q.ss);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qreg[ks] = *reinterpret_cast<const u32x4*>(qrow + 16 * ks + 8 * hh);
  }
  store(lds1_k, rk, sk, true);
  load(rv, vbh, p.v.sb, vss, 0, id_v);
  load(rk, kbh, p.k.sb, kss, 1, id_k);
  sk = scale_of(keb, p.ke.sb, id_k);
  id_v = id_k;
  id_k = page_of(2);
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

  // MFMA phase of tile j: P*V of the tile before and S^T of this one.
  const auto mphase = [&](auto pvc, auto sc_) __attribute__((always_inline)) {
    constexpr bool DO_PV = decltype(pvc)::value;
    constexpr bool DO_S = decltype(sc_)::value;
    constexpr int NPV = DO_PV ? 4 * NDB : 0;
    constexpr int NS = DO_S ? 2 * NKS : 0;
    const char* ck = lds1_k;
    const char* cv = lds0_v;
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

  // Softmax phase of tile j.
  const auto vphase = [&](int j, auto first_c) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(first_c)::value;
    store(lds1_k, rk, sk, true);
    store(lds0_v, rv, sv, false);
    load(rk, kbh, p.k.sb, kss, j + 2, id_k);
    load(rv, vbh, p.v.sb, vss, j + 1, id_v);
    sk = scale_of(keb, p.ke.sb, id_k);
    sv = scale_of(veb, p.ve.sb, id_v);
    id_v = id_k;
    id_k = page_of(j + 3);
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
    l_run += rs0 + rs1;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) pin(pk[mb][kk]);
    phase_barrier();
  };

  phase_barrier();
  if (n > 0) {
    mphase(BF{}, BT{});
    vphase(0, BT{});
    for (int j = 1; j < n; ++j) {
      mphase(BT{}, BT{});
      vphase(j, BF{});
    }
    mphase(BT{}, BF{});
  }
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
  // XOR-swizzled by row; two waves a former stage), so that it leaves as whole
  // rows.
  constexpr int CPR16 = 2 * D / 16, RPI = 64 / CPR16;
  char* ot = (wave < 2 ? lds1_k : lds0_v) + (wave & 1) * (32 * 2 * D);
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
  const int per_bh = p.kv_splits > 0 ? p.n_mblk * p.kv_splits : p.n_mblk;
  const int64_t total = (int64_t)per_bh * p.dm.Hkv * p.dm.B;
  if (total <= 0) return hipSuccess;
  if (total >= (int64_t)1 << 31) return hipErrorInvalidValue;
  set_item_order(p, per_bh, true, kDealPairs(D));
  p.div_mblk = make_fast_div((uint32_t)p.n_mblk);
  p.div_hkv = make_fast_div((uint32_t)p.dm.Hkv);
  p.bm_mul = (65536u + (uint32_t)p.block_m - 1) / (uint32_t)p.block_m;
  if (p.kv_splits > 0)
    hipLaunchKernelGGL((gqa_chunk8_kernel<DT, D, true>), dim3((unsigned)total), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((gqa_chunk8_kernel<DT, D, false>), dim3((unsigned)total), dim3(256), 0, stream, p);
  return hipGetLastError();
}

// p.block_m = kShortRows / G, p.n_mblk accordingly.
hipError_t launch_chunk8(const Fwd8Params& p, int dtype, hipStream_t stream) {
  if (p.block_shift < 4 || p.block_table == nullptr) return hipErrorInvalidValue;
  if (dtype == 0) return p.dm.D == 128 ? launch_chunk8_t<0, 128>(p, stream) : launch_chunk8_t<0, 64>(p, stream);
  return p.dm.D == 128 ? launch_chunk8_t<1, 128>(p, stream) : launch_chunk8_t<1, 64>(p, stream);
}

}  // namespace gqa
