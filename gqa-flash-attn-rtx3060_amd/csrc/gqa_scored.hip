// gqa_scored.hip — single-pass forward with changed scores (gqa_score.hpp):
// prompts, chunks and packed documents, over contiguous or paged K/V.
//
// Rows, tiles and products are those of gqa_fwd.hip (group-packed query rows, S^T
// = K Q^T and O^T += V^T P^T by 32x32x16 MFMAs, 64-key tiles written straight into
// LDS, lazily rescaled online softmax).  The workgroup is not: 128 rows in four
// waves, two workgroups a CU, each with two stages of K and of V (64 KiB at
// head_dim 128).  With changed scores the vector ALU is the bound (gqa_score.hpp),
// and what hides the matrix products, the loads' latency and a workgroup's start
// and end is the other workgroup of the CU, which no barrier couples to this one;
// the two wave groups of gqa_fwd.hip's workgroup wait for each other every phase.
// Measured, us, gqa_fwd.hip's form with the same changes / this one: 8192 causal
// tokens with a cap, head_dim 128 607 / 594, head_dim 64 500 / 406; with a distance
// bias, head_dim 64 380 / 309; documents in 2 x 8192 tokens 208 / 170 (580 TFLOP/s
// of visible pairs); 4 x 777 with a cap and a prefix 42.7 / 39.9; 2 x 500 tokens over
// 6001 keys in 4 chunks at head_dim 64, joined by gqa_split_reduce_kernel, 56.2 / 54.8
// (41-46 with the combine below).  Wave priorities by phase or by slot, a
// workgroup started half a tile late and Q loaded ahead of the spans: all within
// the noise of 2 %, or slower.
//
// Tile j: MFMA phase (P V of the tile before, S of this one), barrier, softmax
// phase, which refills the stages just read (K(j+2), V(j+1)) and waits for the
// loads of the phase before it, barrier.
#include <algorithm>
#include <type_traits>

#include "gqa_common.hpp"
#include "gqa_fwd_parts.hpp"
#include "gqa_lds.hpp"
#include "gqa_params.hpp"
#include "gqa_score.hpp"

namespace gqa {

constexpr int kScoredThreads = 256;

// KC: key chunks (FwdParams::kv_splits > 0), whose partials the combine below
// joins.  Scores, sums and accumulators are fp32; P is rounded to the inputs' type for
// its matrix product with V (half a step of each probability: outputs of bf16
// prompts off by 2.2e-3 of their size against float64, with fp32 probabilities 1.66e-3).
template <int DT, int D, int PG, bool KC>
__global__ __launch_bounds__(kScoredThreads) __attribute__((amdgpu_waves_per_eu(2))) void gqa_scored_kernel(
    FwdModParams p) {
  using E = Elem<DT>;
  using T = typename E::T;
  using ST = FwdStage<D>;
  constexpr int CPR = ST::CPR;
  constexpr bool PAGED = PG != 0;
  constexpr int NDB = D / 32;  // 32-wide d blocks of O^T
  constexpr int NKS = D / 16;  // k-steps of S^T
  constexpr int PF = 6;        // MFMA slots of LDS-read lookahead
  constexpr int TB = ST::kTileBytes;
  // An array a stage, so that the compiler can tell the LDS-DMA targets from the
  // stages being read; all below 64 KiB, the reach of a read's offset field.
  __shared__ __attribute__((aligned(1024))) char lds0_v0[TB];
  __shared__ __attribute__((aligned(1024))) char lds0_v1[TB];
  __shared__ __attribute__((aligned(1024))) char lds1_k0[TB];
  __shared__ __attribute__((aligned(1024))) char lds1_k1[TB];

  const Dims& dm = p.dm;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6) & 3;
  const int i = lane & 31, hh = lane >> 5;
  const bool varlen = p.q_len != nullptr;

  // Work item: a query block of one (b, kv head), heavy (late) blocks first under
  // causal; with key chunks the blocks of one chunk side by side.
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
  const int skv = PAGED ? min(max(load_uniform(p.seq_lens + b), 0), dm.Skv) : dm.Skv;
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
  int tb = span.beg / ST::kKeys, n = (span.end + ST::kKeys - 1) / ST::kKeys - tb;
  if constexpr (KC) {
    const int skip = chunk * p.kv_chunk_tiles;
    tb += skip;
    n = max(min(n - skip, p.kv_chunk_tiles), 0);
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
  auto tile_of = [&](int j) __attribute__((always_inline)) { return tile_at(tb, n, j, back); };

  // Rows up to the last one that the block sees (no padding behind a document is
  // multiplied with its probabilities of zero); what lies past it loads as zeros
  // and is masked.
  const int rows_ld = span.end;
  const uint32_t kssb = (uint32_t)(2 * p.k.ss), vssb = (uint32_t)(2 * p.v.ss);
  const char* kbh = static_cast<const char*>(p.k.ptr) + 2 * ((PAGED ? 0 : (int64_t)b * p.k.sb) + (int64_t)kvh * p.k.sh);
  const char* vbh = static_cast<const char*>(p.v.ptr) + 2 * ((PAGED ? 0 : (int64_t)b * p.v.sb) + (int64_t)kvh * p.v.sh);
  const bool flat = !PAGED && rows_ld > 0;
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(kbh, flat ? (uint32_t)(rows_ld - 1) * kssb + 2 * D : 0u);
  const __amdgpu_buffer_rsrc_t rv = make_rsrc(vbh, flat ? (uint32_t)(rows_ld - 1) * vssb + 2 * D : 0u);
  const int* table_row = PAGED ? p.block_table + (int64_t)b * p.table_stride : nullptr;
  const int lrow = lane / CPR;
  const uint32_t koff =
      (uint32_t)(lrow * kssb) + 16u * (uint32_t)((lane % CPR) ^ ST::gk((wave * ST::RPI + lrow) & 15));
  const uint32_t voff = (uint32_t)(lrow * vssb) + 16u * (uint32_t)((lane % CPR) ^ ST::sv(lrow));
  using Blocks = FwdTileBlocks<D, PG>;
  auto ids = [&](int j) __attribute__((always_inline)) -> Blocks {  // block(s) of the j-th tile
    return tile_blocks<D, PG>(table_row, p.block_shift, rows_ld, tile_of(j), wave);
  };
  auto issue_k = [&](char* stage, int j, const Blocks& blk) __attribute__((always_inline)) {
    issue_fwd_tile<D, PG>(stage, kbh, rk, kssb, koff, p.k.sb, p.block_shift, rows_ld, tile_of(j), blk, true, wave,
                          lane);
  };
  auto issue_v = [&](char* stage, int j, const Blocks& blk) __attribute__((always_inline)) {
    issue_fwd_tile<D, PG>(stage, vbh, rv, vssb, voff, p.v.sb, p.block_shift, rows_ld, tile_of(j), blk, false, wave,
                          lane);
  };

  // Loads in the order of their first use: K(0) and Q, K(1), V(0).  An invalid
  // row loads the block's first one and is zeroed when it has landed.
  Blocks id_v = ids(0), id_k = ids(1);  // of the next V and K tiles to load
  issue_k(lds1_k0, 0, id_v);
  u32x4 qreg[NKS];
  {
    const int ps = valid ? pos : pos_lo;
    const T* qrow = static_cast<const T*>(p.q.ptr) + (int64_t)head * p.q.sh +
                    (varlen ? (tok0 + ps) * p.q.ss : (int64_t)b * p.q.sb + (int64_t)ps * p.q.ss);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qreg[ks] = *reinterpret_cast<const u32x4*>(qrow + 16 * ks + 8 * hh);
  }
  __builtin_amdgcn_sched_barrier(0);
  issue_k(lds1_k1, 1, id_k);
  issue_v(lds0_v0, 0, id_v);
  id_v = id_k;
  id_k = ids(2);

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
    const int f = (CPR == 16) ? (ii >> 2) : ((ii >> 3) & 1);  // sv(rowl) / 4
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

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using BT = std::true_type;
  using BF = std::false_type;

  // MFMA phase of tile j (j even: PAR = 0): P*V of the tile before (V stage 1 -
  // PAR) and S^T of this one (K stage PAR).
  auto mphase = [&](auto par, auto pvc, auto sc_) __attribute__((always_inline)) {
    constexpr int PAR = decltype(par)::value;
    constexpr bool DO_PV = decltype(pvc)::value;
    constexpr bool DO_S = decltype(sc_)::value;
    constexpr int NPV = DO_PV ? 4 * NDB : 0;
    constexpr int NS = DO_S ? 2 * NKS : 0;
    const char* ck = PAR == 0 ? lds1_k0 : lds1_k1;
    const char* cv = PAR == 0 ? lds0_v1 : lds0_v0;
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
  auto vphase = [&](auto par, int j, auto first_c) __attribute__((always_inline)) {
    constexpr int PAR = decltype(par)::value;
    constexpr bool FIRST = decltype(first_c)::value;
    issue_k(PAR == 0 ? lds1_k0 : lds1_k1, j + 2, id_k);
    issue_v(PAR == 0 ? lds0_v1 : lds0_v0, j + 1, id_v);
    id_v = id_k;
    id_k = ids(j + 3);
    const int key0 = tile_of(j) * ST::kKeys;
    float row_t = 0.f;  // added to every score of the lane
    cap_scores<16>(sc, p.mod);
    if (p.mod.slopes != nullptr)
      row_t = bias_scores<16>(sc, slope, key0 + span.rel0, key0 + ST::kKeys - 1 <= qpos_lo,
                              [](int e) { return 32 * (e >> 4) + key_of(e & 15, 0); });
    if (key0 + ST::kKeys > span.full_hi || key0 < span.full_lo) mask_tile_span(sc, span.vis - key0, span.lo - key0);
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
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * ST::NI));  // all but this phase's loads
    phase_barrier();
  };

  __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * ST::NI));  // K(0) and Q
  pin(slope);
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) pin(qreg[ks]);
  if (__builtin_amdgcn_ballot_w64(!valid) != 0) {
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qreg[ks] = valid ? qreg[ks] : u32x4{0u, 0u, 0u, 0u};
  }
  phase_barrier();
  if (n > 0) {
    mphase(I0{}, BF{}, BT{});
    vphase(I0{}, 0, BT{});
    int j = 1;
    for (; j + 2 <= n; j += 2) {
      mphase(I1{}, BT{}, BT{});
      vphase(I1{}, j, BF{});
      mphase(I0{}, BT{}, BT{});
      vphase(I0{}, j + 1, BF{});
    }
    if (j < n) {
      mphase(I1{}, BT{}, BT{});
      vphase(I1{}, j, BF{});
      mphase(I0{}, BT{}, BF{});
    } else {
      mphase(I1{}, BT{}, BF{});
    }
  }
  // No LDS-DMA load may still be writing when the stages are reused, nor when
  // the workgroup ends.
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
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
      p.ws_m[part] = m_run == -__builtin_inff() ? kEmptyRef : log2_ref(p, m_run, c);
      p.ws_l[part] = l_tot;
    }
    return;
  }
  const float inv = l_tot == 0.f ? 0.f : 1.0f / l_tot;  // (a row that sees no key: zeros)
  if (p.lse != nullptr && valid && hh == 0) {
    const int64_t li = varlen ? (tok0 + pos) * dm.Hq + head : ((int64_t)b * dm.Hq + head) * dm.Sq + pos;
    p.lse[li] = (log2_ref(p, m_run, c) + __log2f(l_tot)) * kLn2;
  }
  // The wave's 32 x D output goes through LDS (row-major, 16-byte chunks
  // XOR-swizzled by row; two waves a former stage), so that it leaves as whole
  // rows.
  constexpr int CPR16 = 2 * D / 16, RPI = 64 / CPR16;
  char* ot = (wave < 2 ? lds1_k0 : lds1_k1) + (wave & 1) * (32 * 2 * D);
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

// Joins the key chunks' partials of each row: m* = max m_s, l = sum 2^(m_s - m*)
// l_s, o = sum 2^(m_s - m*) acc_s / l, over the partials with a sum.  A row's D / 4
// lanes take four columns each; NSG such groups share a row's chunks and meet in
// LDS, 1024 / (D NSG) rows a workgroup.  Memory-bound: a group takes four chunks
// at a time, and the accumulators of those with a sum.  Few chunks of many rows
// want many rows a workgroup (gqa_split_reduce_kernel, one row a workgroup, / this,
// us: 16000 rows of 4 chunks at head_dim 64 17.4 / 6.5, 32768 of 2 at head_dim 128
// 23 / 9.8, 3.5 TB/s).
template <int DT, int D, int NSG> __global__ __launch_bounds__(256) void gqa_scored_combine_kernel(ReduceParams p) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int ND4 = D / 4, R = 256 / (ND4 * NSG), BATCH = 4;
  const int t = threadIdx.x, d4 = t % ND4, sg = (t / ND4) % NSG, r = t / (ND4 * NSG);
  const int row = xcd_remap(blockIdx.x, gridDim.x) * R + r;
  const int bh = fast_div(row, p.div_sq.mul, p.div_sq.shift), pos = row - bh * p.Sq;
  const int b = fast_div(bh, p.div_hq.mul, p.div_hq.shift), h = bh - b * p.Hq;
  const bool varlen = p.q_len != nullptr;
  const bool live = row < p.B * p.Hq * p.Sq && (!varlen || pos < p.q_len[b]);
  const int S = live ? p.splits : 0;
  const float* wm = p.ws_m + (int64_t)row * p.splits;
  const float* wl = p.ws_l + (int64_t)row * p.splits;
  const float* wa = p.ws_acc + (int64_t)row * p.splits * D + 4 * d4;
  float m = kEmptyRef, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = sg; s0 < S; s0 += BATCH * NSG) {
    float mv[BATCH], lv[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int s = s0 + k * NSG;
      mv[k] = s < S ? wm[s] : kEmptyRef;
      lv[k] = s < S ? wl[s] : 0.f;
    }
    f32x4 av[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      av[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (lv[k] != 0.f) av[k] = *reinterpret_cast<const f32x4*>(wa + (int64_t)(s0 + k * NSG) * D);
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
  if constexpr (NSG > 1) {
    __shared__ float red_m[256], red_l[256];
    __shared__ f32x4 red_o[256];
    red_m[t] = m;
    red_l[t] = l;
    red_o[t] = o;
    __syncthreads();
    if (sg != 0) return;
#pragma unroll
    for (int k = 1; k < NSG; ++k) {
      const int at = t + k * ND4;
      const float mb = fmaxf(m, red_m[at]), a0 = fast_exp2(m - mb), a1 = fast_exp2(red_m[at] - mb);
      l = l * a0 + red_l[at] * a1;
      o = o * a0 + red_o[at] * a1;
      m = mb;
    }
  }
  if (!live) return;
  const int64_t tok = varlen ? (int64_t)p.q_start[b] + pos : 0;
  if (p.lse != nullptr && d4 == 0) p.lse[varlen ? tok * p.Hq + h : row] = (m + __log2f(l)) * kLn2;
  const float inv = l == 0.f ? 0.f : 1.0f / l;  // (a row that sees no key: zeros)
  T* orow = static_cast<T*>(const_cast<void*>(p.o.ptr)) +
            (varlen ? tok * p.o.ss + (int64_t)h * p.o.sh
                    : (int64_t)b * p.o.sb + (int64_t)h * p.o.sh + (int64_t)pos * p.o.ss);
  u32x2 x;
  x[0] = E::pack2(o[0] * inv, o[1] * inv);
  x[1] = E::pack2(o[2] * inv, o[3] * inv);
  *reinterpret_cast<u32x2*>(orow + 4 * d4) = x;
}

template <int DT, int D> static hipError_t launch_combine_t(ReduceParams p, hipStream_t stream) {
  const int64_t rows = (int64_t)p.B * p.Hq * p.Sq;
  if (rows <= 0) return hipSuccess;
  if (rows >= (int64_t)1 << 24) return hipErrorInvalidValue;
  p.div_sq = make_fast_div((uint32_t)p.Sq);
  p.div_hq = make_fast_div((uint32_t)p.Hq);
  const auto grid = [&](int nsg) { return dim3((unsigned)((rows * (D / 4) * nsg + 255) / 256)); };
  // (A thread's loop of chunks in at most two rounds of loads, up to one row a
  // workgroup.)
  constexpr int kMax = 1024 / D;
  if (p.splits <= 8)
    hipLaunchKernelGGL((gqa_scored_combine_kernel<DT, D, 1>), grid(1), dim3(256), 0, stream, p);
  else if (p.splits <= 32)
    hipLaunchKernelGGL((gqa_scored_combine_kernel<DT, D, 4>), grid(4), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((gqa_scored_combine_kernel<DT, D, kMax>), grid(kMax), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_scored_combine(const ReduceParams& p, int dtype, hipStream_t stream) {
  if (dtype == 0) return p.D == 128 ? launch_combine_t<0, 128>(p, stream) : launch_combine_t<0, 64>(p, stream);
  return p.D == 128 ? launch_combine_t<1, 128>(p, stream) : launch_combine_t<1, 64>(p, stream);
}

template <int DT, int D, int PG> static hipError_t launch_scored_t(FwdModParams p, hipStream_t stream) {
  const int per_bh = p.kv_splits > 0 ? p.n_mblk * p.kv_splits : p.n_mblk;
  const int64_t total = (int64_t)per_bh * p.dm.Hkv * p.dm.B;
  if (total <= 0) return hipSuccess;
  if (total >= (int64_t)1 << 31) return hipErrorInvalidValue;
  set_item_order(p, per_bh, PG > 0 || total > 2 * device_cu_count(), kDealPairs(D));
  p.div_mblk = make_fast_div((uint32_t)p.n_mblk);
  p.div_hkv = make_fast_div((uint32_t)p.dm.Hkv);
  p.bm_mul = (65536u + (uint32_t)p.block_m - 1) / (uint32_t)p.block_m;
  if (p.kv_splits > 0)
    hipLaunchKernelGGL((gqa_scored_kernel<DT, D, PG, true>), dim3((unsigned)total), dim3(kScoredThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((gqa_scored_kernel<DT, D, PG, false>), dim3((unsigned)total), dim3(kScoredThreads), 0, stream,
                       p);
  return hipGetLastError();
}

template <int PG> static hipError_t launch_scored_pg(const FwdModParams& p, int dtype, hipStream_t stream) {
  if (dtype == 0)
    return p.dm.D == 128 ? launch_scored_t<0, 128, PG>(p, stream) : launch_scored_t<0, 64, PG>(p, stream);
  return p.dm.D == 128 ? launch_scored_t<1, 128, PG>(p, stream) : launch_scored_t<1, 64, PG>(p, stream);
}

// p.block_m = kShortRows / G, p.n_mblk accordingly; paged as launch_paged_fwd.
hipError_t launch_scored(const FwdParams& in, int dtype, hipStream_t stream, const ScoreMod& mod) {
  FwdModParams p;
  static_cast<FwdParams&>(p) = in;
  p.mod = mod;
  if (p.n_split != 0) return hipErrorInvalidValue;
  if (p.block_table == nullptr) return launch_scored_pg<0>(p, dtype, stream);
  if ((1 << p.block_shift) < 512 / p.dm.D) return hipErrorInvalidValue;
  if (p.block_shift >= 6) return launch_scored_pg<1>(p, dtype, stream);
  const bool medium = p.block_shift >= 4 && (p.dm.D != 64 || (2 * p.k.ss) % 64 == 0);
  return medium ? launch_scored_pg<3>(p, dtype, stream) : launch_scored_pg<2>(p, dtype, stream);
}

}  // namespace gqa
