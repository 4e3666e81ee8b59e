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
template <int DT, int D>
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
  const float slope = row_slope(p.mod, head);
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

  FlatWalk<FlatWave<UNIT>, true> walk;
  walk.start(flat_wave, s);
  int from, cnt;
  while (walk.next(flat_wave, from, cnt)) {
    const int b = walk.b, skv = walk.skv;
    const int c0 = from * UNIT;
    const int sq = varlen ? min(max(load_uniform(p.q_len + b), 0), dm.Sq) : dm.Sq;
    const int64_t tok0 = varlen ? (int64_t)load_uniform(p.q_start + b) : 0;
    const bool valid = pos < sq;
    const int qpos = pos + (skv - sq), qpos_lo = skv - sq;
    const int prefix = seq_prefix(p.mod, b, skv);
    const int seen = max(qpos, prefix - 1), seen_lo = max(qpos_lo, prefix - 1);
    int c1 = min(c0 + cnt * UNIT, skv);
    if (dm.causal) c1 = min(c1, max(skv - 1, prefix - 1) + 1);
    const int tiles = max(c1 - c0 + TW - 1, 0) / TW;
    const int n = (tiles - wave + 3) >> 2;  // this wave's: wave, wave + 4, ...
    const int* table_row = p.block_table + (int64_t)b * p.table_stride;

    struct Pages {
      int id[NB];
    };
    const auto pages_of = [&](int it) {  // (not read past the piece's last key)
      Pages pg;
#pragma unroll
      for (int bl = 0; bl < NB; ++bl) {
        const int key = c0 + (4 * it + wave) * TW + 16 * bl;
        pg.id[bl] = key < c1 ? load_uniform(table_row + (key >> p.block_shift)) : -1;
      }
      return pg;
    };
    struct Scales {
      float k[NB], v[NB];
    };
    const auto scales_of = [&](const Pages& pg) {
      Scales sc;
#pragma unroll
      for (int bl = 0; bl < NB; ++bl) {
        const int64_t id = max(pg.id[bl], 0);
        sc.k[bl] = sc.v[bl] = 1.f;
        if (pg.id[bl] >= 0) {
          sc.k[bl] = exp_scale(clamp_exp(load_uniform(keb + id * p.ke.sb)));
          sc.v[bl] = exp_scale(clamp_exp(load_uniform(veb + id * p.ve.sb)));
        }
      }
      return sc;
    };
    const auto issue = [&](int it, char* stage, const Pages& pg) __attribute__((always_inline)) {
      typedef __attribute__((address_space(3))) void lds_void;
#pragma unroll
      for (int bl = 0; bl < NB; ++bl) {
        const int key = c0 + (4 * it + wave) * TW + 16 * bl, rows = c1 - key;
        __amdgpu_buffer_rsrc_t tk = make_rsrc(kbase, 0u), tv = make_rsrc(vbase, 0u);
        if (rows > 0) {
          const int64_t slot = key & ((1 << p.block_shift) - 1);
          const uint32_t last = (uint32_t)(min(rows, 16) - 1);
          tk = make_rsrc(kbase + (int64_t)pg.id[bl] * p.k.sb + slot * p.k.ss, last * kss + D);
          tv = make_rsrc(vbase + (int64_t)pg.id[bl] * p.v.sb + slot * p.v.ss, last * vss + D);
        }
#pragma unroll
        for (int i = 0; i < IPB; ++i) {
          const int row = 16 * bl + RPI * i + lrow;
          const uint32_t ko = (uint32_t)lrow * kss + 16u * (uint32_t)(lch ^ fk(row));
          const uint32_t vo = (uint32_t)lrow * vss + 16u * (uint32_t)(lch ^ fv(row));
          const int at = (bl * IPB + i) * 1024;
          __builtin_amdgcn_raw_ptr_buffer_load_lds(tk, (lds_void*)(stage + at), 16, ko, (uint32_t)(i * RPI) * kss, 0,
                                                   kDmaStream);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(tv, (lds_void*)(stage + 4096 + at), 16, vo,
                                                   (uint32_t)(i * RPI) * vss, 0, kDmaStream);
        }
      }
    };

    Pages next = pages_of(0);
    Scales sc_a, sc_b;
    if (n > 0) {
      issue(0, la, next);
      sc_a = scales_of(next);
    }
    next = pages_of(1);
    u32x4 qreg[NKS];
    {
      const char* qrow = static_cast<const char*>(p.q.ptr) +
                         2 * ((varlen ? (tok0 + pos) * p.q.ss : (int64_t)b * p.q.sb + (int64_t)pos * p.q.ss) +
                              (int64_t)head * p.q.sh + (D / 4) * lg);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        qreg[ks] = valid ? *reinterpret_cast<const u32x4*>(qrow + 16 * ks) : u32x4{0u, 0u, 0u, 0u};
    }
    if (n > 1) {
      issue(1, lb, next);
      sc_b = scales_of(next);
    }
    next = pages_of(2);

    f32x4 acc[NDB] = {};
    float m_run = -__builtin_inff(), l_run = 0.f;

    // Tile `it` out of its stage, then its stage's next one.
    const auto step = [&](int it, char* stage, Scales& sc) __attribute__((always_inline)) {
      if (it + 1 < n) wave_wait<vmcnt_imm(NLD)>();
      else wave_wait<vmcnt_imm(0)>();
      const char* ck = stage;
      const char* cv = stage + 4096;
      f32x4 sx[NB];
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        sx[kb] = f32x4{};
#pragma unroll
        for (int x = 0; x < NKS / 2; ++x) {
          const u32x4 raw = *reinterpret_cast<const u32x4*>(ck + kb * 16 * D + ka[x]);
          sx[kb] = E::mfma16(widen8<DT>(raw[0], sc.k[kb], raw[1], sc.k[kb]), qreg[2 * x], sx[kb]);
          sx[kb] = E::mfma16(widen8<DT>(raw[2], sc.k[kb], raw[3], sc.k[kb]), qreg[2 * x + 1], sx[kb]);
        }
      }
      const int key0 = c0 + (4 * it + wave) * TW;
      float row_t = 0.f;  // added to every score of the lane
      cap_scores<4>(sx, p.mod);
      if (p.mod.slopes != nullptr)
        row_t = bias_scores<4>(sx, slope, key0 + 4 * lg - qpos, key0 + TW - 1 <= qpos_lo,
                               [](int e) { return 16 * (e >> 2) + (e & 3); });
      if (key0 + TW > c1 || (dm.causal && key0 + TW - 1 > seen_lo)) {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const int key = key0 + 16 * kb + 4 * lg + v;
            const bool off = key >= c1 || (dm.causal && key > seen);
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
        const u32x4 pk = u32x4{E::pack2(pv[2 * jj][0], pv[2 * jj][1]), E::pack2(pv[2 * jj][2], pv[2 * jj][3]),
                               E::pack2(pv[2 * jj + 1][0], pv[2 * jj + 1][1]),
                               E::pack2(pv[2 * jj + 1][2], pv[2 * jj + 1][3])};
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const u32x2 raw = ld_tr8(cv + 32 * jj * D + (va ^ (uint32_t)(16 * db)));
          acc[db] = E::mfma16(widen8<DT>(raw[0], sc.v[2 * jj], raw[1], sc.v[2 * jj + 1]), pk, acc[db]);
        }
      }
      if (it + 2 < n) {
        wave_wait<kLgkm0>();  // (the stage has been read)
        issue(it + 2, stage, next);
        sc = scales_of(next);
        next = pages_of(it + 3);
      }
    };
    for (int it = 0; it < n; it += 2) {
      step(it, la, sc_a);
      if (it + 1 < n) step(it + 1, lb, sc_b);
    }

    // The four waves' states meet in the first stage, each in its wave's part.
    const float l_tot = xhalf_sum(xquad_sum(l_run));
    wave_wait<kLgkm0>();
    f32x4* xa = reinterpret_cast<f32x4*>(la);
#pragma unroll
    for (int db = 0; db < NDB; ++db) xa[db * 64 + lane] = acc[db];
    if (lg == 0) {
      st_m[wave][i16] = m_run;
      st_l[wave][i16] = l_tot;
    }
    __syncthreads();
    float ms = st_m[0][i16];
#pragma unroll
    for (int x = 1; x < 4; ++x) ms = fmaxf(ms, st_m[x][i16]);
    const float mu = ms == -__builtin_inff() ? 0.f : ms;
    float a[4], l = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      a[x] = fast_exp2((st_m[x][i16] - mu) * c);
      l += a[x] * st_l[x][i16];
    }
    const int64_t row = partial_row(p, true, b, head, pos, s);
    float* wa = p.ws_acc + row * D + 4 * lg;
    if (valid) {
#pragma unroll
      for (int k = 0; k < NDB / 4; ++k) {
        const int db = (NDB / 4) * wave + k;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 4; ++x) o += a[x] * reinterpret_cast<const f32x4*>(lds_a + x * 8192)[db * 64 + lane];
        *reinterpret_cast<f32x4*>(wa + 16 * db) = o;
      }
      if (wave == 0 && lg == 0) {
        p.ws_m[row] = ms == -__builtin_inff() ? kEmptyRef : __builtin_fmaf(ms, c, p.mod.shift2);
        p.ws_l[row] = l;
      }
    }
    __syncthreads();  // before the next piece's loads into the first stage
  }
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
  hipLaunchKernelGGL((gqa_decode8_kernel<DT, D>), dim3((unsigned)(total + 1)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_decode8(const Split8Params& p, int dtype, hipStream_t stream) {
  if (p.dm.G * p.dm.Sq > kDecode8Rows || p.block_shift < 4) return hipErrorInvalidValue;
  if (dtype == 0) return p.dm.D == 128 ? launch_decode8_t<0, 128>(p, stream) : launch_decode8_t<0, 64>(p, stream);
  return p.dm.D == 128 ? launch_decode8_t<1, 128>(p, stream) : launch_decode8_t<1, 64>(p, stream);
}

}  // namespace gqa
