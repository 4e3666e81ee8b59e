// gqa_decode.hip — the decode-shaped first passes (gqa_decode_kernel.hpp)
// without changed scores, and which calls they take.
#include "gqa_decode_kernel.hpp"

namespace gqa {

bool decode_kernel_fits(const SplitParams& p) {
  const int D = p.dm.D;
  // Flat splits: one 32-row block per kv head (two or four with the walk's
  // state spill registers); 32-bit products of units and slots.
  const bool flat = p.slots > 0;
  if (flat && (p.n_rblk != 1 || p.counters != nullptr)) return false;
  const int unit = decode_unit(D);
  if (flat && ((int64_t)((p.dm.Skv + unit - 1) / unit) * p.dm.B + 1) * (p.slots + 1) >= ((int64_t)1 << 31))
    return false;
  // Head_dim 64: the 16-row first pass only (at most 16 packed rows per kv
  // head), in the two-launch form (no fused combine at that width).
  if (D == 64) {
    if (p.dm.G * p.dm.Sq > 16 || p.counters != nullptr) return false;
  } else if (D != kDecD) {
    return false;
  }
  const bool paged = p.block_table != nullptr;
  // Paged: whole LDS-DMA instructions (512 / D rows) in a page, and
  // 64-key-aligned chunks (so a tile lies in a page of >= 64 keys).
  if (paged && ((1 << p.block_shift) < 512 / D || (p.chunk & 63) != 0)) return false;
  // 32-bit descriptor offsets: (contiguous) a chunk plus the padding step
  // past it (two steps of 64 keys at head_dim 128, of 128 at 64), (paged) a
  // 64-row sub-tile; the whole accumulator workspace.
  const int64_t span = paged ? 64 : (int64_t)p.chunk + (D == 64 ? 256 : 128);
  if (span * p.k.ss * 2 >= ((int64_t)1 << 31) || span * p.v.ss * 2 >= ((int64_t)1 << 31)) return false;
  const int64_t acc_bytes =
      (flat ? (int64_t)p.slots + p.dm.B : (int64_t)p.dm.B * p.splits) * p.dm.Hq * p.dm.Sq * D * 4;
  // ... and a kv head's query group (its G heads x Sq rows).
  const int64_t q_bytes = 2 * ((int64_t)(p.dm.G - 1) * p.q.sh + (int64_t)(p.dm.Sq - 1) * p.q.ss + D);
  return acc_bytes <= 0xFFFFFFF0ll && q_bytes < ((int64_t)1 << 31);
}

hipError_t launch_decode_first(const SplitParams& p, int dtype, hipStream_t stream, const ScoreMod* mod) {
  if (mod != nullptr) return launch_decode_first_mod(p, dtype, stream, *mod);
  return launch_decode_p(p, dtype, stream);
}

}  // namespace gqa
