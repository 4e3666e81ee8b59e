// gqa_abi_rope.hpp — argument checks that the entry points of gqa_abi_ops.hip and
// gqa_abi_cache8.hip share: rows, and a call's gqa_rope.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/gqa_attn.h"
#include "gqa_params.hpp"

namespace gqa {

inline int to_code(hipError_t e) { return e == hipSuccess ? GQA_OK : static_cast<int>(e); }

inline bool unaligned(const void* p, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; }

// n - 1 outer strides of n: unit last stride, 16-byte aligned rows.
inline int check_rows(const void* ptr, const int64_t* st, int n) {
  if (ptr == nullptr || st == nullptr) return GQA_E_NULL;
  if (st[n - 1] != 1 || unaligned(ptr, 15u)) return GQA_E_STRIDE;
  for (int i = 0; i + 1 < n; ++i)
    if (st[i] % 8 != 0) return GQA_E_STRIDE;
  return GQA_OK;
}

// tokens: their number (none: no positions needed).
inline int rope_params(const gqa_rope* r, int head_dim, int dtype, int64_t tokens, RopeParams& p) {
  if (r == nullptr) return GQA_E_NULL;
  if (head_dim != 64 && head_dim != 128) return GQA_E_HEAD_DIM;
  if (dtype != GQA_DTYPE_BF16 && dtype != GQA_DTYPE_FP16) return GQA_E_DTYPE;
  if (r->table != nullptr) {
    if (r->max_positions < 1 || r->rotary_dim < 16 || r->rotary_dim > head_dim || r->rotary_dim % 16 != 0 ||
        r->axes < 1 || r->axes > 4)
      return GQA_E_ROPE;
    if (r->positions == nullptr && tokens > 0) return GQA_E_NULL;
    if (unaligned(r->table, 15u) || unaligned(r->positions, r->positions64 ? 7u : 3u)) return GQA_E_STRIDE;
    for (int i = 0; i < r->rotary_dim / 2; ++i)
      if (r->axes > 1 && (int)((r->pair_axis[i >> 4] >> (2 * (i & 15))) & 3u) >= r->axes) return GQA_E_ROPE;
  }
  if (unaligned(r->q_weight, 15u) || unaligned(r->k_weight, 15u)) return GQA_E_STRIDE;
  if ((r->q_weight != nullptr || r->k_weight != nullptr) && !(r->eps >= 0.f)) return GQA_E_ROPE;
  p.table = r->table;
  p.max_pos = r->max_positions;
  p.R = r->rotary_dim;
  p.interleaved = r->interleaved != 0;
  p.pos = r->positions;
  p.pos64 = r->positions64 != 0;
  p.axes = r->axes;
  for (int i = 0; i < 4; ++i) p.pair_axis[i] = r->pair_axis[i];
  p.wq = r->q_weight;
  p.wk = r->k_weight;
  p.w32 = r->weights32 != 0;
  p.eps = r->eps;
  p.D = head_dim;
  return GQA_OK;
}

}  // namespace gqa
