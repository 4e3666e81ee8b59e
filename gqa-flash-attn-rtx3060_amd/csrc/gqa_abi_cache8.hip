// gqa_abi_cache8.hip — extern "C" entry points of the paged cache in 8 bits
// (include/gqa_attn.h).  Every check comes before the first HIP call; nothing here
// allocates.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/gqa_attn.h"
#include "gqa_abi_rope.hpp"
#include "gqa_params.hpp"

namespace {

using gqa::TensorRef;

constexpr int kTile = gqa::kFwdTileKeys;

int check_sizes(int num_kv_heads, int head_dim, int dtype, int block_size) {
  if (num_kv_heads <= 0) return GQA_E_SHAPE;
  if (head_dim != 64 && head_dim != 128) return GQA_E_HEAD_DIM;
  if (dtype != GQA_DTYPE_BF16 && dtype != GQA_DTYPE_FP16) return GQA_E_DTYPE;
  if (block_size < 16 || block_size > GQA_MAX_BLOCK_SIZE || (block_size & (block_size - 1)) != 0) return GQA_E_CACHE8;
  return GQA_OK;
}

int check_cache(const gqa_cache8* c, int head_dim) {
  if (c == nullptr || c->codes == nullptr || c->exponents == nullptr) return GQA_E_NULL;
  if (c->stride[3] != 1 || gqa::unaligned(c->codes, 15u) || gqa::unaligned(c->exponents, 3u)) return GQA_E_STRIDE;
  for (int i = 0; i < 3; ++i)
    if (c->stride[i] % 16 != 0) return GQA_E_STRIDE;
  if (c->stride[1] < 0 || 15 * c->stride[1] + head_dim >= ((int64_t)1 << 31)) return GQA_E_CACHE8;
  return GQA_OK;
}

// A store's slots and heads have memory of their own.
bool shares(const gqa_cache8* c, int num_kv_heads) {
  return c->stride[1] == 0 || (num_kv_heads > 1 && (c->stride[2] == 0 || c->exp_stride[1] == 0));
}

TensorRef cache_ref(const gqa_cache8* c) { return TensorRef{c->codes, c->stride[0], c->stride[2], c->stride[1]}; }
gqa::Exponents exp_ref(const gqa_cache8* c) { return gqa::Exponents{c->exponents, c->exp_stride[0], c->exp_stride[1]}; }
TensorRef ref4(const void* ptr, const int64_t* st) { return TensorRef{ptr, st[0], st[1], st[2]}; }
TensorRef token_ref(const void* ptr, const int64_t* st) { return TensorRef{ptr, 0, st[1], st[0]}; }

// Units of the flat split and slots that its walk can multiply in 32 bits.
bool flat_fits(int batch, int max_seq_len, int slots) {
  const int64_t units = ((int64_t)max_seq_len + gqa::kDecode8Unit - 1) / gqa::kDecode8Unit;
  return (units * batch + 1) * (slots + 1) < ((int64_t)1 << 31);
}

// Tiles of all sequences that the cut into key pieces can add up in 32 bits.
bool pieces_fit(int batch, int max_seq_len) {
  return ((int64_t)max_seq_len + kTile - 1) / kTile * batch < ((int64_t)1 << 31) - GQA_MAX_SPLITS;
}

}  // namespace

extern "C" {

int gqa_paged8_plan(int batch, int num_heads, int num_kv_heads, int seq_q, int max_seq_len, int head_dim, int cu_count,
                    int* form, int* parts) {
  if (form == nullptr || parts == nullptr) return GQA_E_NULL;
  if (batch < 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || seq_q < 0 ||
      max_seq_len < 0 || cu_count < 1)
    return GQA_E_SHAPE;
  if (head_dim != 64 && head_dim != 128) return GQA_E_HEAD_DIM;
  const int G = num_heads / num_kv_heads;
  if (G > gqa::kShortRows) return GQA_E_GROUP;
  if (max_seq_len > GQA_MAX_CACHE8_KEYS) return GQA_E_CACHE8;
  *form = GQA_FORM_SINGLE;
  *parts = 0;
  if (batch == 0 || seq_q == 0 || max_seq_len == 0) return GQA_OK;
  if ((int64_t)G * seq_q <= gqa::kDecode8Rows) {
    const int64_t unit = gqa::kDecode8Unit, units = (max_seq_len + unit - 1) / unit * batch;
    int64_t slots = std::min<int64_t>({std::max(2 * cu_count / num_kv_heads, 1), units, GQA_MAX_SPLITS});
    while (slots > 1 && !flat_fits(batch, max_seq_len, (int)slots)) slots /= 2;
    if (flat_fits(batch, max_seq_len, (int)slots)) {
      *form = GQA_FORM_FLAT;
      *parts = (int)slots;
      return GQA_OK;
    }
  }
  const int rows = gqa::chunk8_rows(G, seq_q, max_seq_len, head_dim), block_m = rows / G;
  const int64_t blocks = ((int64_t)seq_q + block_m - 1) / block_m * num_kv_heads;
  const int64_t tiles = (max_seq_len + kTile - 1) / kTile;
  const int64_t slots = (rows > gqa::kShortRows ? 1 : head_dim == 64 ? 3 : 2) * cu_count;
  const int64_t pieces = std::min<int64_t>({slots / blocks, batch * (tiles / 4), GQA_MAX_SPLITS});
  // Pieces that fill the device once, where there are five for four sequences or more.  The
  // single pass / these, us, 32/8 heads of 128, lengths 2000-9000 and all 5000: 8 x 160
  // queries (9 pieces) 217 / 201 and 136 / 149, 4 x 384 (5) 221 / 165 and 136 / 151, 4 x 320
  // (6) 220 / 140 and 135 / 150, 4 x 256 (8) 218 / 107 and 134 / 100.  Twice as many, for two
  // rounds, take 232 / 209 and 164 / 196 (8 x 256 queries, 16).  Not where the queries are
  // more than half of the keys: causal blocks then see few keys of most pieces (1024 tokens
  // over themselves 32.9 / 36.7, 512 18.5 / 21.6; 512 over 1024 30.8 / 27.4, 1024 over 2048
  // 56.7 / 56.9).
  if (4 * pieces >= 5 * (int64_t)batch && max_seq_len / 2 >= seq_q && pieces_fit(batch, max_seq_len)) {
    *form = GQA_FORM_CHUNKS;
    *parts = (int)pieces;
  }
  return GQA_OK;
}

size_t gqa_paged8_workspace_bytes(int form, int parts, int batch, int num_heads, int seq_q, int head_dim) {
  if (form != GQA_FORM_FLAT && form != GQA_FORM_CHUNKS) return 0;
  return gqa_split_flat_workspace_bytes(batch, num_heads, seq_q, head_dim, parts);
}

int gqa_paged8_launch(int form, const void* q, const int64_t q_stride[4], const gqa_cache8* k_cache,
                      const gqa_cache8* v_cache, const int* block_table, int table_stride, const int* seq_lens,
                      const int* q_start, const int* q_len, int block_size, int max_seq_len, void* o,
                      const int64_t o_stride[4], float* lse, float* workspace, int parts, int batch, int num_heads,
                      int num_kv_heads, int seq_q, int head_dim, float scale_log2, int causal, int dtype,
                      const gqa_score* score, void* stream) {
  int rc = check_sizes(num_kv_heads, head_dim, dtype, block_size);
  if (rc) return rc;
  if (batch < 0 || num_heads <= 0 || seq_q < 0 || max_seq_len < 0 || num_heads % num_kv_heads != 0) return GQA_E_SHAPE;
  const int G = num_heads / num_kv_heads;
  if (G > gqa::kShortRows) return GQA_E_GROUP;
  if (table_stride < 0 || (int64_t)table_stride * block_size < (int64_t)max_seq_len) return GQA_E_BLOCK;
  if (max_seq_len > GQA_MAX_CACHE8_KEYS) return GQA_E_CACHE8;
  if (form != GQA_FORM_FLAT && form != GQA_FORM_CHUNKS && form != GQA_FORM_SINGLE) return GQA_E_CACHE8;
  if (form == GQA_FORM_FLAT && ((int64_t)G * seq_q > gqa::kDecode8Rows || max_seq_len < 1)) return GQA_E_CACHE8;
  if (form != GQA_FORM_SINGLE && (parts < 1 || parts > GQA_MAX_SPLITS)) return GQA_E_SPLITS;
  if (form == GQA_FORM_FLAT && !flat_fits(batch, max_seq_len, parts)) return GQA_E_CACHE8;
  if (form == GQA_FORM_CHUNKS && (parts < batch || !pieces_fit(batch, max_seq_len))) return GQA_E_SPLITS;
  gqa::ScoreMod mod{};
  if (score != nullptr) {
    if ((rc = gqa::score_mod(score, scale_log2, causal, true, seq_q, max_seq_len, mod))) return rc;
  } else if (!(scale_log2 > 0.f) || !std::isfinite(scale_log2)) {
    return GQA_E_CACHE8;
  }
  if (batch == 0 || seq_q == 0) return GQA_OK;
  if (seq_lens == nullptr || (max_seq_len > 0 && block_table == nullptr)) return GQA_E_NULL;
  if (gqa::unaligned(seq_lens, 3u) || gqa::unaligned(block_table, 3u) || gqa::unaligned(lse, 3u)) return GQA_E_STRIDE;
  if ((q_start == nullptr) != (q_len == nullptr)) return GQA_E_NULL;
  if (gqa::unaligned(q_start, 3u) || gqa::unaligned(q_len, 3u)) return GQA_E_STRIDE;
  if ((rc = gqa::check_rows(q, q_stride, 4)) || (rc = gqa::check_rows(o, o_stride, 4))) return rc;
  if (max_seq_len > 0 && ((rc = check_cache(k_cache, head_dim)) || (rc = check_cache(v_cache, head_dim)))) return rc;
  if (form != GQA_FORM_SINGLE) {
    if (workspace == nullptr) return GQA_E_NULL;
    if (gqa::unaligned(workspace, 15u)) return GQA_E_STRIDE;
  }
  const gqa::Dims dm{batch, num_heads, num_kv_heads, seq_q, max_seq_len, head_dim, G, scale_log2, causal ? 1 : 0};
  int shift = 0;
  while ((1 << shift) < block_size) ++shift;
  const gqa_cache8 none{};
  const gqa_cache8 *kc = k_cache != nullptr ? k_cache : &none, *vc = v_cache != nullptr ? v_cache : &none;
  hipStream_t st = static_cast<hipStream_t>(stream);
  gqa::ReduceParams r{};
  r.o = ref4(o, o_stride);
  r.B = batch;
  r.Hq = num_heads;
  r.Sq = seq_q;
  r.D = head_dim;
  r.splits = parts;
  r.lse = lse;
  r.q_start = q_start;
  r.q_len = q_len;
  if (form == GQA_FORM_FLAT) {
    gqa::Split8Params p{};
    p.q = ref4(q, q_stride);
    p.k = cache_ref(kc);
    p.v = cache_ref(vc);
    p.dm = dm;
    const size_t rows = ((size_t)parts + batch) * num_heads * seq_q;
    p.ws_acc = workspace;
    p.ws_m = workspace + rows * head_dim;
    p.ws_l = p.ws_m + rows;
    p.plan = reinterpret_cast<int*>(p.ws_l + rows);
    p.splits = 1;
    p.slots = parts;
    p.block_table = block_table;
    p.seq_lens = seq_lens;
    p.table_stride = table_stride;
    p.block_shift = shift;
    p.q_start = q_start;
    p.q_len = q_len;
    p.mod = mod;
    p.ke = exp_ref(kc);
    p.ve = exp_ref(vc);
    if ((rc = gqa::to_code(gqa::launch_decode8(p, dtype, st)))) return rc;
    r.ws_acc = p.ws_acc;
    r.ws_m = p.ws_m;
    r.ws_l = p.ws_l;
    r.plan = p.plan;
    r.slots = parts;
    return gqa::to_code(gqa::launch_decode8_join(r, G, dtype, st));
  }
  gqa::Fwd8Params p{};
  p.q = ref4(q, q_stride);
  p.k = cache_ref(kc);
  p.v = cache_ref(vc);
  p.o = r.o;
  p.dm = dm;
  p.block_m = gqa::chunk8_rows(G, seq_q, max_seq_len, head_dim) / G;
  p.n_mblk = (seq_q + p.block_m - 1) / p.block_m;
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.table_stride = table_stride;
  p.block_shift = shift;
  p.q_start = q_start;
  p.q_len = q_len;
  p.mod = mod;
  p.ke = exp_ref(kc);
  p.ve = exp_ref(vc);
  if (form == GQA_FORM_SINGLE) {
    p.lse = lse;
    return gqa::to_code(gqa::launch_chunk8(p, dtype, st));
  }
  p.kv_splits = parts;
  const size_t rows = ((size_t)parts + batch) * num_heads * seq_q;
  p.ws_acc = workspace;
  p.ws_m = workspace + rows * head_dim;
  p.ws_l = p.ws_m + rows;
  p.plan = reinterpret_cast<int*>(p.ws_l + rows);
  if ((rc = gqa::to_code(gqa::launch_chunk8(p, dtype, st)))) return rc;
  r.ws_acc = p.ws_acc;
  r.ws_m = p.ws_m;
  r.ws_l = p.ws_l;
  r.plan = p.plan;
  r.slots = parts;
  return gqa::to_code(gqa::launch_decode8_join(r, G, dtype, st));
}

int gqa_cache8_write_launch(const void* q, const int64_t q_stride[3], const void* k, const int64_t k_stride[3],
                            const void* v, const int64_t v_stride[3], void* q_out, const int64_t q_out_stride[3],
                            const gqa_cache8* k_cache, const gqa_cache8* v_cache, const int64_t* slot_mapping,
                            const gqa_rope* rope, int num_tokens, int num_heads, int num_kv_heads, int head_dim,
                            int block_size, int dtype, void* stream) {
  int rc = check_sizes(num_kv_heads, head_dim, dtype, block_size);
  if (rc) return rc;
  if (num_tokens < 0 || num_tokens >= GQA_MAX_ROPE_TOKENS || (q != nullptr && num_heads <= 0)) return GQA_E_SHAPE;
  gqa::Store8Params p{};
  if (rope != nullptr) {
    if ((rc = gqa::rope_params(rope, head_dim, dtype, num_tokens, p))) return rc;
  } else if (q != nullptr) {
    return GQA_E_NULL;
  }
  if (num_tokens == 0) return GQA_OK;
  if (slot_mapping == nullptr || (q == nullptr) != (q_out == nullptr)) return GQA_E_NULL;
  if (gqa::unaligned(slot_mapping, 7u)) return GQA_E_STRIDE;
  if (q != nullptr && ((rc = gqa::check_rows(q, q_stride, 3)) || (rc = gqa::check_rows(q_out, q_out_stride, 3))))
    return rc;
  if ((rc = gqa::check_rows(k, k_stride, 3)) || (rc = gqa::check_rows(v, v_stride, 3)) ||
      (rc = check_cache(k_cache, head_dim)) || (rc = check_cache(v_cache, head_dim)))
    return rc;
  if (shares(k_cache, num_kv_heads) || shares(v_cache, num_kv_heads) || k_cache->codes == v_cache->codes ||
      k_cache->exponents == v_cache->exponents)
    return GQA_E_CACHE8;
  if (q != nullptr) {
    p.q = token_ref(q, q_stride);
    p.qo = token_ref(q_out, q_out_stride);
  }
  p.k = token_ref(k, k_stride);
  p.v = token_ref(v, v_stride);
  p.kc = cache_ref(k_cache);
  p.vc = cache_ref(v_cache);
  p.ke = exp_ref(k_cache);
  p.ve = exp_ref(v_cache);
  p.slots = slot_mapping;
  while ((1 << p.block_shift) < block_size) ++p.block_shift;
  p.n_tokens = num_tokens;
  p.S = num_tokens;
  p.Hq = num_heads;
  p.Hkv = num_kv_heads;
  p.D = head_dim;
  p.limit = 1.875f * (dtype == GQA_DTYPE_FP16 ? 0x1p15f : 0x1p127f);
  return gqa::to_code(gqa::launch_store8(p, dtype, static_cast<hipStream_t>(stream)));
}

int gqa_cache8_read_launch(const gqa_cache8* k_cache, const gqa_cache8* v_cache, const int64_t* slot_mapping, void* k,
                           const int64_t k_stride[3], void* v, const int64_t v_stride[3], int num_tokens,
                           int num_kv_heads, int head_dim, int block_size, int dtype, void* stream) {
  int rc = check_sizes(num_kv_heads, head_dim, dtype, block_size);
  if (rc) return rc;
  if (num_tokens < 0) return GQA_E_SHAPE;
  if (num_tokens == 0) return GQA_OK;
  if (slot_mapping == nullptr) return GQA_E_NULL;
  if (gqa::unaligned(slot_mapping, 7u)) return GQA_E_STRIDE;
  if ((rc = gqa::check_rows(k, k_stride, 3)) || (rc = gqa::check_rows(v, v_stride, 3)) ||
      (rc = check_cache(k_cache, head_dim)) || (rc = check_cache(v_cache, head_dim)))
    return rc;
  gqa::Read8Params p{};
  p.kc = cache_ref(k_cache);
  p.vc = cache_ref(v_cache);
  p.ke = exp_ref(k_cache);
  p.ve = exp_ref(v_cache);
  p.k = token_ref(k, k_stride);
  p.v = token_ref(v, v_stride);
  p.slots = slot_mapping;
  p.n_tokens = num_tokens;
  p.Hkv = num_kv_heads;
  p.D = head_dim;
  while ((1 << p.block_shift) < block_size) ++p.block_shift;
  return gqa::to_code(gqa::launch_read8(p, dtype, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
