// gqa_abi_ops.hip — extern "C" entry points around the attention: norms and
// rotation of queries and keys, document spans, block tables (include/gqa_attn.h).
// Every check comes before the first HIP call; nothing here allocates.
#include <hip/hip_runtime.h>

#include "../../include/gqa_attn.h"
#include "gqa_params.hpp"

namespace {

using gqa::TensorRef;

int to_code(hipError_t e) { return e == hipSuccess ? GQA_OK : static_cast<int>(e); }

bool unaligned(const void* p, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; }

// n - 1 outer strides of n: unit last stride, 16-byte aligned rows.
int check_rows(const void* ptr, const int64_t* st, int n) {
  if (ptr == nullptr || st == nullptr) return GQA_E_NULL;
  if (st[n - 1] != 1 || unaligned(ptr, 15u)) return GQA_E_STRIDE;
  for (int i = 0; i + 1 < n; ++i)
    if (st[i] % 8 != 0) return GQA_E_STRIDE;
  return GQA_OK;
}

int block_shift_of(int block_size) {
  int s = 0;
  while ((1 << s) < block_size) ++s;
  return s;
}
bool bad_block(int block_size) {
  return block_size < 1 || block_size > GQA_MAX_BLOCK_SIZE || (block_size & (block_size - 1)) != 0;
}

// tokens: their number (none: no positions needed).
int rope_params(const gqa_rope* r, int head_dim, int dtype, int64_t tokens, gqa::RopeParams& p) {
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

TensorRef ref4(const void* ptr, const int64_t* st) { return TensorRef{ptr, st[0], st[1], st[2]}; }
TensorRef token_ref(const void* ptr, const int64_t* st) { return TensorRef{ptr, 0, st[1], st[0]}; }

}  // namespace

extern "C" {

int gqa_qk_norm_rope_launch(const void* q, const int64_t q_stride[4], const void* k, const int64_t k_stride[4],
                            void* q_out, const int64_t q_out_stride[4], void* k_out, const int64_t k_out_stride[4],
                            const gqa_rope* rope, int batch, int num_heads, int num_kv_heads, int seq, int head_dim,
                            int dtype, void* stream) {
  if (batch < 0 || seq < 0 || num_heads <= 0 || num_kv_heads <= 0 || (int64_t)batch * seq >= GQA_MAX_ROPE_TOKENS)
    return GQA_E_SHAPE;
  gqa::RopeParams p{};
  int rc = rope_params(rope, head_dim, dtype, (int64_t)batch * seq, p);
  if (rc) return rc;
  if (batch == 0 || seq == 0) return GQA_OK;
  if ((k == nullptr) != (k_out == nullptr)) return GQA_E_NULL;
  if ((rc = check_rows(q, q_stride, 4)) || (rc = check_rows(q_out, q_out_stride, 4))) return rc;
  if (k != nullptr && ((rc = check_rows(k, k_stride, 4)) || (rc = check_rows(k_out, k_out_stride, 4)))) return rc;
  p.q = ref4(q, q_stride);
  p.qo = ref4(q_out, q_out_stride);
  if (k != nullptr) {
    p.k = ref4(k, k_stride);
    p.ko = ref4(k_out, k_out_stride);
  }
  p.n_tokens = batch * seq;
  p.S = seq;
  p.Hq = num_heads;
  p.Hkv = num_kv_heads;
  return to_code(gqa::launch_rope(p, dtype, static_cast<hipStream_t>(stream)));
}

int gqa_qk_norm_rope_write_launch(const void* q, const int64_t q_stride[3], const void* k, const int64_t k_stride[3],
                                  const void* v, const int64_t v_stride[3], void* q_out,
                                  const int64_t q_out_stride[3], void* k_cache, const int64_t k_cache_stride[4],
                                  void* v_cache, const int64_t v_cache_stride[4], const int64_t* slot_mapping,
                                  const gqa_rope* rope, int num_tokens, int num_heads, int num_kv_heads, int head_dim,
                                  int block_size, int dtype, void* stream) {
  if (num_tokens < 0 || num_tokens >= GQA_MAX_ROPE_TOKENS || num_heads <= 0 || num_kv_heads <= 0) return GQA_E_SHAPE;
  if (bad_block(block_size)) return GQA_E_BLOCK;
  gqa::RopeParams p{};
  int rc = rope_params(rope, head_dim, dtype, num_tokens, p);
  if (rc) return rc;
  if (num_tokens == 0) return GQA_OK;
  if (slot_mapping == nullptr) return GQA_E_NULL;
  if (unaligned(slot_mapping, 7u)) return GQA_E_STRIDE;
  if ((rc = check_rows(q, q_stride, 3)) || (rc = check_rows(k, k_stride, 3)) || (rc = check_rows(v, v_stride, 3)) ||
      (rc = check_rows(q_out, q_out_stride, 3)) || (rc = check_rows(k_cache, k_cache_stride, 4)) ||
      (rc = check_rows(v_cache, v_cache_stride, 4)))
    return rc;
  p.q = token_ref(q, q_stride);
  p.k = token_ref(k, k_stride);
  p.v = token_ref(v, v_stride);
  p.qo = token_ref(q_out, q_out_stride);
  p.kc = TensorRef{k_cache, k_cache_stride[0], k_cache_stride[2], k_cache_stride[1]};
  p.vc = TensorRef{v_cache, v_cache_stride[0], v_cache_stride[2], v_cache_stride[1]};
  p.slots = slot_mapping;
  p.block_shift = block_shift_of(block_size);
  p.n_tokens = num_tokens;
  p.S = num_tokens;
  p.Hq = num_heads;
  p.Hkv = num_kv_heads;
  return to_code(gqa::launch_rope(p, dtype, static_cast<hipStream_t>(stream)));
}

int gqa_document_spans_launch(const int* ids, int64_t row_stride, int* lo, int* hi, int batch, int seq, void* stream) {
  if (batch < 0 || seq < 0 || seq > (1 << 30) || row_stride < 0) return GQA_E_SHAPE;
  if (batch == 0 || seq == 0) return GQA_OK;
  if (ids == nullptr || lo == nullptr || hi == nullptr) return GQA_E_NULL;
  if (unaligned(ids, 3u) || unaligned(lo, 3u) || unaligned(hi, 3u)) return GQA_E_STRIDE;
  return to_code(gqa::launch_spans(gqa::SpanParams{ids, row_stride, lo, hi, batch, seq},
                                   static_cast<hipStream_t>(stream)));
}

size_t gqa_extend_tables_scratch_bytes(int pool_rows, int batch) {
  if (pool_rows < 0 || batch < 0) return 0;
  return ((size_t)pool_rows + 2 * (size_t)batch + 1) * sizeof(int);
}

int gqa_extend_tables_launch(int* block_tables, int64_t table_stride, int table_width, int* pool_lens, int pool_rows,
                             const int* rows, const int* query_lens, const int* free_blocks, int* free_count,
                             int num_blocks, int block_size, int update, int batch, int num_tokens, int* seq_lens,
                             int* query_start, int* query_lens_out, int64_t* slot_mapping, int* positions,
                             int* batch_tables, int* new_free_count, int* refused, int* scratch, void* stream) {
  if (pool_rows < 0 || batch < 0 || num_tokens < 0 || num_blocks < 0 || table_width < 1 || table_stride < table_width)
    return GQA_E_SHAPE;
  if (rows == nullptr && batch > pool_rows) return GQA_E_SHAPE;
  if (bad_block(block_size) || (int64_t)table_width * block_size >= ((int64_t)1 << 31) ||
      (int64_t)num_blocks * block_size >= ((int64_t)1 << 40))
    return GQA_E_BLOCK;
  if ((int64_t)batch * table_width + num_tokens >= ((int64_t)1 << 31)) return GQA_E_SHAPE;  // (an item a thread)
  if (free_count == nullptr || new_free_count == nullptr || refused == nullptr || scratch == nullptr) return GQA_E_NULL;
  if (num_blocks > 0 && free_blocks == nullptr) return GQA_E_NULL;
  if (batch > 0 && (block_tables == nullptr || pool_lens == nullptr || query_lens == nullptr || seq_lens == nullptr ||
                    query_start == nullptr || query_lens_out == nullptr || batch_tables == nullptr))
    return GQA_E_NULL;
  if (num_tokens > 0 && (slot_mapping == nullptr || positions == nullptr)) return GQA_E_NULL;
  if (unaligned(slot_mapping, 7u)) return GQA_E_STRIDE;
  for (const int* x : {static_cast<const int*>(block_tables), static_cast<const int*>(pool_lens), rows, query_lens,
                       free_blocks, static_cast<const int*>(free_count), static_cast<const int*>(seq_lens),
                       static_cast<const int*>(query_start), static_cast<const int*>(query_lens_out),
                       static_cast<const int*>(positions), static_cast<const int*>(batch_tables),
                       static_cast<const int*>(new_free_count), static_cast<const int*>(refused),
                       static_cast<const int*>(scratch)})
    if (unaligned(x, 3u)) return GQA_E_STRIDE;
  gqa::TablesParams p{};
  p.tables = block_tables;
  p.stride = table_stride;
  p.width = table_width;
  p.lens = pool_lens;
  p.n_rows = pool_rows;
  p.rows = rows;
  p.new_lens = query_lens;
  p.free_blocks = free_blocks;
  p.free_count = free_count;
  p.n_free = num_blocks;
  p.block_shift = block_shift_of(block_size);
  p.update = update != 0;
  p.B = batch;
  p.n_tokens = num_tokens;
  p.seq_lens = seq_lens;
  p.query_start = query_start;
  p.query_lens = query_lens_out;
  p.slots = slot_mapping;
  p.positions = positions;
  p.batch_tables = batch_tables;
  p.new_free = new_free_count;
  p.refused = refused;
  p.scratch = scratch;
  return to_code(gqa::launch_tables(p, static_cast<hipStream_t>(stream)));
}

int gqa_release_blocks_launch(const int* block_tables, int64_t table_stride, int table_width, int* pool_lens,
                              int pool_rows, const int* rows, int batch, int* free_blocks, int* free_count,
                              int num_blocks, int block_size, int* scratch, void* stream) {
  if (pool_rows < 0 || batch < 0 || num_blocks < 0 || table_width < 1 || table_stride < table_width)
    return GQA_E_SHAPE;
  if (bad_block(block_size) || (int64_t)table_width * block_size >= ((int64_t)1 << 31)) return GQA_E_BLOCK;
  if (batch == 0) return GQA_OK;
  if (block_tables == nullptr || pool_lens == nullptr || rows == nullptr || free_blocks == nullptr ||
      free_count == nullptr || scratch == nullptr)
    return GQA_E_NULL;
  for (const int* x : {block_tables, static_cast<const int*>(pool_lens), rows, static_cast<const int*>(free_blocks),
                       static_cast<const int*>(free_count), static_cast<const int*>(scratch)})
    if (unaligned(x, 3u)) return GQA_E_STRIDE;
  gqa::ReleaseParams p{};
  p.tables = block_tables;
  p.stride = table_stride;
  p.width = table_width;
  p.lens = pool_lens;
  p.n_rows = pool_rows;
  p.rows = rows;
  p.B = batch;
  p.free_blocks = free_blocks;
  p.free_count = free_count;
  p.n_free = num_blocks;
  p.block_shift = block_shift_of(block_size);
  p.scratch = scratch;
  return to_code(gqa::launch_release(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
