// gqa_tables.hip — what describes a batch to the attention kernels, built on
// the device: the spans of documents, and a step's block tables, slots and
// positions from the requests' lengths and a free list that lives there too.
#include <algorithm>

#include "gqa_common.hpp"
#include "gqa_params.hpp"

namespace gqa {

namespace {

constexpr int kPlanThreads = 1024;

// Inclusive sum over the workgroup's kPlanThreads threads; `total` gets the
// sum.  tmp: kPlanThreads / 64 values; every thread calls it.
__device__ inline int64_t block_scan(int64_t x, int64_t* tmp, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();  // tmp's readers of the call before
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += tmp[w];
    total += tmp[w];
  }
  return before + x;
}

}  // namespace

// A workgroup a row's kSpanChunk tokens, kSpanPer a thread.  The run that reaches
// into them starts at the last change before them, the one that leaves them ends at
// the first change behind.  In rows of up to kSpanWalk tokens both are looked for a
// thread's width at a time (the chunk beside it holds them unless a document is
// longer than that); in longer ones, where that would grow with the square of a
// document, those ends are left open (kOpen) for a second launch.  Measured, us, one
// launch / two, documents of 100 tokens and one of the whole row: 2 x 8192 ids 6.9,
// 7.9 / 9.1, 9.8; 16384 7.3, 10.8 / 10.5, 11.8; 32768 7.4, 16.8 / 11.0, 11.9; 131072 7.5,
// 52 / 11.8, 12.1; 2^20 9.3, 384 / 16.9, 14.4 (2^30 in one document 0.3 s).  Bound by
// barriers and dependent reads (bytes: 0.03 us for the first).
constexpr int kSpanPer = 4, kSpanChunk = kPlanThreads * kSpanPer, kSpanWalk = 32768, kOpen = -1;

// Inclusive running maximum over the workgroup; kPlanThreads / 64 ints.
__device__ inline int block_max_scan(int x, int* tmp) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xA, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xC, 0xF, false));
  __syncthreads();  // tmp's readers of the call before
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w)
    if (w < wave) x = max(x, tmp[w]);
  return x;
}

template <bool WALK> __global__ __launch_bounds__(kPlanThreads) void gqa_spans_kernel(SpanParams p) {
  __shared__ int s_id[kSpanChunk + 2], s_scan[kPlanThreads], tmp[kPlanThreads / 64], s_found;
  const int t = threadIdx.x;
  const int* ids = p.ids + blockIdx.y * p.stride;
  const int c0 = blockIdx.x * kSpanChunk, c1 = min(c0 + kSpanChunk, p.S);
  int* lo = p.lo + (int64_t)blockIdx.y * p.S;
  int* hi = p.hi + (int64_t)blockIdx.y * p.S;
  // s_id[i]: the id of token c0 - 1 + i.
  for (int i = t; i < c1 - c0 + 2; i += kPlanThreads) {
    const int at = c0 - 1 + i;
    s_id[i] = at >= 0 && at < p.S ? ids[at] : 0;
  }
  // The first change at or behind c1 (S: none), the last one at or before c0.
  constexpr int kFar = 0x7fffffff;
  int behind = p.S, before = kOpen;
  if constexpr (WALK) {
    for (int a = c1; a < p.S; a += kPlanThreads) {
      const int at = a + t;
      if (t == 0) s_found = p.S;
      __syncthreads();
      if (at < p.S && ids[at] != ids[at - 1]) atomicMin(&s_found, at);
      __syncthreads();
      behind = s_found;
      __syncthreads();
      if (behind < p.S) break;
    }
    before = 0;
    for (int a = c0; a > 0; a -= kPlanThreads) {
      const int at = a - t;
      if (t == 0) s_found = 0;
      __syncthreads();
      if (at > 0 && ids[at] != ids[at - 1]) atomicMax(&s_found, at);
      __syncthreads();
      before = s_found;
      __syncthreads();
      if (before > 0) break;
    }
  }
  __syncthreads();  // s_id
  if constexpr (!WALK) behind = c1 == p.S || s_id[c1 - c0 + 1] != s_id[c1 - c0] ? c1 : kFar;
  // This thread's tokens a .. a + 3, and the changes among them.
  const int a = t * kSpanPer;
  int id[kSpanPer];
  bool change[kSpanPer];
  int last = kOpen, first = kFar;
#pragma unroll
  for (int i = 0; i < kSpanPer; ++i) {
    id[i] = a + i < c1 - c0 ? s_id[a + i + 1] : 0;
    change[i] = a + i < c1 - c0 && (c0 + a + i == 0 || s_id[a + i] != id[i]);
    if (change[i]) {
      last = c0 + a + i;
      first = min(first, c0 + a + i);
    }
  }
  // Running maximum of the last changes from the left, and (thread order turned
  // round) of the negated first ones from the right.
  s_scan[t] = block_max_scan(last, tmp);
  __syncthreads();
  int start = max(t > 0 ? s_scan[t - 1] : kOpen, before);
  __syncthreads();
  s_scan[kPlanThreads - 1 - t] = -first;
  __syncthreads();
  const int turned = block_max_scan(s_scan[t], tmp);
  __syncthreads();
  s_scan[t] = turned;
  __syncthreads();
  int end = t + 1 < kPlanThreads ? min(-s_scan[kPlanThreads - 2 - t], behind) : behind;
  int st[kSpanPer], en[kSpanPer];
#pragma unroll
  for (int i = 0; i < kSpanPer; ++i) {
    if (change[i]) start = c0 + a + i;
    st[i] = id[i] < 0 ? 0 : start;
  }
#pragma unroll
  for (int i = kSpanPer - 1; i >= 0; --i) {
    en[i] = id[i] < 0 ? 0 : end == kFar ? kOpen : end;
    if (change[i]) end = c0 + a + i;
  }
#pragma unroll
  for (int i = 0; i < kSpanPer; ++i)
    if (a + i < c1 - c0) {
      lo[c0 + a + i] = st[i];
      hi[c0 + a + i] = en[i];
    }
}

// The open ends.  A run that enters a chunk starts where the run of the last token
// of the nearest chunk before it does whose start is known: the chunks between are
// that run from end to end (1024 of them looked at a round).  Other workgroups may
// be filling theirs: what is read is open or right.
__global__ __launch_bounds__(kPlanThreads) void gqa_spans_join_kernel(SpanParams p) {
  __shared__ int s_near;
  const int t = threadIdx.x, chunk = blockIdx.x, chunks = gridDim.x;
  const int c0 = chunk * kSpanChunk, c1 = min(c0 + kSpanChunk, p.S);
  int* lo = p.lo + (int64_t)blockIdx.y * p.S;
  int* hi = p.hi + (int64_t)blockIdx.y * p.S;
  const auto load = [](int* x) { return __hip_atomic_load(x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  const auto fill = [](int* x, int v) {
    if (*x == kOpen) __hip_atomic_store(x, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  const bool open_lo = load(lo + c0) == kOpen, open_hi = load(hi + c1 - 1) == kOpen;
  if (!open_lo && !open_hi) return;
  int start = 0, end = 0;
  for (int k0 = chunk - 1; open_lo && k0 >= 0; k0 -= kPlanThreads) {
    const int k = k0 - t;
    if (t == 0) s_near = -1;
    __syncthreads();
    if (k >= 0 && load(lo + (k + 1) * kSpanChunk - 1) != kOpen) atomicMax(&s_near, k);
    __syncthreads();
    const int near = s_near;
    __syncthreads();
    if (near < 0) continue;
    start = load(lo + (near + 1) * kSpanChunk - 1);
    break;
  }
  for (int k0 = chunk + 1; open_hi && k0 < chunks; k0 += kPlanThreads) {
    const int k = k0 + t;
    if (t == 0) s_near = chunks;
    __syncthreads();
    if (k < chunks && load(hi + k * kSpanChunk) != kOpen) atomicMin(&s_near, k);
    __syncthreads();
    const int near = s_near;
    __syncthreads();
    if (near == chunks) continue;
    end = load(hi + near * kSpanChunk);
    break;
  }
  for (int i = c0 + t; i < c1; i += kPlanThreads) {
    if (open_lo) fill(lo + i, start);
    if (open_hi) fill(hi + i, end);
  }
}

hipError_t launch_spans(const SpanParams& p, hipStream_t stream) {
  if (p.B <= 0 || p.S <= 0) return hipSuccess;
  // (Rows in the grid's second dimension, at most 65535 a launch.)
  for (int b = 0; b < p.B; b += 65535) {
    SpanParams q = p;
    q.ids += b * p.stride;
    q.lo += (int64_t)b * p.S;
    q.hi += (int64_t)b * p.S;
    const dim3 grid((p.S + kSpanChunk - 1) / kSpanChunk, std::min(p.B - b, 65535));
    if (p.S <= kSpanWalk) {
      hipLaunchKernelGGL(gqa_spans_kernel<true>, grid, dim3(kPlanThreads), 0, stream, q);
    } else {
      hipLaunchKernelGGL(gqa_spans_kernel<false>, grid, dim3(kPlanThreads), 0, stream, q);
      hipLaunchKernelGGL(gqa_spans_join_kernel, grid, dim3(kPlanThreads), 0, stream, q);
    }
  }
  return hipGetLastError();
}

// The first request of each pool row owns it; owner[row] = that request.
// Rows outside the pool have none.
__device__ inline void claim_rows(const int* rows, int B, int n_rows, int* owner) {
  for (int b = threadIdx.x; b < B; b += kPlanThreads) {
    const int r = rows != nullptr ? rows[b] : b;
    if (r >= 0 && r < n_rows) __hip_atomic_store(&owner[r], 0x7fffffff, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __threadfence();
  __syncthreads();
  for (int b = threadIdx.x; b < B; b += kPlanThreads) {
    const int r = rows != nullptr ? rows[b] : b;
    if (r >= 0 && r < n_rows) atomicMin(&owner[r], b);
  }
  __threadfence();
  __syncthreads();
}
__device__ inline bool owns(const int* owner, int r, int b) {
  return __hip_atomic_load(const_cast<int*>(owner + r), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == b;
}

// First launch of a step, one workgroup: which requests are served, their new
// lengths, and how many free blocks are taken before each one's.
__global__ __launch_bounds__(kPlanThreads) void gqa_tables_plan_kernel(TablesParams p) {
  __shared__ int64_t tmp[kPlanThreads / 64];
  __shared__ int s_refused;
  int* owner = p.scratch;
  int* old_len = p.scratch + p.n_rows;
  int* base = old_len + p.B;
  const int have_free = min(max(*p.free_count, 0), p.n_free);
  const int mask = (1 << p.block_shift) - 1;
  if (threadIdx.x == 0) {
    s_refused = 0;
    base[p.B] = have_free;  // for the second launch
  }
  claim_rows(p.rows, p.B, p.n_rows, owner);
  int64_t tokens = 0, blocks = 0, taken = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    int r = -1, fresh = 0, old = 0;
    bool fits = false;
    if (b < p.B) {
      r = p.rows != nullptr ? p.rows[b] : b;
      fresh = max(p.new_lens[b], 0);
      fits = r >= 0 && r < p.n_rows && owns(owner, r, b);
      old = fits ? min(max(p.lens[r], 0), p.width << p.block_shift) : 0;
    }
    int64_t total;
    const int64_t upto = block_scan(fresh, tmp, total) + tokens;
    tokens += total;
    const int64_t start = upto - fresh;
    const int64_t len = (int64_t)old + fresh;
    fits = fits && len <= ((int64_t)p.width << p.block_shift) && upto <= p.n_tokens;
    const int pages = (old + mask) >> p.block_shift;
    const int need = fits ? (int)((len + mask) >> p.block_shift) - pages : 0;
    const int64_t bl = block_scan(need, tmp, total) + blocks;
    blocks += total;
    const bool ok = fits && (need == 0 || bl <= have_free);
    block_scan(ok ? need : 0, tmp, total);
    taken += total;
    if (b < p.B) {
      const int now = ok ? (int)len : old;
      p.seq_lens[b] = now;
      p.query_start[b] = (int)min(start, (int64_t)0x7fffffff);
      p.query_lens[b] = ok ? fresh : 0;
      old_len[b] = old;
      base[b] = (int)min(bl - need, (int64_t)0x7fffffff);
      if (ok && p.update) p.lens[r] = now;
      // (A negative row is an empty place of the batch.)
      if (!ok && r >= 0) atomicAdd(&s_refused, 1);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    *p.new_free = have_free - (int)taken;
    *p.refused = s_refused;
    if (p.update) *p.free_count = have_free - (int)taken;
  }
}

// Second launch: one thread an item, the tokens' slots and positions, then the
// entries of the batch's tables (new pages also go to the pool's).
__global__ __launch_bounds__(256) void gqa_tables_expand_kernel(TablesParams p) {
  const int* old_len = p.scratch + p.n_rows;
  const int* base = old_len + p.B;
  const int mask = (1 << p.block_shift) - 1;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t n_entries = (int64_t)p.B * p.width;
  if (item >= p.n_tokens + n_entries) return;
  // The block of page `page` of request b: the pool's, or a new one.
  const auto block_of = [&](int b, int page, bool& fresh) {
    const int pages = (old_len[b] + mask) >> p.block_shift;
    fresh = page >= pages;
    const int r = p.rows != nullptr ? p.rows[b] : b;
    return fresh ? p.free_blocks[base[p.B] - 1 - base[b] - (page - pages)]
                 : p.tables[r * p.stride + page];
  };
  if (item < p.n_tokens) {
    const int t = (int)item;
    int b = 0;  // the last request that starts at or before t
    for (int n = p.B; n > 1;) {
      const int half = n >> 1;
      if (p.query_start[b + half] <= t) b += half;
      n -= half;
    }
    // (Requests without tokens start where the next one does: the last of
    // them is the one that holds t, if it has any.)
    const int j = p.B > 0 ? t - p.query_start[b] : 0;
    int64_t slot = -1;
    int pos = 0;
    if (p.B > 0 && j < p.query_lens[b]) {
      pos = old_len[b] + j;
      bool fresh;
      slot = ((int64_t)block_of(b, pos >> p.block_shift, fresh) << p.block_shift) + (pos & mask);
    }
    p.slots[t] = slot;
    p.positions[t] = pos;
    return;
  }
  const int64_t e = item - p.n_tokens;
  const int b = (int)(e / p.width), page = (int)(e - (int64_t)b * p.width);
  int x = 0;
  if (page < ((p.seq_lens[b] + mask) >> p.block_shift)) {
    bool fresh;
    x = block_of(b, page, fresh);
    if (fresh) p.tables[(p.rows != nullptr ? p.rows[b] : b) * p.stride + page] = x;
  }
  p.batch_tables[e] = x;
}

// The step in one launch, for batches whose plan fits LDS: every workgroup makes
// the plan for itself (two dependent reads and two sums over the batch) and then
// its share of the tokens and of the tables' rows; nothing that another
// workgroup's plan reads is written (the pool's lengths and the free count move
// on in a launch behind, gqa_tables_update_kernel; with one workgroup at its end).
// Bound by that chain of reads, not by its bytes: 256 requests of up to 8000 keys
// as a plan 6.1 us (plan and expansion in a launch each: 15.3), 256 of 4000 keys with
// the launch behind 6.9, 41663 tokens of 48 prompts as a plan 7.3.
constexpr int kStepMaxBatch = 2048, kStepMaxRows = 4096, kStepMaxTokens = 1 << 18;  // (48 KiB of LDS)

__device__ inline int block_sum_scan(int x, int* tmp, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  __syncthreads();  // tmp's readers of the call before
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    const int y = tmp[w];
    if (w < wave) before += y;
    total += y;
  }
  return before + x;
}

// block_sum_scan of counts from 0 to 2^31 - 1, which may pass 32 bits together: a
// wave that has one over 2^17 says -2^27 in place of its sum (the others' are 2^23 at
// most), which makes the total negative, and the sums are made in 64.
__device__ inline int64_t block_count_scan(int n, int* tmp, int64_t* tmp64, int64_t& total) {
  const bool large = __builtin_amdgcn_ballot_w64(n > (1 << 17)) != 0;
  int sum;
  const int upto = block_sum_scan(large ? ((threadIdx.x & 63) == 0 ? -(1 << 27) : 0) : n, tmp, sum);
  total = sum;
  return __builtin_expect(sum < 0, 0) ? block_scan(n, tmp64, total) : upto;
}

__global__ __launch_bounds__(kPlanThreads) void gqa_tables_step_kernel(TablesParams p) {
  extern __shared__ int lds[];
  __shared__ int tmp[kPlanThreads / 64], s_refused, s_taken;
  __shared__ int64_t tmp64[kPlanThreads / 64];
  int* s_start = lds;           // (B) first token
  int* s_old = s_start + p.B;   // (B) keys before
  int* s_new = s_old + p.B;     // (B) new tokens, 0 if refused
  int* s_base = s_new + p.B;    // (B) free blocks taken before
  int* owner = s_base + p.B;    // (n_rows), with rows
  const int t = threadIdx.x;
  const int have_free = min(max(load_uniform(p.free_count), 0), p.n_free);
  const int mask = (1 << p.block_shift) - 1;
  if (t == 0) s_refused = s_taken = 0;
  if (p.rows != nullptr) {
    for (int r = t; r < p.n_rows; r += kPlanThreads) owner[r] = 0x7fffffff;
    __syncthreads();
    for (int b = t; b < p.B; b += kPlanThreads) {
      const int r = p.rows[b];
      if (r >= 0 && r < p.n_rows) atomicMin(&owner[r], b);
    }
  }
  __syncthreads();
  int64_t tokens = 0;
  int blocks = 0;
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + t;
    int r = -1, fresh = 0, old = 0;
    bool fits = false;
    if (b < p.B) {
      r = p.rows != nullptr ? p.rows[b] : b;
      fresh = max(p.new_lens[b], 0);
      fits = r >= 0 && r < p.n_rows && (p.rows == nullptr || owner[r] == b);
      old = fits ? min(max(p.lens[r], 0), p.width << p.block_shift) : 0;
    }
    int total;
    int64_t asked;
    const int64_t upto = block_count_scan(fresh, tmp, tmp64, asked) + tokens;
    tokens += asked;
    const int64_t len = (int64_t)old + fresh;
    fits = fits && len <= ((int64_t)p.width << p.block_shift) && upto <= p.n_tokens;
    const int pages = (old + mask) >> p.block_shift;
    const int need = fits ? (int)((len + mask) >> p.block_shift) - pages : 0;
    const int bl = block_sum_scan(need, tmp, total) + blocks;
    blocks += total;
    const bool ok = fits && (need == 0 || bl <= have_free);
    if (b < p.B) {
      s_start[b] = (int)min(upto - fresh, (int64_t)0x7fffffff);
      s_old[b] = old;
      s_new[b] = ok ? fresh : 0;
      s_base[b] = bl - need;
      if (ok && need > 0) atomicMax(&s_taken, bl);  // (served requests' sums come before any refused one's)
      if (!ok && r >= 0) atomicAdd(&s_refused, 1);
    }
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int b = t; b < p.B; b += kPlanThreads) {
      p.seq_lens[b] = s_old[b] + s_new[b];
      p.query_start[b] = s_start[b];
      p.query_lens[b] = s_new[b];
    }
    if (t == 0) {
      *p.new_free = have_free - s_taken;
      *p.refused = s_refused;
    }
  }
  // The block of page `page` of request b: the pool's, or a new one.
  const auto block_of = [&](int b, int r, int page) {
    const int pages = (s_old[b] + mask) >> p.block_shift;
    return page >= pages ? p.free_blocks[have_free - 1 - s_base[b] - (page - pages)] : p.tables[r * p.stride + page];
  };
  // Tokens, one a thread; the request by bisection.
  for (int i = blockIdx.x * kPlanThreads + t; i < p.n_tokens; i += gridDim.x * kPlanThreads) {
    int b = 0;  // the last request that starts at or before token i
    for (int n = p.B; n > 1;) {
      const int half = n >> 1;
      if (s_start[b + half] <= i) b += half;
      n -= half;
    }
    int64_t slot = -1;
    int pos = 0;
    const int at = p.B > 0 ? i - s_start[b] : 0;
    if (p.B > 0 && at < s_new[b]) {
      pos = s_old[b] + at;
      const int r = p.rows != nullptr ? p.rows[b] : b;
      slot = ((int64_t)block_of(b, r, pos >> p.block_shift) << p.block_shift) + (pos & mask);
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
  }
  // Table rows, one a wave.
  const int lane = t & 63;
  for (int b = blockIdx.x * (kPlanThreads / 64) + (t >> 6); b < p.B; b += gridDim.x * (kPlanThreads / 64)) {
    const int r = p.rows != nullptr ? p.rows[b] : b;
    const int n = (s_old[b] + s_new[b] + mask) >> p.block_shift, pages = (s_old[b] + mask) >> p.block_shift;
    int* out = p.batch_tables + (int64_t)b * p.width;
#pragma unroll 4
    for (int page = lane; page < p.width; page += 64) {
      int x = 0;
      if (page < n) {
        x = block_of(b, r, page);
        if (page >= pages) p.tables[r * p.stride + page] = x;
      }
      out[page] = x;
    }
  }
  if (gridDim.x > 1 || !p.update) return;
  // One workgroup, which has read all that its plan reads: the pool moves on here.
  for (int b = t; b < p.B; b += kPlanThreads)
    if (s_new[b] > 0) p.lens[p.rows != nullptr ? p.rows[b] : b] = s_old[b] + s_new[b];
  if (t == 0) *p.free_count = have_free - s_taken;
}

// The pool moves on: lengths of the served requests, the free count.
__global__ __launch_bounds__(256) void gqa_tables_update_kernel(TablesParams p) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < p.B && p.query_lens[b] > 0) p.lens[p.rows != nullptr ? p.rows[b] : b] = p.seq_lens[b];
  if (b == 0) *p.free_count = *p.new_free;
}

hipError_t launch_tables(const TablesParams& p, hipStream_t stream) {
  const int64_t entries = (int64_t)p.B * p.width;
  if (p.B <= kStepMaxBatch && p.n_rows <= kStepMaxRows && p.n_tokens < kStepMaxTokens && entries < (int64_t)1 << 30) {
    // A table row a wave, a few thousand tokens a workgroup.  Small steps that move
    // the pool on: one workgroup, and no launch behind it (us on the GPU and on the
    // host, several / one: 1-16 requests of 500 pages 6.0 and 8.8 / 4.8 and 6.0, 32 of
    // them 6.2 and 8.8 / 6.5 and 5.8, 8 with 4096 tokens 5.2 and 8.9 / 4.4 and 5.9; more
    // rows, 256 of 32 pages 5.1 / 8.6, or tokens, 8192 of 48 5.9 / 8.0, not).
    int wgs = std::min(std::max({(p.B + 15) / 16, (p.n_tokens + 2047) / 2048, 1}), 256);
    if (p.update && p.B <= 32 && p.n_tokens <= 4096 && entries <= 16 * kPlanThreads) wgs = 1;
    const size_t lds = sizeof(int) * (4 * (size_t)p.B + (p.rows != nullptr ? p.n_rows : 0));
    hipLaunchKernelGGL(gqa_tables_step_kernel, dim3(wgs), dim3(kPlanThreads), lds, stream, p);
    if (p.update && wgs > 1)
      hipLaunchKernelGGL(gqa_tables_update_kernel, dim3((p.B + 255) / 256 + (p.B == 0)), dim3(256), 0, stream, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(gqa_tables_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
  const int64_t items = p.n_tokens + entries;
  if (items > 0)
    hipLaunchKernelGGL(gqa_tables_expand_kernel, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

// Blocks of released rows go back on the free list, the rows' lengths to zero;
// one workgroup.
__global__ __launch_bounds__(kPlanThreads) void gqa_release_kernel(ReleaseParams p) {
  __shared__ int64_t tmp[kPlanThreads / 64];
  __shared__ int s_row[kPlanThreads], s_at[kPlanThreads], s_n[kPlanThreads];
  const int mask = (1 << p.block_shift) - 1;
  claim_rows(p.rows, p.B, p.n_rows, p.scratch);
  int64_t at = min(max(*p.free_count, 0), p.n_free);
  for (int b0 = 0; b0 < p.B; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    int r = -1, n = 0;
    if (b < p.B) {
      r = p.rows[b];
      if (r >= 0 && r < p.n_rows && owns(p.scratch, r, b))
        n = (min(max(p.lens[r], 0), p.width << p.block_shift) + mask) >> p.block_shift;
      else
        r = -1;
    }
    int64_t total;
    const int64_t upto = block_scan(n, tmp, total);
    s_row[threadIdx.x] = r;
    s_at[threadIdx.x] = (int)min(at + upto - n, (int64_t)0x7fffffff);
    s_n[threadIdx.x] = n;
    __syncthreads();
    for (int w = threadIdx.x >> 6; w < kPlanThreads; w += kPlanThreads / 64)
      for (int i = threadIdx.x & 63; i < s_n[w]; i += 64)
        // (Never past the list, whatever the pool's lengths claim.)
        if (s_at[w] + i < p.n_free) p.free_blocks[s_at[w] + i] = p.tables[s_row[w] * p.stride + i];
    if (r >= 0) p.lens[r] = 0;
    at += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.free_count = (int)min(at, (int64_t)p.n_free);
}

hipError_t launch_release(const ReleaseParams& p, hipStream_t stream) {
  if (p.B <= 0) return hipSuccess;
  hipLaunchKernelGGL(gqa_release_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace gqa
