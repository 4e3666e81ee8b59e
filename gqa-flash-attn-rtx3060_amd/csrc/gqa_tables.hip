// gqa_tables.hip — what describes a batch to the attention kernels, built on
// the device: the spans of documents, and a step's block tables, slots and
// positions from the requests' lengths and a free list that lives there too.
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

// One workgroup a row: thread t takes S / 1024 consecutive tokens; the start of
// the run that reaches into them is the last change before them, the end of
// the run that leaves them the first change behind.
__global__ __launch_bounds__(kPlanThreads) void gqa_spans_kernel(SpanParams p) {
  __shared__ int s_last[kPlanThreads], s_first[kPlanThreads];
  const int t = threadIdx.x;
  const int* ids = p.ids + blockIdx.x * p.stride;
  int* lo = p.lo + (int64_t)blockIdx.x * p.S;
  int* hi = p.hi + (int64_t)blockIdx.x * p.S;
  const int per = (p.S + kPlanThreads - 1) / kPlanThreads;
  const int a = min(t * per, p.S), e = min(a + per, p.S);
  int first = p.S, last = -1;  // changes among the thread's tokens
  for (int i = a; i < e; ++i)
    if (i == 0 || ids[i] != ids[i - 1]) {
      last = i;
      if (first == p.S) first = i;
    }
  s_last[t] = last;
  s_first[t] = first;
  __syncthreads();
  for (int o = 1; o < kPlanThreads; o <<= 1) {  // running maximum from the left, minimum from the right
    const int x = t >= o ? s_last[t - o] : -1, y = t + o < kPlanThreads ? s_first[t + o] : p.S;
    __syncthreads();
    s_last[t] = max(s_last[t], x);
    s_first[t] = min(s_first[t], y);
    __syncthreads();
  }
  int start = t > 0 ? s_last[t - 1] : -1;
  for (int i = a; i < e; ++i) {
    if (i == 0 || ids[i] != ids[i - 1]) start = i;
    lo[i] = ids[i] < 0 ? 0 : start;
  }
  int end = t + 1 < kPlanThreads ? s_first[t + 1] : p.S;
  for (int i = e - 1; i >= a; --i) {
    hi[i] = ids[i] < 0 ? 0 : end;
    if (i == 0 || ids[i] != ids[i - 1]) end = i;
  }
}

hipError_t launch_spans(const SpanParams& p, hipStream_t stream) {
  if (p.B <= 0 || p.S <= 0) return hipSuccess;
  hipLaunchKernelGGL(gqa_spans_kernel, dim3(p.B), dim3(kPlanThreads), 0, stream, p);
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

hipError_t launch_tables(const TablesParams& p, hipStream_t stream) {
  if (p.B <= 0 && p.n_tokens <= 0) return hipSuccess;
  hipLaunchKernelGGL(gqa_tables_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p);
  const int64_t items = p.n_tokens + (int64_t)p.B * p.width;
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
      if (r >= 0 && r < p.n_rows && owns(p.scratch, r, b)) n = (min(max(p.lens[r], 0), p.width << p.block_shift) + mask) >> p.block_shift;
      else r = -1;
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
