// Page tables of many sequences from their lengths (tlm_op_paged_reserve).
#include <algorithm>

#include "tlm_device.h"
#include "tlm_paged.h"

namespace tlm {
namespace {

// Per sequence s with L = lengths[s] and R rows to come, the pages in use are those of
// paged_use(L, R).  What its table holds besides goes back (refs - 1).  What it lacks
// of those past L is taken: the sequences in their order, the free pages (refs 0)
// lowest first, as long as the sum of what has been asked for so far is no more than
// the free pages.  A sequence that lacks one that holds positions below L gets nothing.
constexpr int kSegment = 4096;  // pages whose free ones a block counts

// a.work: want[seqs] (pages that a sequence lacks, -1 where positions are lost), then
// base[seqs] (before it, or -1: it gets none), the free pages before each segment, the
// number taken, and the pages taken in order.
struct Work {
  int32_t *want, *base, *segment, *taken, *pages;
  int segments;
};
__host__ __device__ inline Work work_of(const ReserveArgs& a) {
  Work w;
  w.segments = (a.num_pages + kSegment - 1) / kSegment;
  w.want = a.work;
  w.base = w.want + a.seqs;
  w.segment = w.base + a.seqs;
  w.taken = w.segment + w.segments;
  w.pages = w.taken + 1;
  return w;
}

struct Seq {
  int length, rows;
  PagedUse use;
  bool bad;
  __device__ __forceinline__ bool used(int i) const { return i < use.sink || (i >= use.first && i < use.end); }
};
__device__ __forceinline__ Seq seq_of(const ReserveArgs& a, int s) {
  Seq q;
  q.length = a.lengths[s];
  q.rows = paged_rows(q.length, a.counts ? a.counts[s] : a.tokens, a.tokens, a.limit, &q.bad);
  q.use = PagedUse{0, 0, 0};
  if (q.length >= 0) {
    // a length past the limit keeps what the table can hold of it
    q.use = paged_use(min(q.length, a.limit), q.rows, a.window, a.sinks, a.page_shift);
  }
  return q;
}

__device__ __forceinline__ int sum64(int v) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) v += __shfl_xor(v, w);
  return v;
}

__global__ __launch_bounds__(256) void reserve_copy_kernel(ReserveArgs a) {
  for (int i = blockIdx.x * 256 + threadIdx.x; i < a.num_pages; i += gridDim.x * 256) a.out_refs[i] = a.refs[i];
}

// What goes back and what is lacking: a wave per sequence.
__global__ __launch_bounds__(256) void reserve_rows_kernel(ReserveArgs a) {
  const int s = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (s >= a.seqs) return;
  const Seq q = seq_of(a, s);
  const int32_t* const from = a.tables + (size_t)s * a.width;
  int32_t* const to = a.out_tables + (size_t)s * a.width;
  int want = 0, lost = 0;
  for (int i = lane; i < a.width; i += 64) {
    const int p = from[i];
    const bool has = p >= 0 && p < a.num_pages, used = q.used(i);
    if (has && !used) atomicSub(a.out_refs + p, 1);
    const bool lacks = used && !has, old = ((int64_t)i << a.page_shift) < q.length;
    want += lacks && !old;
    lost += lacks && old;
    to[i] = has && used ? p : -1;
  }
  want = sum64(want);
  lost = sum64(lost);
  if (lane == 0) {
    work_of(a).want[s] = lost ? -1 : want;
    const int bits = (q.bad ? kPagedStatusRows : 0) | (lost ? kPagedStatusPage : 0);
    if (bits) __hip_atomic_fetch_or(a.status, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

// Sum over a block's threads before each, and over all.
struct Scan {
  int sh[16];
};
__device__ __forceinline__ int64_t scan1024(int v, Scan& sc, int64_t* all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int incl = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(incl, d);
    if (lane >= d) incl += x;
  }
  __syncthreads();
  if (lane == 63) sc.sh[w] = incl;
  __syncthreads();
  int64_t before = incl - v, sum = 0;
  for (int i = 0; i < 16; i++) {
    if (i < w) before += sc.sh[i];
    sum += sc.sh[i];
  }
  *all = sum;
  return before;
}

// Free pages of each segment; the last block turns them into running sums and shares
// them out.
__global__ __launch_bounds__(1024) void reserve_count_kernel(ReserveArgs a) {
  __shared__ Scan sc;
  __shared__ int last;
  const Work w = work_of(a);
  const int tid = threadIdx.x;
  int n = 0;
#pragma unroll
  for (int k = 0; k < kSegment / 1024; k++) {
    const int64_t i = (int64_t)blockIdx.x * kSegment + k * 1024 + tid;
    n += i < a.num_pages && a.out_refs[i] == 0;
  }
  int64_t all;
  scan1024(n, sc, &all);
  if (tid == 0) {
    __hip_atomic_store(w.segment + blockIdx.x, (int)all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = __hip_atomic_fetch_add(a.arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  if (tid == 0) __hip_atomic_store(a.arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  int64_t free = 0;
  for (int b = 0; b < w.segments; b += 1024) {
    const int v = b + tid < w.segments
                      ? __hip_atomic_load(w.segment + b + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                      : 0;
    const int64_t before = scan1024(v, sc, &all) + free;
    if (b + tid < w.segments) w.segment[b + tid] = (int)before;
    free += all;
  }
  int64_t asked = 0, taken = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 1024) {
    const int s = s0 + tid, want = s < a.seqs ? w.want[s] : -1;
    const int64_t before = scan1024(max(want, 0), sc, &all) + asked;
    const bool gets = want == 0 || (want > 0 && before + want <= free);
    if (s < a.seqs) w.base[s] = gets ? (int)before : -1;
    taken = max(taken, gets ? before + want : 0);
    asked += all;
  }
  // the sequences that get some are the first that ask: the largest end is the number
  for (int d = 1; d < 64; d <<= 1) taken = max(taken, (int64_t)__shfl_xor((int)taken, d));
  __syncthreads();
  if ((tid & 63) == 0) sc.sh[tid >> 6] = (int)taken;
  __syncthreads();
  if (tid == 0) {
    int most = 0;
    for (int i = 0; i < 16; i++) most = max(most, sc.sh[i]);
    *w.taken = most;
  }
}

// The free pages in order, those taken.
__global__ __launch_bounds__(1024) void reserve_take_kernel(ReserveArgs a) {
  __shared__ Scan sc;
  const Work w = work_of(a);
  const int taken = *w.taken;
  int64_t before = w.segment[blockIdx.x], all;
  if (before >= taken) return;
  for (int k = 0; k < kSegment / 1024; k++) {
    const int64_t i = (int64_t)blockIdx.x * kSegment + k * 1024 + threadIdx.x;
    const int free = i < a.num_pages && a.out_refs[i] == 0;
    const int64_t rank = scan1024(free, sc, &all) + before;
    if (free && rank < taken) {
      w.pages[rank] = (int)i;
      a.out_refs[i] = 1;
    }
    before += all;
  }
}

// The pages into the tables, the first positions and the slots: a wave per sequence.
__global__ __launch_bounds__(256) void reserve_fill_kernel(ReserveArgs a) {
  const int s = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (s >= a.seqs) return;
  const Work w = work_of(a);
  const Seq q = seq_of(a, s);
  const int want = w.want[s], base = w.base[s];
  int32_t* const to = a.out_tables + (size_t)s * a.width;
  const int page = 1 << a.page_shift;
  const bool served = q.rows > 0 && base >= 0;
  // what is lacking is all past the length
  const int i0 = max((int)(((int64_t)q.length + page - 1) >> a.page_shift), 0);
  int at = base;
  for (int b = i0; served && want > 0 && b < q.use.end; b += 64) {
    const int i = b + lane;
    const bool lacks = i < q.use.end && to[i] < 0;
    const uint64_t m = __ballot(lacks);
    if (lacks) to[i] = w.pages[at + __popcll(m & ((1ull << lane) - 1))];
    at += __popcll(m);
  }
  if (lane == 0) a.starts[s] = served ? q.length : -1;
  if (!a.slots) return;
  __threadfence_block();
  for (int j = lane; j < a.tokens; j += 64) {
    const int p = q.length + j;
    int64_t slot = -1;
    if (served && j < q.rows) slot = ((int64_t)to[p >> a.page_shift] << a.page_shift) + (p & (page - 1));
    a.slots[(size_t)s * a.tokens + j] = slot;
  }
}

}  // namespace

size_t reserve_work(const ReserveArgs& a) {
  const Work w = work_of(a);
  // a sequence's new rows lie in at most tokens / page pages that begin past its length, rounded up
  const int64_t most = (int64_t)a.seqs * (((int64_t)a.tokens + (1 << a.page_shift) - 1) >> a.page_shift);
  return (size_t)2 * a.seqs + w.segments + 1 + (size_t)std::min<int64_t>(most, a.num_pages);
}

void launch_reserve(const ReserveArgs& a, hipStream_t st) {
  const Work w = work_of(a);
  const dim3 rows((unsigned)((a.seqs + 3) / 4));
  if (a.refs != a.out_refs)
    hipLaunchKernelGGL(reserve_copy_kernel, dim3((unsigned)std::min(1024, (a.num_pages + 255) / 256)), dim3(256), 0, st, a);
  hipLaunchKernelGGL(reserve_rows_kernel, rows, dim3(256), 0, st, a);
  hipLaunchKernelGGL(reserve_count_kernel, dim3((unsigned)w.segments), dim3(1024), 0, st, a);
  hipLaunchKernelGGL(reserve_take_kernel, dim3((unsigned)w.segments), dim3(1024), 0, st, a);
  hipLaunchKernelGGL(reserve_fill_kernel, rows, dim3(256), 0, st, a);
}

}  // namespace tlm
