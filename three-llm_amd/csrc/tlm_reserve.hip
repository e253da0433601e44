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
constexpr int kSegment = 4096;  // pages whose free ones are counted together
constexpr int kPiece = 512;     // entries of a table that a wave looks at at a time
constexpr int kLost = 1 << 30;  // in want: positions are lost

// Waves that share a sequence's table: enough of them to fill the chip (1024 sequences of
// 1025 entries, pieces of 256 / 512 / 1024 a wave: 14.9 / 15.3 / 15.3 us in all; bound by the
// three launches, of which this one moves 9 MB in 6.4 us, 1.4 of it the counts' atomics; in
// place too, as entries that stay are written back: 7.2).
__host__ __device__ inline int waves_of(const ReserveArgs& a) {
  int n = 1;
  while (2 * n <= 16 && 2 * n * a.seqs <= 4096 && n * kPiece < a.width) n *= 2;
  return n;
}

// a.work: a bit per page, set where it is free; want[seqs][waves] (pages that a sequence
// lacks); the free pages of each segment; of many sequences or segments
// (reserve_share_kernel) also base[seqs] (what the sequences before one lack, or -1: it
// gets none), and of each segment the free pages before it.
struct Work {
  uint64_t* mask;
  int32_t *want, *base, *segment;
  int segments, waves;
};
__host__ __device__ inline Work work_of(const ReserveArgs& a) {
  Work w;
  w.segments = (a.num_pages + kSegment - 1) / kSegment;
  w.waves = waves_of(a);
  w.mask = reinterpret_cast<uint64_t*>(a.work);
  w.want = a.work + (size_t)w.segments * (kSegment / 32);
  w.base = w.want + (size_t)a.seqs * w.waves;
  w.segment = w.base + a.seqs;
  return w;
}

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4u __attribute__((ext_vector_type(4), aligned(4)));  // from any 4-byte address
__device__ __forceinline__ i32x4u four(const int32_t* p, int i, int n, int none) {
  i32x4u v = {none, none, none, none};
  if (i + 4 <= n) return *(const TLM_GLOBAL i32x4u*)(p + i);
#pragma unroll
  for (int e = 0; e < 3; e++)
    if (i + e < n) v[e] = p[i + e];
  return v;
}
__device__ __forceinline__ void put_four(int32_t* p, int i, int n, i32x4u v) {
  if (i + 4 <= n) {
    *(TLM_GLOBAL i32x4u*)(p + i) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 3; e++)
      if (i + e < n) p[i + e] = v[e];
  }
}

struct Seq {
  int length, rows, past;  // past: the first page that begins at its length or later
  PagedUse use;
  bool bad;
  __device__ __forceinline__ bool used(int i) const { return i < use.sink || (i >= use.first && i < use.end); }
};
__device__ __forceinline__ Seq seq_of(const ReserveArgs& a, int s) {
  Seq q;
  q.length = a.lengths[s];
  q.rows = paged_rows(q.length, a.counts ? a.counts[s] : a.tokens, a.tokens, a.limit, &q.bad);
  q.use = PagedUse{0, 0, 0};
  q.past = (int)(((int64_t)q.length + (1 << a.page_shift) - 1) >> a.page_shift);
  if (q.length >= 0) {
    // a length past the limit keeps what the table can hold of it
    q.use = paged_use(min(q.length, a.limit), q.rows, a.window, a.sinks, a.page_shift);
  }
  return q;
}

__device__ __forceinline__ int sum64(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// One entry, `p`, of a sequence's table: what becomes of it; whether the sequence lacks a
// page there, and whether with positions that it has.
struct Entry {
  int becomes;
  bool back, lacks, lost;
};
__device__ __forceinline__ Entry entry_of(const ReserveArgs& a, const Seq& q, int i, int p) {
  const bool has = p >= 0 && p < a.num_pages, used = q.used(i), old = i < q.past;
  return Entry{has && used ? p : -1, has && !used, used && !has && !old, used && !has && old};
}

__device__ __forceinline__ void report(const ReserveArgs& a, bool bad, bool lost) {
  const int bits = (bad ? kPagedStatusRows : 0) | (lost ? kPagedStatusPage : 0);
  if (bits) __hip_atomic_fetch_or(a.status, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The counts as they are, where they do not change in place and the pool is past kReserveBack pages.
__global__ __launch_bounds__(256) void reserve_copy_kernel(ReserveArgs a) {
  const int64_t step = (int64_t)gridDim.x * 1024;
  for (int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x); i < a.num_pages; i += step)
    put_four(a.out_refs, (int)i, a.num_pages, four(a.refs, (int)i, a.num_pages, 0));
}

// What goes back and what is lacking.
__global__ __launch_bounds__(256) void reserve_rows_kernel(ReserveArgs a) {
  const Work w = work_of(a);
  const int item = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, s = item / w.waves;
  if (s >= a.seqs) return;
  const int32_t* const from = a.tables + (size_t)s * a.width;
  int32_t* const to = a.out_tables + (size_t)s * a.width;
  const Seq q = seq_of(a, s);
  int want = 0, lost = 0;
  for (int64_t i0 = item % w.waves * kPiece; i0 < a.width; i0 += w.waves * kPiece) {
    i32x4u v[kPiece / 256];
#pragma unroll
    for (int k = 0; k < kPiece / 256; k++) v[k] = four(from, (int)i0 + 256 * k + 4 * lane, a.width, -1);
#pragma unroll
    for (int k = 0; k < kPiece / 256; k++) {
      const int i = (int)i0 + 256 * k + 4 * lane;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (i + e >= a.width) continue;
        const Entry x = entry_of(a, q, i + e, v[k][e]);
        if (x.back && a.back) atomicAdd(a.back + v[k][e], 1);
        if (x.back && !a.back) atomicSub(a.out_refs + v[k][e], 1);
        want += x.lacks;
        lost |= x.lost;
        v[k][e] = x.becomes;
      }
      put_four(to, i, a.width, v[k]);
    }
  }
  want = sum64(want);
  lost = __ballot(lost) != 0;
  if (lane == 0) {
    w.want[item] = lost ? kLost : want;
    report(a, q.bad && item % w.waves == 0, lost);
  }
}

// Sum over a block's threads before each, and over all.
struct Scan {
  int sh[16];
};
__device__ __forceinline__ int64_t scan1024(int v, Scan& sc, int64_t* all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int incl = wave_scan(v);
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

// The counts without what goes back (a.back: cleared again), which pages are free and how
// many of each segment, a block each.
__global__ __launch_bounds__(1024) void reserve_count_kernel(ReserveArgs a) {
  __shared__ int sh[16];
  const Work w = work_of(a);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int32_t* const from = a.back ? a.refs : a.out_refs;
  int c[kSegment / 1024], b[kSegment / 1024], free = 0;
#pragma unroll
  for (int k = 0; k < kSegment / 1024; k++) {
    const int64_t i = (int64_t)blockIdx.x * kSegment + 1024 * k + tid;
    c[k] = i < a.num_pages ? from[i] : 1;
    b[k] = i < a.num_pages && a.back ? a.back[i] : 0;
  }
#pragma unroll
  for (int k = 0; k < kSegment / 1024; k++) {
    const int64_t i = (int64_t)blockIdx.x * kSegment + 1024 * k + tid;
    c[k] -= b[k];
    if (b[k]) a.back[i] = 0;
    if (i < a.num_pages && a.back && (b[k] || a.refs != a.out_refs)) a.out_refs[i] = c[k];
    const uint64_t m = __ballot(c[k] == 0);
    if (lane == 0) w.mask[(size_t)blockIdx.x * (kSegment / 64) + 16 * k + wave] = m;
    free += __popcll(m);
  }
  if (lane == 0) sh[wave] = free;
  __syncthreads();
  int all = 0;
  for (int i = 0; i < 16; i++) all += sh[i];
  if (tid == 0) w.segment[blockIdx.x] = all;
}

// What sequence s lacks in all (kLost: positions).
__device__ __forceinline__ int want_of(const Work& w, int s) {
  int x[16], want = 0, lost = 0;
#pragma unroll
  for (int k = 0; k < 16; k++) x[k] = k < w.waves ? w.want[(size_t)s * w.waves + k] : 0;
#pragma unroll
  for (int k = 0; k < 16; k++) want += x[k] & ~kLost, lost |= x[k] & kLost;
  return lost ? kLost : want;
}
// Where its pages begin among the free ones, or -1: none are left for it.
__device__ __forceinline__ int base_of(int want, int64_t before, int64_t free) {
  return want != kLost && (want == 0 || before + want <= free) ? (int)before : -1;
}

// Running sums over many sequences or segments, by one block; up to 1024 of each the
// kernels below work them out for themselves.
constexpr int kInPlace = 1024;
__global__ __launch_bounds__(1024) void reserve_share_kernel(ReserveArgs a) {
  __shared__ Scan sc;
  const Work w = work_of(a);
  const int tid = threadIdx.x;
  int64_t free = 0, asked = 0, all;
  for (int b = 0; b < w.segments; b += 1024) {
    const int64_t before = scan1024(b + tid < w.segments ? w.segment[b + tid] : 0, sc, &all) + free;
    if (b + tid < w.segments) w.segment[b + tid] = (int)before;
    free += all;
  }
  for (int s0 = 0; s0 < a.seqs; s0 += 1024) {
    const int s = s0 + tid, want = s < a.seqs ? want_of(w, s) : kLost;
    const int64_t before = scan1024(want == kLost ? 0 : want, sc, &all) + asked;
    if (s < a.seqs) w.base[s] = base_of(want, before, free);
    asked += all;
  }
}

// The last segment before which there are at most `rank` free pages (which holds that
// one), 64 at a time.
template <typename B>
__device__ __forceinline__ int segment_of(int rank, int segments, int lane, B before) {
  int lo = 0, len = segments;
  while (true) {
    const int step = (len + 63) / 64, i = lane * step;
    const int k = __popcll(__ballot(i < len && before(lo + min(i, len - 1)) <= rank)) - 1;  // the first is
    lo += k * step;
    len = min(step, len - k * step);
    if (step == 1) return lo;
  }
}

// The free pages of ranks at .. at + n - 1, n <= 64, a lane each (`pick`: the wave's 64 words of LDS);
// -1 where none is, which is so only if the inputs change during the call.
template <typename B>
__device__ __forceinline__ int pages_at(const Work& w, int at, int n, int lane, int* pick, B before) {
  __hip_atomic_store(pick + lane, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  for (int r = at; r < at + n;) {
    const int g = segment_of(r, w.segments, lane, before);
    uint64_t word = w.mask[(size_t)g * (kSegment / 64) + lane];
    const int c = __popcll(word), incl = wave_scan(c);
    int rank = before(g) + incl - c;
    if (rank + c <= r) word = 0;
    for (; word && rank < at + n; word &= word - 1, rank++)
      if (rank >= r)
        __hip_atomic_store(pick + rank - at, g * kSegment + 64 * lane + __builtin_ctzll(word), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_WORKGROUP);
    r = max(r + 1, before(g) + __builtin_amdgcn_readlane(incl, 63));
  }
  // a wave's LDS instructions are done in their order
  return __hip_atomic_load(pick + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// The pages that a sequence gets into its table, its first position and its slots: a wave.
// `entry`: its table's at the first of the pages past its length + lane.
template <typename B>
__device__ __forceinline__ void fill(const ReserveArgs& a, const Work& w, const Seq& q, int s, int base, int lane,
                                     int entry, int* pick, B before) {
  int32_t* const to = a.out_tables + (size_t)s * a.width;
  const int page = 1 << a.page_shift;
  const bool served = q.rows > 0 && base >= 0;
  // what is lacking is all past the length
  const int i0 = max(q.past, 0);
  int at = base;
  for (int b = i0; served && b < q.use.end; b += 64) {
    const int i = b + lane;
    const bool lacks = i < q.use.end && (b == i0 ? entry : to[i]) < 0;
    const uint64_t m = __ballot(lacks);
    const int n = __popcll(m);
    if (n) {
      const int got = pages_at(w, at, n, lane, pick, before);
      const int p = __shfl(got, __popcll(m & ((1ull << lane) - 1)));
      if (lacks && p >= 0) {
        to[i] = p;
        a.out_refs[p] = 1;
      }
    }
    at += n;
  }
  if (lane == 0) a.starts[s] = served ? q.length : -1;
  if (!a.slots) return;
  __threadfence_block();
  for (int j = lane; j < a.tokens; j += 64) {
    int64_t slot = -1;
    if (served && j < q.rows) {
      const int p = q.length + j;
      slot = ((int64_t)to[p >> a.page_shift] << a.page_shift) + (p & (page - 1));
    }
    a.slots[(size_t)s * a.tokens + j] = slot;
  }
}

template <bool SHARED>
__global__ __launch_bounds__(1024) void reserve_fill_kernel(ReserveArgs a) {
  __shared__ Scan sc;
  __shared__ int base[kInPlace], segment[kInPlace], picks[1024];
  const Work w = work_of(a);
  const int tid = threadIdx.x, s = blockIdx.x * 16 + (tid >> 6);
  int* const pick = picks + (tid & ~63);
  Seq q;
  int entry = 0;  // on its way while the sums are made
  if (s < a.seqs) {
    q = seq_of(a, s);
    const int i = max(q.past, 0) + (tid & 63);
    if (i < q.use.end) entry = a.out_tables[(size_t)s * a.width + i];
  }
  if (!SHARED) {
    const int want = tid < a.seqs ? want_of(w, tid) : kLost, mine = tid < w.segments ? w.segment[tid] : 0;
    int64_t free, all;
    segment[tid] = (int)scan1024(mine, sc, &free);
    const int64_t before = scan1024(want == kLost ? 0 : want, sc, &all);
    base[tid] = base_of(want, before, free);
    __syncthreads();
  }
  if (s >= a.seqs) return;
  if (SHARED)
    fill(a, w, q, s, w.base[s], tid & 63, entry, pick, [&](int g) { return w.segment[g]; });
  else
    fill(a, w, q, s, base[s], tid & 63, entry, pick, [&](int g) { return segment[g]; });
}

// Few sequences over a small pool: all of it by one block, with the counts, what is
// shared out and the pages of the new rows in LDS, in place of three launches.
// us a call, so / by launches: 16 sequences of 32 pages 4.3 / 10.2, 64 of 128 7.8 / 11.5, 60 of 313
// 11.9 / 12.2, 60 of 469 15.6 / 12.1, 256 of 125 17.6 / 12.5.  It is the instructions of one CU, about 40 an entry.
constexpr int kOnePages = 16384, kOneSeqs = 1024, kOneEntries = 20480, kOneRows = 4096, kOneSlots = 65536;
__host__ __device__ inline int span_of(const ReserveArgs& a) {  // pages that a sequence's new rows may touch
  return ((a.tokens - 1) >> a.page_shift) + 2;
}
// n / d for n * d below 2^32, by = by_of(d).
__host__ __device__ inline uint32_t by_of(int d) { return (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); }
__device__ __forceinline__ int over(int n, int d, uint32_t by) { return d == 1 ? n : (int)__umulhi((uint32_t)n, by); }

__global__ __launch_bounds__(1024) void reserve_one_kernel(ReserveArgs a, uint32_t by_width, uint32_t by_tokens) {
  constexpr int A = 8;  // entries in flight a thread
  __shared__ __align__(16) int refs[kOnePages];
  __shared__ uint16_t pages[kOnePages];
  __shared__ Seq seqs[kOneSeqs];
  __shared__ int want[kOneSeqs];
  __shared__ bool served[kOneSeqs];
  __shared__ int rowpage[kOneRows];  // of the pages from the one of position `length` on
  __shared__ Scan sc;
  const int tid = threadIdx.x, cells = a.seqs * a.width, span = span_of(a);
  int entry[A];
#pragma unroll
  for (int k = 0; k < A; k++) entry[k] = tid + 1024 * k < cells ? a.tables[tid + 1024 * k] : -1;
  for (int i = 4 * tid; i < a.num_pages; i += 4096)
    *reinterpret_cast<i32x4*>(refs + i) = four(a.refs, i, a.num_pages, 1);
  if (tid < a.seqs) {
    const Seq q = seq_of(a, tid);
    seqs[tid] = q;
    want[tid] = 0;
    report(a, q.bad, false);
  }
  __syncthreads();
  // what goes back and what is lacking
  for (int c0 = tid; c0 < cells; c0 += A * 1024) {
#pragma unroll
    for (int k = 0; k < A; k++) {
      const int c = c0 + 1024 * k, p = entry[k];
      if (c >= cells) continue;
      const int s = over(c, a.width, by_width), i = c - s * a.width;
      const Seq q = seqs[s];
      const Entry x = entry_of(a, q, i, p);
      if (x.back) atomicSub(refs + p, 1);
      if (x.lacks) atomicAdd(want + s, 1);
      if (x.lost) atomicOr(want + s, kLost);
      const int at = i - (q.length >> a.page_shift);
      if (at >= 0 && at < span) rowpage[s * span + at] = x.lacks ? -2 : x.becomes;
      a.out_tables[c] = x.becomes;
      entry[k] = c + A * 1024 < cells ? a.tables[c + A * 1024] : -1;
    }
  }
  __syncthreads();
  // the free pages that are asked for, lowest first; a sequence gets what it lacks while
  // it is no more than these
  const int mine = tid < a.seqs ? want[tid] : kLost;
  const bool lost = mine & kLost;
  int64_t asked, free = 0;
  const int64_t before = scan1024(lost ? 0 : mine, sc, &asked);
  for (int b = 0; b < a.num_pages && free < asked; b += 4096) {
    const int i = b + 4 * tid;
    i32x4 v = {1, 1, 1, 1};
    if (i < a.num_pages) v = *reinterpret_cast<const i32x4*>(refs + i);
    int64_t all;
    int64_t rank = free + scan1024((v[0] == 0) + (v[1] == 0) + (v[2] == 0) + (v[3] == 0), sc, &all);
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (v[e] == 0 && rank < asked) pages[rank++] = (uint16_t)(i + e);
    free += all;
  }
  __syncthreads();
  if (tid < a.seqs) {
    const bool gets = !lost && (mine == 0 || before + mine <= free);
    const Seq q = seqs[tid];
    const bool serve = q.rows > 0 && gets;
    report(a, false, lost);
    a.starts[tid] = serve ? q.length : -1;
    served[tid] = serve;
    const int first = q.length >> a.page_shift;
    int at = (int)before;
    for (int k = 0; serve && k < span && first + k < q.use.end; k++)
      if (rowpage[tid * span + k] == -2) {
        const int p = pages[at++];
        rowpage[tid * span + k] = p;
        refs[p] = 1;
        a.out_tables[tid * a.width + first + k] = p;
      }
  }
  __syncthreads();
  for (int i = 4 * tid; i < a.num_pages; i += 4096)
    put_four(a.out_refs, i, a.num_pages, *reinterpret_cast<const i32x4*>(refs + i));
  if (!a.slots) return;
  for (int c = tid; c < a.seqs * a.tokens; c += 1024) {
    const int s = over(c, a.tokens, by_tokens), j = c - s * a.tokens;
    const Seq& q = seqs[s];
    int64_t slot = -1;
    if (served[s] && j < q.rows) {
      const int p = q.length + j, k = (p >> a.page_shift) - (q.length >> a.page_shift);
      slot = ((int64_t)rowpage[s * span + k] << a.page_shift) + (p & ((1 << a.page_shift) - 1));
    }
    a.slots[c] = slot;
  }
}

}  // namespace

size_t reserve_work(const ReserveArgs& a) {
  const Work w = work_of(a);
  return (size_t)(w.segment - a.work) + w.segments;
}

// Past one block: three launches; the running sums are one more past kInPlace sequences or
// segments, the counts' copy another past kReserveBack pages where the result is not in place.
void launch_reserve(const ReserveArgs& a, hipStream_t st) {
  if (a.num_pages <= kOnePages && a.seqs <= kOneSeqs && (int64_t)a.seqs * a.width <= kOneEntries &&
      (int64_t)a.seqs * span_of(a) <= kOneRows && (int64_t)a.seqs * a.tokens <= kOneSlots) {
    hipLaunchKernelGGL(reserve_one_kernel, dim3(1), dim3(1024), 0, st, a, by_of(a.width), by_of(a.tokens));
    return;
  }
  const Work w = work_of(a);
  const dim3 segments((unsigned)w.segments);
  if (!a.back && a.refs != a.out_refs)
    hipLaunchKernelGGL(reserve_copy_kernel, dim3((unsigned)std::min(1024, a.num_pages / 1024 + 1)), dim3(256), 0, st, a);
  hipLaunchKernelGGL(reserve_rows_kernel, dim3((unsigned)((a.seqs * w.waves + 3) / 4)), dim3(256), 0, st, a);
  hipLaunchKernelGGL(reserve_count_kernel, segments, dim3(1024), 0, st, a);
  const dim3 rows((unsigned)((a.seqs + 15) / 16));
  if (a.seqs > kInPlace || w.segments > kInPlace) {
    hipLaunchKernelGGL(reserve_share_kernel, dim3(1), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(reserve_fill_kernel<true>, rows, dim3(1024), 0, st, a);
  } else {
    hipLaunchKernelGGL(reserve_fill_kernel<false>, rows, dim3(1024), 0, st, a);
  }
}

}  // namespace tlm
