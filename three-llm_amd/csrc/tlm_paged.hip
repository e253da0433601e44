// Serving many sequences from a paged cache: the new rows of every sequence
// rotated and appended to its pages (tlm_op_paged_append), and their attention
// over those pages (tlm_op_paged_attention).
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "tlm_device.h"
#include "tlm_paged.h"

namespace tlm {
namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // a row from any 4-byte address

__device__ __forceinline__ void paged_flag(int* status, int bit) {
  __hip_atomic_fetch_or(status, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The append: q' = R(p) q, k' = R(p) k (rotate-half over the first rd dims) and v,
// k' and v rounded to the cache's type.  Three kernels.
//
// Element by element, a block per row: rotary dimensions that are no multiple of 16.
template <typename KT>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedArgs a) {
  constexpr int E = 16 / sizeof(KT);
  const int s = blockIdx.x / a.tokens, j = blockIdx.x % a.tokens;
  const int start = a.starts[s];
  bool bad;
  const int rows = paged_rows(start, a.counts ? a.counts[s] : a.tokens, a.tokens, a.limit, &bad);
  if (bad && j == 0 && threadIdx.x == 0) paged_flag(a.status, kPagedStatusRows);
  if (j >= rows) return;
  const int pos = start + j;
  const int page = paged_page(a.tables + (size_t)s * a.width, pos, a.page_shift, a.num_pages);
  if (page < 0 && threadIdx.x == 0) paged_flag(a.status, kPagedStatusPage);
  const int D = a.D, half = a.rd / 2, n = (a.Hq + 2 * a.Hkv) * D;
  const float* x = a.x + (size_t)blockIdx.x * n;
  const float* cs = a.rope_cos + (size_t)pos * half;
  const float* sn = a.rope_sin + (size_t)pos * half;
  const int tok = pos & ((1 << a.page_shift) - 1);
  for (int e = threadIdx.x; e < n; e += 256) {
    const int h = e / D, d = e % D;
    float v = x[e];
    if (h < a.Hq + a.Hkv && d < a.rd) {
      const int i = d < half ? d : d - half;
      v = v * cs[i] + (d < half ? -x[e + half] : x[e - half]) * sn[i];
    }
    if (h < a.Hq) {
      if (a.q) a.q[(size_t)blockIdx.x * a.Hq * D + e] = v;
    } else if (page >= 0) {
      const bool is_v = h >= a.Hq + a.Hkv;
      const int hk = h - a.Hq - (is_v ? a.Hkv : 0);
      KT* pool = static_cast<KT*>(is_v ? a.vc : a.kc) + paged_head_at(page, hk, a.Hkv, a.page_shift, D);
      pool[is_v ? paged_v_at(tok, d, D, E) : paged_k_at(tok, d, D, E)] = kv_store<KT>(v);
    }
  }
}

// Eight consecutive dims of a row.
struct Oct {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* x) {
    a = *(const TLM_GLOBAL f32x4u*)(x);
    b = *(const TLM_GLOBAL f32x4u*)(x + 4);
  }
  __device__ __forceinline__ void store(float* x) const {
    *(TLM_GLOBAL f32x4u*)(x) = a;
    *(TLM_GLOBAL f32x4u*)(x + 4) = b;
  }
};
__device__ __forceinline__ f32x4 rotated(f32x4 x, f32x4 partner, f32x4 c, f32x4 s) { return x * c + partner * s; }

// Octs of a head that a thread takes: the first `half / 8` with their partners half
// dims further on, and those past the rotary dims alone.
struct Octs {
  int n, half, rd;
  __device__ __forceinline__ Octs(int D, int rotary) : n((D - rotary) / 8 + rotary / 16), half(rotary / 2), rd(rotary) {}
  __device__ __forceinline__ bool pair(int o) const { return 8 * o < half; }
  __device__ __forceinline__ int dim(int o) const { return pair(o) ? 8 * o : rd + 8 * o - half; }
};

// Dims d .. d + 7 of a token's K: one 16-byte piece of fp16, two of fp32.
template <typename KT>
__device__ __forceinline__ void put_k(KT* head, int tok, int d, int D, const Oct& x) {
  constexpr int E = 16 / sizeof(KT);
  if (E == 8) {
    u32x4 y;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float lo = e < 2 ? x.a[2 * e & 3] : x.b[2 * e & 3], hi = e < 2 ? x.a[(2 * e & 3) + 1] : x.b[(2 * e & 3) + 1];
      y[e] = (uint32_t)kv_store<uint16_t>(lo) | (uint32_t)kv_store<uint16_t>(hi) << 16;
    }
    *(TLM_GLOBAL u32x4*)(head + paged_k_at(tok, d, D, E)) = y;
  } else {
    *(TLM_GLOBAL f32x4*)(head + paged_k_at(tok, d, D, E)) = x.a;
    *(TLM_GLOBAL f32x4*)(head + paged_k_at(tok, d + 4, D, E)) = x.b;
  }
}

// Few rows: a block per row, a thread per oct of a rotated head and per oct of V.
template <typename KT>
__global__ __launch_bounds__(256) void paged_append_row_kernel(PagedArgs a) {
  constexpr int E = 16 / sizeof(KT);
  const int s = blockIdx.x / a.tokens, j = blockIdx.x % a.tokens, D = a.D;
  const Octs oc(D, a.rd);
  const int nrot = (a.Hq + a.Hkv) * oc.n, n = nrot + a.Hkv * (D / 8);
  const float* x = a.x + (size_t)blockIdx.x * (a.Hq + 2 * a.Hkv) * D;
  // the first item's elements are requested before the position is known
  auto fetch = [&](int i, Oct* v) {
    if (i < nrot) {
      const int o = i % oc.n;
      const float* p = x + i / oc.n * D + oc.dim(o);
      v[0].load(p);
      if (oc.pair(o)) v[1].load(p + oc.half);
    } else if (i < n) {
      v[0].load(x + (a.Hq + a.Hkv) * D + 8 * (i - nrot));
    }
  };
  Oct v[2] = {};
  fetch(threadIdx.x, v);
  const int start = a.starts[s];
  bool bad;
  const int rows = paged_rows(start, a.counts ? a.counts[s] : a.tokens, a.tokens, a.limit, &bad);
  if (bad && j == 0 && threadIdx.x == 0) paged_flag(a.status, kPagedStatusRows);
  if (j >= rows) return;
  const int pos = start + j, tok = pos & ((1 << a.page_shift) - 1);
  const int page = paged_page(a.tables + (size_t)s * a.width, pos, a.page_shift, a.num_pages);
  if (page < 0 && threadIdx.x == 0) paged_flag(a.status, kPagedStatusPage);
  for (int i = threadIdx.x; i < n; i += 256) {
    if (i != threadIdx.x) fetch(i, v);
    if (i < nrot) {
      const int h = i / oc.n, o = i % oc.n, d = oc.dim(o);
      if (oc.pair(o)) {
        Oct c, w;
        c.load(a.rope_cos + (size_t)pos * oc.half + d);
        w.load(a.rope_sin + (size_t)pos * oc.half + d);
        const Oct y = v[0];
        v[0].a = rotated(y.a, -v[1].a, c.a, w.a), v[0].b = rotated(y.b, -v[1].b, c.b, w.b);
        v[1].a = rotated(v[1].a, y.a, c.a, w.a), v[1].b = rotated(v[1].b, y.b, c.b, w.b);
      }
      if (h < a.Hq) {
        if (!a.q) continue;
        float* q = a.q + ((size_t)blockIdx.x * a.Hq + h) * D + d;
        v[0].store(q);
        if (oc.pair(o)) v[1].store(q + oc.half);
      } else if (page >= 0) {
        KT* k = static_cast<KT*>(a.kc) + paged_head_at(page, h - a.Hq, a.Hkv, a.page_shift, D);
        put_k<KT>(k, tok, d, D, v[0]);
        if (oc.pair(o)) put_k<KT>(k, tok, d + oc.half, D, v[1]);
      }
    } else if (page >= 0) {
      const int d = 8 * (i - nrot) % D;
      KT* p = static_cast<KT*>(a.vc) + paged_head_at(page, 8 * (i - nrot) / D, a.Hkv, a.page_shift, D);
#pragma unroll
      for (int e = 0; e < 8; e++) p[paged_v_at(tok, d + e, D, E)] = kv_store<KT>(e < 4 ? v[0].a[e & 3] : v[0].b[e & 3]);
    }
  }
}

// Many rows: for each kv head (with its G query heads) and aligned group of 32
// positions, so that V's pieces of 4 or 8 tokens are whole and go out 16 bytes at a
// time.  A thread has one item, `slices` blocks of 256 share the group's:
//   queries: four dims of a token with their partners, head after head (cos and sin
//     are read once for the G heads; a wave covers whole cache lines);
//   K: eight dims with their partners;
//   V: a dim of the E tokens of a piece, 4 q .. 4 q + 3 of each of SUB sixteens.
// Latency and bandwidth: 3548 rows of Llama-3.2-3B (115 MB) 27.1 us, 4.2 TB/s; one
// block for all of a group's items, one after the other, 36.1.
struct AppendItems {
  int q, k, v, slices;
};
__host__ __device__ inline AppendItems append_items(int D, int rd, int E, bool queries) {
  AppendItems n;
  n.q = queries ? 32 * (D / 4 - rd / 8) : 0;
  n.k = 32 * ((D - rd) / 8 + rd / 16);
  n.v = 32 * D / E;
  n.slices = (n.q + n.k + n.v + 255) / 256;
  return n;
}

template <typename KT>
__global__ __launch_bounds__(256) void paged_append_group_kernel(PagedArgs a, int groups) {
  constexpr int E = 16 / sizeof(KT), SUB = E / 4;
  const AppendItems n = append_items(a.D, a.rd, E, a.q != nullptr);
  const int block = blockIdx.x / n.slices, hk = block % a.Hkv, first = block / a.Hkv % groups;
  const int s = block / a.Hkv / groups, D = a.D, half = a.rd / 2;
  int item = blockIdx.x % n.slices * 256 + threadIdx.x;
  const int start = a.starts[s];
  bool bad;
  const int rows = paged_rows(start, a.counts ? a.counts[s] : a.tokens, a.tokens, a.limit, &bad);
  if (bad && first == 0 && hk == 0 && item == 0) paged_flag(a.status, kPagedStatusRows);
  if (rows < 1) return;
  const int p0 = ((start >> 5) + first) << 5, last = start + rows - 1;  // positions p0 .. p0 + 31
  if (p0 > last) return;
  const int page = paged_page(a.tables + (size_t)s * a.width, p0, a.page_shift, a.num_pages);
  if (page < 0 && item == 0) paged_flag(a.status, kPagedStatusPage);
  const int tok0 = p0 & ((1 << a.page_shift) - 1), N = (a.Hq + 2 * a.Hkv) * D;
  const size_t at = paged_head_at(max(page, 0), hk, a.Hkv, a.page_shift, D);
  const size_t row0 = (size_t)s * a.tokens - start;  // + position: the row
  if (item < n.q) {
    const int quads = n.q / 32, f = item % quads, pos = p0 + item / quads, d = 4 * f < half ? 4 * f : 4 * f + half;
    if (pos < start || pos > last) return;
    const bool pair = d < half;
    const float* x = a.x + (row0 + pos) * N + (size_t)hk * a.G * D + d;
    float* q = a.q + ((row0 + pos) * a.Hq + hk * a.G) * D + d;
    f32x4 c = {1.f, 1.f, 1.f, 1.f}, w = {0.f, 0.f, 0.f, 0.f};
    if (pair) {
      c = *(const TLM_GLOBAL f32x4*)(a.rope_cos + (size_t)pos * half + d);
      w = *(const TLM_GLOBAL f32x4*)(a.rope_sin + (size_t)pos * half + d);
    }
    const int to = pair ? half : 0;
    f32x4 lo = *(const TLM_GLOBAL f32x4u*)(x), hi = *(const TLM_GLOBAL f32x4u*)(x + to);
    for (int g = 0; g < a.G; g++) {
      const float* y = x + (size_t)min(g + 1, a.G - 1) * D;  // the next head's, in flight meanwhile
      const f32x4 nlo = *(const TLM_GLOBAL f32x4u*)(y), nhi = *(const TLM_GLOBAL f32x4u*)(y + to);
      *(TLM_GLOBAL f32x4u*)(q + g * D) = pair ? rotated(lo, -hi, c, w) : lo;
      if (pair) *(TLM_GLOBAL f32x4u*)(q + g * D + half) = rotated(hi, lo, c, w);
      lo = nlo, hi = nhi;
    }
    return;
  }
  if (page < 0) return;
  item -= n.q;
  if (item < n.k) {
    KT* const k = static_cast<KT*>(a.kc) + at;
    const Octs oc(D, a.rd);
    const int o = item % oc.n, t = item / oc.n, pos = p0 + t, d = oc.dim(o);
    if (pos < start || pos > last) return;
    const float* x = a.x + (row0 + pos) * N + (a.Hq + hk) * D + d;
    Oct lo;
    lo.load(x);
    if (oc.pair(o)) {
      Oct c, w, hi, y;
      hi.load(x + half);
      c.load(a.rope_cos + (size_t)pos * half + d);
      w.load(a.rope_sin + (size_t)pos * half + d);
      y.a = rotated(hi.a, lo.a, c.a, w.a), y.b = rotated(hi.b, lo.b, c.b, w.b);
      lo.a = rotated(lo.a, -hi.a, c.a, w.a), lo.b = rotated(lo.b, -hi.b, c.b, w.b);
      put_k<KT>(k, tok0 + t, d + half, D, y);
    }
    put_k<KT>(k, tok0 + t, d, D, lo);
    return;
  }
  item -= n.k;
  if (item >= n.v) return;
  const int d = item % D, t = item / D % 4 * 4 + item / D / 4 * 16;
  const float* x = a.x + (row0 + p0) * N + (a.Hq + a.Hkv + hk) * D + d;
  float v[E];
  bool all = true;
#pragma unroll
  for (int e = 0; e < E; e++) {
    const int u = t + 16 * (e / 4) + (e & 3);
    const bool in = p0 + u >= start && p0 + u <= last;
    all &= in;
    v[e] = in ? x[(size_t)u * N] : 0.f;
  }
  KT* const p = static_cast<KT*>(a.vc) + at + paged_v_at(tok0 + t, d, D, E);
  if (all) {
    u32x4 y;
#pragma unroll
    for (int e = 0; e < 4; e++)
      y[e] = SUB == 2 ? (uint32_t)kv_store<uint16_t>(v[2 * e % E]) | (uint32_t)kv_store<uint16_t>(v[(2 * e + 1) % E]) << 16
                      : __float_as_uint(v[e]);
    *(TLM_GLOBAL u32x4*)(p) = y;
  } else {
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int u = p0 + t + 16 * (e / 4) + (e & 3);
      if (u >= start && u <= last) p[e] = kv_store<KT>(v[e]);
    }
  }
}

typedef _Float16 ph8_t __attribute__((ext_vector_type(8)));
// Attention of the rows of a step.  A kv head's rows r = j G + g (token j, head g
// of its group) are the columns of 16-column matrix-core tiles, so that K and V are
// read once for 16 of them; a block has one column tile (a unit is a kv head and a
// row group).  Several tiles a block were slower everywhere, as their outputs leave
// room for fewer waves (16 x 16 Llama-3.2-3B up to 2000 positions 31.9 us with four, 22.1 so;
// Qwen2.5-0.5B 16 x 5 20.5 and 10.2; a 2048-token prompt of Llama-3.2-1B 112 and 65).  The W
// waves take the position tiles of one chunk of the sequence in turn:
//   * scores S^T (positions x rows) = K Q^T, K the A operand, q the B operand;
//   * softmax with a running maximum and sum per row, base 2.  The maximum is a whole
//     number at or above the scores, so that rescaling is exact and a weight takes one
//     fma before its exponential;
//   * O^T (dims x rows) += V^T P^T, V^T the A operand, P^T from the score registers.
// The pages hold K and V in operand order (tlm_paged.h), so a tile's operands are
// loaded straight into registers, 1 KB in a row per wave and instruction.
// fp16 caches: 32 positions a tile, v_mfma_f32_16x16x32_f16 with q and P as hi +
// lo pairs (K and V are exact): an element of q to 2^-22 of itself or 2^-39 of the
// row's largest, P to 2^-22 of itself or 2^-39 of the largest.  That takes both times
// 2^15, the largest power of two in fp16's range: as numbers up to 1 they end at
// 2^-25, and many small weights beside one large are lost while the sum has them.  q's
// factor is taken out of the scores, P's is in L and O alike.
// fp32 caches: 16 positions a tile, v_mfma_f32_16x16x4_f32.
template <typename KT>
struct PagedTile {
  static constexpr int SUB = 4 / sizeof(KT);  // 16-position score tiles
  static constexpr int TS = 16 * SUB;         // positions
  static constexpr int SHIFT = SUB == 2 ? 5 : 4;
  static constexpr float kLift = SUB == 2 ? 15.f : 0.f;  // log2 of q's and P's factor
};

// A sequence's part in a call: its rows and the position tiles that they attend to.
struct SeqWork {
  int start, rows, first, tiles;
};
template <int SHIFT>
__device__ __forceinline__ SeqWork seq_work(const PagedArgs& a, int s, bool* bad) {
  SeqWork w;
  w.start = a.starts[s];
  w.rows = paged_rows(w.start, a.counts ? a.counts[s] : a.tokens, a.tokens, a.limit, bad);
  const int first = a.window > 0 ? max(0, w.start - a.window + 1) : 0;
  w.first = first >> SHIFT;
  w.tiles = w.rows > 0 ? ((w.start + w.rows - 1) >> SHIFT) - w.first + 1 : 0;
  return w;
}

// Values that another block of the same launch reads: past the XCD's L2.
__device__ __forceinline__ void publish2(float* p, float x, float y) {
  const unsigned long long v = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 published2(const float* p) {
  const unsigned long long v = __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32)));
}

// Sum over the wave's lanes up to each, over integers.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1, within 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// Chunks of equal size over sequences of unequal length, c tiles each: all
// sequences together have at most a.chunks more of them than sequences.  Up to
// kPlanInPlace sequences every wave works it out for itself from the starts (which
// only the device knows): the sum of the tiles, then a running sum of the sequences'
// chunks up to chunk g.  Its time grows with the sequences in each of a number of
// blocks that does, too; past that a launch of one block leaves c and the running
// sums before each 64 sequences, which a wave searches.  us a call in place / so, one
// token each at 300 positions of Llama-3.2-1B: 300 sequences 35.0 / 35.8, 512 64.8 / 59.2,
// 1024 160 / 114, 2048 416 / 228.
// slot: records of partial results before the sequence's (one of a single chunk has
// none).  False: there is no chunk g.
constexpr int kPlanInPlace = 384;
constexpr int kPlanThreads = 1024;
struct SeqChunk {
  SeqWork w;
  int s, n, chunk, slot;  // sequence, its chunks, which of them
};
// a.plan: c, then the chunks and the slots before each 64 sequences
__host__ __device__ inline int plan_groups(int seqs) { return (seqs + 63) / 64; }
__device__ __forceinline__ int plan_part(const PagedArgs& a, int tiles) {  // their sum stays in 31 bits
  return (tiles + (1 << a.plan_shift) - 1) >> a.plan_shift;
}
__device__ __forceinline__ int plan_chunk(const PagedArgs& a, int total) {
  return max(a.chunk_min, ((total + a.chunks - 1) / a.chunks) << a.plan_shift);
}
__device__ __forceinline__ int plan_chunks_of(const PagedArgs& a, int c, int tiles) {
  return tiles <= a.whole ? min(tiles, 1) : (tiles + c - 1) / c;
}

template <int SHIFT>
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedArgs a) {
  constexpr int W = kPlanThreads / 64;
  __shared__ int sh[2][W];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = plan_groups(a.seqs);
  bool any = false, bad;
  int sum = 0;
  for (int s = tid; s < a.seqs; s += kPlanThreads) {
    sum += plan_part(a, seq_work<SHIFT>(a, s, &bad).tiles);
    any |= bad;
  }
  if (any) paged_flag(a.status, kPagedStatusRows);
  sum = __builtin_amdgcn_readlane(wave_scan(sum), 63);
  if (lane == 0) sh[0][w] = sum;
  __syncthreads();
  int total = 0;
  for (int i = 0; i < W; i++) total += sh[0][i];
  const int c = plan_chunk(a, total);
  if (tid == 0) a.plan[0] = c;
  int before = 0, slots = 0;
  for (int g0 = 0; g0 < groups; g0 += W) {  // a wave per 64 sequences
    const int s = 64 * (g0 + w) + lane;
    const int n = s < a.seqs ? plan_chunks_of(a, c, seq_work<SHIFT>(a, s, &bad).tiles) : 0;
    const int chunks = __builtin_amdgcn_readlane(wave_scan(n), 63);
    const int parts = __builtin_amdgcn_readlane(wave_scan(n > 1 ? n : 0), 63);
    __syncthreads();  // sh of the round before has been read
    if (lane == 0) sh[0][w] = chunks, sh[1][w] = parts;
    __syncthreads();
    for (int i = 0; i < W; i++) {
      if (i == w && lane == 0 && g0 + w < groups) {
        a.plan[1 + g0 + w] = before;
        a.plan[1 + groups + g0 + w] = slots;
      }
      before += sh[0][i];
      slots += sh[1][i];
    }
  }
}

template <int SHIFT>
__device__ __forceinline__ bool plan(const PagedArgs& a, int g, SeqChunk& r) {
  const int lane = threadIdx.x & 63;
  const SeqWork none{0, 0, 0, 0};
  bool b;
  int c = 0, before = 0, slots = 0;
  // whether chunk g is one of the 64 sequences' from s0 on, a lane each
  auto find = [&](const SeqWork& w, int s0) {
    const int n = plan_chunks_of(a, c, w.tiles), incl = wave_scan(n), m = n > 1 ? n : 0, sincl = wave_scan(m);
    const unsigned long long hit = __ballot(before + incl > g);
    if (!hit) {
      before += __builtin_amdgcn_readlane(incl, 63);
      slots += __builtin_amdgcn_readlane(sincl, 63);
      return false;
    }
    const int l = __builtin_ctzll(hit);
    r.s = s0 + l;
    r.w.start = __builtin_amdgcn_readlane(w.start, l);
    r.w.rows = __builtin_amdgcn_readlane(w.rows, l);
    r.w.first = __builtin_amdgcn_readlane(w.first, l);
    r.w.tiles = __builtin_amdgcn_readlane(w.tiles, l);
    r.n = __builtin_amdgcn_readlane(n, l);
    r.chunk = g - before - __builtin_amdgcn_readlane(incl - n, l);
    r.slot = slots + __builtin_amdgcn_readlane(sincl - m, l);
    return true;
  };
  if (a.plan) {
    // the last 64 sequences before which there are at most g chunks, by 64 at a time
    const int groups = plan_groups(a.seqs);
    int lo = 0, len = groups;
    while (true) {
      const int step = (len + 63) / 64, i = lane * step;
      const int k = __builtin_popcountll(__ballot(i < len && a.plan[1 + lo + min(i, len - 1)] <= g)) - 1;  // the first is
      lo += k * step;
      len = min(step, len - k * step);
      if (step == 1) break;
    }
    c = a.plan[0], before = a.plan[1 + lo], slots = a.plan[1 + groups + lo];
    const int s0 = 64 * lo;
    return find(s0 + lane < a.seqs ? seq_work<SHIFT>(a, s0 + lane, &b) : none, s0);
  }
  // the first kSeqs times 64 sequences stay in registers, a lane each
  constexpr int kSeqs = 4;
  SeqWork w[kSeqs];
  bool bad[kSeqs];
  int sum = 0;
#pragma unroll
  for (int k = 0; k < kSeqs; k++) {
    w[k] = none, bad[k] = false;
    if (64 * k < a.seqs && 64 * k + lane < a.seqs) w[k] = seq_work<SHIFT>(a, 64 * k + lane, &bad[k]);
  }
#pragma unroll
  for (int k = 0; k < kSeqs; k++) sum += plan_part(a, w[k].tiles);
  bool any = bad[0] || bad[1] || bad[2] || bad[3];
  for (int s = 64 * kSeqs + lane; s < a.seqs; s += 64) {
    sum += plan_part(a, seq_work<SHIFT>(a, s, &b).tiles);
    any |= b;
  }
  if (any && blockIdx.x == 0 && threadIdx.x < 64) paged_flag(a.status, kPagedStatusRows);
  c = plan_chunk(a, __builtin_amdgcn_readlane(wave_scan(sum), 63));
  if (a.seqs <= 64) {
    // few sequences: all their chunks in one round of blocks
    const int live = __builtin_popcountll(__ballot(w[0].tiles > 0));
    if (2 * live <= a.round)
      while (__builtin_amdgcn_readlane(wave_scan(plan_chunks_of(a, c, w[0].tiles)), 63) > a.round) c += (c + 7) / 8;
  }
#pragma unroll
  for (int k = 0; k < kSeqs; k++)
    if (64 * k < a.seqs && find(w[k], 64 * k)) return true;
  for (int s0 = 64 * kSeqs; s0 < a.seqs; s0 += 64) {
    const SeqWork v = s0 + lane < a.seqs ? seq_work<SHIFT>(a, s0 + lane, &b) : none;
    if (find(v, s0)) return true;
  }
  return false;
}

// Partial results: per slot, unit (kv head and row group) and row of its 16 the
// unscaled output, then the maximum in base 2 and the sum.
__device__ __forceinline__ float* part_row(const PagedArgs& a, int slot, int unit, int row, int DT) {
  return a.part + (((size_t)slot * a.units + unit) * 16 + row) * (DT + 2);
}

template <typename KT, int DT, int W, bool STREAM>
__global__ __launch_bounds__(64 * W, DT <= 64 ? 4 : 2) void paged_attention_kernel(PagedArgs a) {
  using T = PagedTile<KT>;
  constexpr int SUB = T::SUB, TS = T::TS, NF = DT / 16;  // 1 KB operand pieces of a tile's K, of its V
  constexpr bool F16 = sizeof(KT) == 2;
  constexpr int RS = DT + 2;  // floats of a row's record: maximum, sum, output
  constexpr int LDSF = W * 16 * RS;
  __shared__ __align__(16) float lds[LDSF];
  // the row groups from the last one on: a prompt's last rows attend to the most
  const int unit = blockIdx.x % a.units, hk = unit % a.Hkv, r0 = (a.units - 1 - unit) / a.Hkv * 16;
  const int g = blockIdx.x / a.units;
  SeqChunk sc;
  if (!plan<T::SHIFT>(a, g, sc)) return;
  const int ci = sc.chunk, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = sc.w.rows * a.G;  // rows of the kv head
  if (r0 >= R) return;
  const int i16 = lane & 15, qd = lane >> 4;
  // positions that some row of the block attends to, and that all do
  const int ja = r0 / a.G, jb = (min(r0 + 16, R) - 1) / a.G, start = sc.w.start;
  const int lo_any = a.window > 0 ? max(0, start + ja - a.window + 1) : 0, hi_any = start + jb;
  const int lo_all = a.window > 0 ? max(0, start + jb - a.window + 1) : 0, hi_all = start + ja;
  const int per = (sc.w.tiles + sc.n - 1) / sc.n;
  const int t0 = max(sc.w.first + ci * per, lo_any >> T::SHIFT);
  const int t1 = min(min(sc.w.first + (ci + 1) * per, sc.w.first + sc.w.tiles), (hi_any >> T::SHIFT) + 1);
  const int32_t* const table = a.tables + (size_t)sc.s * a.width;
  const int tpp = a.page_shift - T::SHIFT;  // log2 of the tiles of a page

  struct Tile {
    u32x4 k[NF], v[NF];
  };
  auto load = [&](u32x4* x, const void* pool, int t, int page) {
    const size_t at = paged_head_at(max(page, 0), hk, a.Hkv, a.page_shift, DT) +
                      (size_t)(t & ((1 << tpp) - 1)) * (TS * DT) + lane * (16 / sizeof(KT));
    const TLM_GLOBAL u32x4* p = gl(reinterpret_cast<const u32x4*>(static_cast<const KT*>(pool) + at));
#pragma unroll
    for (int f = 0; f < NF; f++) x[f] = STREAM ? __builtin_nontemporal_load(p + 64 * f) : p[64 * f];
  };
  // The wave's tiles t0 + w, t0 + w + W, ...  Their pages, 64 at a time, a lane each;
  // the first tile is on its way while q is prepared.
  int tb = t0 + w, n = 0, page = -1;
  auto pages = [&] {
    const int tl = tb + lane * W;
    n = min(64, (t1 - tb + W - 1) / W);
    page = paged_page(table, min(tl, t1 - 1) << T::SHIFT, a.page_shift, a.num_pages);
    if (page < 0 && tl < t1) paged_flag(a.status, kPagedStatusPage);
  };
  auto page_of = [&](int i) { return __builtin_amdgcn_readlane(page, i); };
  auto load_k = [&](Tile& x, int i) { load(x.k, a.kc, tb + i * W, page_of(i)); };
  auto load_v = [&](Tile& x, int i) { load(x.v, a.vc, tb + i * W, page_of(i)); };
  // This lane's row (its column of the tiles): its positions' bounds, and q scaled by
  // a power of two to at most 1, or 2^15 as fp16.  q is requested before the first
  // tile: loads return in order.
  const int row = r0 + i16, rc = min(row, R - 1), hi = start + rc / a.G;
  const int lo = a.window > 0 ? hi - a.window + 1 : 0;
  u32x4 qreg[NF];
  f32x4 qx[NF];
  const float* const q = a.x + (((size_t)sc.s * a.tokens + rc / a.G) * a.Hq + hk * a.G + rc % a.G) * DT;
#pragma unroll
  for (int f = 0; f < NF; f++)  // fp16: dims 32 (f / 2) + 8 qd + 4 (f % 2) ..; fp32: 16 f + 4 qd ..
    qx[f] = *(const TLM_GLOBAL f32x4u*)(q + (F16 ? 32 * (f / 2) + 8 * qd + 4 * (f & 1) : 16 * f + 4 * qd));
  __builtin_amdgcn_sched_barrier(0);
  Tile x;
  if (tb < t1) {
    pages();
    load_k(x, 0);
    load_v(x, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
  float qmax = 0.f;
#pragma unroll
  for (int f = 0; f < NF; f++)
#pragma unroll
    for (int e = 0; e < 4; e++) qmax = fmaxf(qmax, fabsf(qx[f][e]));
  qmax = fmaxf(qmax, lane_swap16(qmax));
  qmax = fmaxf(qmax, lane_swap32(qmax));
  const int qe = __builtin_amdgcn_frexp_expf(qmax);
  const int ex = F16 ? max(-100, qe - (int)T::kLift) : max(-120, min(120, qe));
#pragma unroll
  for (int f = 0; f < NF; f++)
#pragma unroll
    for (int e = 0; e < 4; e++) qx[f][e] = row < R ? ldexpf(qx[f][e], -ex) : 0.f;
  // log2 e: the softmax runs in base 2; above 0, as masked scores are -inf before it
  const float mult = fmaxf(ldexpf(a.scale * 1.4426950408889634f, ex), FLT_TRUE_MIN);
#pragma unroll
  for (int f = 0; f < NF; f++) {
    if (!F16) {
      qreg[f] = __builtin_bit_cast(u32x4, qx[f]);
    } else if (f % 2 == 0) {  // dims of one slab of 32: the high parts, then the low ones
      ph8_t h, l;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const float v = qx[f + e / 4][e & 3];
        h[e] = (_Float16)v;
        l[e] = (_Float16)(v - (float)h[e]);
      }
      qreg[f] = __builtin_bit_cast(u32x4, h);
      qreg[f + 1] = __builtin_bit_cast(u32x4, l);
    }
  }

  f32x4 o[NF];
  float mrun = -FLT_MAX, lrun = 0.f;  // running maximum, this lane's share of the sum
#pragma unroll
  for (int f = 0; f < NF; f++) o[f] = (f32x4){0.f, 0.f, 0.f, 0.f};

  // V with positions outside [first, last] taken out (0 times what they hold may be NaN)
  auto keep = [&](const u32x4& v, int p, int first, int last) {
    u32x4 y;
#pragma unroll
    for (int d = 0; d < 4; d++) {
      if (F16) {  // dword d: positions 16 (d / 2) + 4 qd + 2 (d % 2) + {0, 1}
        const int x = p + 16 * (d / 2) + 4 * qd + 2 * (d & 1);
        y[d] = v[d] & ((x >= first && x <= last ? 0xFFFFu : 0u) | (x + 1 >= first && x + 1 <= last ? 0xFFFF0000u : 0u));
      } else {
        const int x = p + 4 * qd + d;
        y[d] = x >= first && x <= last ? v[d] : 0u;
      }
    }
    return y;
  };
  auto not_finite = [](unsigned v) -> unsigned {  // the sign bits' places of values that are not finite
    return F16 ? ((v & 0x7C007C00u) + 0x04000400u) & 0x80008000u : ((v & 0x7F800000u) + 0x00800000u) & 0x80000000u;
  };
  // tile t; k_read() and v_read() run once x.k and x.v have been read
  auto process = [&](Tile& x, int t, auto k_read, auto v_read) {
    const int p = t << T::SHIFT;
    const bool edge = p < lo_all || p + TS - 1 > hi_all;  // some row does not see all of it (wave-uniform)
    bool apart = false;
    if (edge) {
      // only a value that is not finite could reach a row that masks its position
      unsigned nf = 0;
#pragma unroll
      for (int f = 0; f < NF; f++) {
        x.v[f] = keep(x.v[f], p, lo_any, hi_any);
#pragma unroll
        for (int d = 0; d < 4; d++) nf |= not_finite(x.v[f][d]);
      }
      apart = ja != jb && __ballot(nf != 0) != 0;
    }
    f32x4 acc[2] = {(f32x4){0.f, 0.f, 0.f, 0.f}, (f32x4){0.f, 0.f, 0.f, 0.f}};
    if (F16) {
#pragma unroll
      for (int jj = 0; jj < NF / 2; jj++) {
        const ph8_t qh = __builtin_bit_cast(ph8_t, qreg[2 * jj]), ql = __builtin_bit_cast(ph8_t, qreg[2 * jj + 1]);
#pragma unroll
        for (int st = 0; st < SUB; st++) {
          const ph8_t k = __builtin_bit_cast(ph8_t, x.k[st * (NF / SUB) + jj]);
          acc[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh, acc[st], 0, 0, 0);
          acc[st] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql, acc[st], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; f++) {
        const f32x4 qf = __builtin_bit_cast(f32x4, qreg[f]), k = __builtin_bit_cast(f32x4, x.k[f]);
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], qf[e], acc[e & 1], 0, 0, 0);
      }
      acc[0] += acc[1];
    }
    // lane (row i16, qd): positions p + 16 st + 4 qd + e
    float sv[4 * SUB];
#pragma unroll
    for (int st = 0; st < SUB; st++)
#pragma unroll
      for (int e = 0; e < 4; e++) sv[4 * st + e] = acc[st][e];
    if (edge) {
#pragma unroll
      for (int i = 0; i < 4 * SUB; i++) {
        const int y = p + 16 * (i / 4) + 4 * qd + (i & 3);
        if (y < lo || y > hi) sv[i] = -INFINITY;
      }
    }
    float mx = sv[0];
#pragma unroll
    for (int i = 1; i < 4 * SUB; i++) mx = fmaxf(mx, sv[i]);
    mx = fmaxf(mx, lane_swap16(mx));
    mx = fmaxf(mx, lane_swap32(mx));
    const float mn = fmaxf(mrun, ceilf(mx * mult));  // finite: it starts at -FLT_MAX
    if (__ballot(fabsf(mn) >= 0x1p22f)) {
      // kLift - mn is rounded there, and an unrounded product passes the maximum by as much
#pragma clang fp contract(off)
#pragma unroll
      for (int i = 0; i < 4 * SUB; i++) sv[i] = (sv[i] * mult - mn) + T::kLift;
    } else {
      const float lift = T::kLift - mn;
#pragma unroll
      for (int i = 0; i < 4 * SUB; i++) sv[i] = fmaf(sv[i], mult, lift);
    }
    const float corr = __builtin_amdgcn_exp2f(mrun - mn);
    float ps = 0.f;
    u32x4 ph, pl;  // fp16: high and low parts
    if (F16) {
      ph8_t h, l;
#pragma unroll
      for (int i = 0; i < 4 * SUB; i++) {
        const float v = __builtin_amdgcn_exp2f(sv[i]);
        ps += v;
        h[i % 8] = (_Float16)v;
        l[i % 8] = (_Float16)(v - (float)h[i % 8]);
      }
      ph = __builtin_bit_cast(u32x4, h);
      pl = __builtin_bit_cast(u32x4, l);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float v = __builtin_amdgcn_exp2f(sv[i]);
        ps += v;
        ph[i] = __float_as_uint(v);
      }
    }
    lrun = fmaf(lrun, corr, ps);
    mrun = mn;
    if (__ballot(corr != 1.f)) {
#pragma unroll
      for (int f = 0; f < NF; f++) o[f] *= corr;
    }
    k_read();
    auto weigh = [&](const u32x4& v, f32x4 y) -> f32x4 {
      if (F16) {
        const ph8_t vh = __builtin_bit_cast(ph8_t, v);
        y = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, __builtin_bit_cast(ph8_t, ph), y, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(vh, __builtin_bit_cast(ph8_t, pl), y, 0, 0, 0);
      }
      const f32x4 vf = __builtin_bit_cast(f32x4, v), pf = __builtin_bit_cast(f32x4, ph);
#pragma unroll
      for (int e = 0; e < 4; e++) y = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[e], pf[e], y, 0, 0, 0);
      return y;
    };
    if (apart) {
      // a row that does give such a value a weight becomes NaN there; the others get 0
      // times 0
#pragma unroll
      for (int f = 0; f < NF; f++) {
        u32x4 one;
#pragma unroll
        for (int d = 0; d < 4; d++) {
          const unsigned t = not_finite(x.v[f][d]);  // a bit per value, its highest
          one[d] = F16 ? (t >> 15) * 0x3C00u : (t >> 31) * 0x3F800000u;
          x.v[f][d] &= ~(F16 ? (t >> 15) * 0xFFFFu : (t >> 31) * 0xFFFFFFFFu);
        }
        const f32x4 y = weigh(one, (f32x4){0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (y[e] > 0.f) o[f][e] = __uint_as_float(0x7FC00000u);
      }
    }
#pragma unroll
    for (int f = 0; f < NF; f++) o[f] = weigh(x.v[f], o[f]);
    v_read();
  };

  // The next tile's K goes out when this one's has been read, its V likewise: half a
  // tile or more in flight a wave, and the registers of one (with two, 8 waves a CU
  // instead of 16 at head_dim 64 and less in flight: 128 x 1 Llama-3.2-1B up to
  // 1000 positions 31.8 instead of 28.1 us).
  while (tb < t1) {
    for (int i = 0; i < n; i++) {
      const bool more = i + 1 < n;
      if (page_of(i) >= 0) {
        process(x, tb + i * W, [&] { if (more) load_k(x, i + 1); }, [&] { if (more) load_v(x, i + 1); });
      } else if (more) {
        load_k(x, i + 1);
        load_v(x, i + 1);
      }
    }
    tb += 64 * W;
    if (tb < t1) {
      pages();
      load_k(x, 0);
      load_v(x, 0);
    }
  }

  // the waves' results joined through LDS
  const bool whole = sc.n == 1;
  auto put = [&](int r, int d, float y0, float y1) {  // dims d and d + 1 of row r
    const size_t at = (((size_t)sc.s * a.tokens + r / a.G) * a.Hq + hk * a.G + r % a.G) * DT + d;
    if (a.out_f32) {
      static_cast<float*>(a.out)[at] = y0;
      static_cast<float*>(a.out)[at + 1] = y1;
    } else {
      static_cast<uint16_t*>(a.out)[at] = kv_store<uint16_t>(y0);
      static_cast<uint16_t*>(a.out)[at + 1] = kv_store<uint16_t>(y1);
    }
  };
  lrun += lane_swap16(lrun);
  lrun += lane_swap32(lrun);
  float* const rec = lds + (w * 16 + i16) * RS;
#pragma unroll
  for (int f = 0; f < NF; f++)
#pragma unroll
    for (int e = 0; e < 4; e++) rec[2 + 16 * f + 4 * qd + e] = o[f][e];
  if (qd == 0) rec[0] = mrun, rec[1] = lrun;
  __syncthreads();
  const int rows = min(16, R - r0);
  for (int e = tid; e < rows * (DT / 2); e += 64 * W) {
    const int i = e / (DT / 2), d = 2 * (e % (DT / 2));
    float M = -FLT_MAX, L = 0.f, O0 = 0.f, O1 = 0.f;
#pragma unroll
    for (int x = 0; x < W; x++) M = fmaxf(M, lds[(x * 16 + i) * RS]);
#pragma unroll
    for (int x = 0; x < W; x++) {
      const float* y = lds + (x * 16 + i) * RS;
      const float f = __builtin_amdgcn_exp2f(y[0] - M);
      L = fmaf(y[1], f, L);
      O0 = fmaf(y[2 + d], f, O0);
      O1 = fmaf(y[3 + d], f, O1);
    }
    if (whole) {
      put(r0 + i, d, L == 0.f ? 0.f : O0 / L, L == 0.f ? 0.f : O1 / L);  // 0: no position has a page
    } else {
      float* p = part_row(a, sc.slot + ci, unit, i, DT);
      publish2(p + d, O0, O1);
      if (d == 0) publish2(p + DT, M, L);
    }
  }
  if (whole) return;

  // The last of the sequence's blocks joins the chunks: it counts last, when every
  // block's results have been performed, and clears the count.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's results are performed
  __syncthreads();                                  // and every wave's
  unsigned* const count = a.arrived + (size_t)sc.slot * a.units + unit;
  if (tid == 0) lds[0] = __uint_as_float(__hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  __syncthreads();
  if (__float_as_uint(lds[0]) != (unsigned)sc.n - 1) return;
  __syncthreads();  // lds[0] has been read
  if (tid == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // A thread per row and four dims, the chunks in `groups` where there are threads for
  // it; four chunks' values in flight at a time.
  constexpr int TH = 64 * W, P = DT / 4;
  const int items = rows * P, groups = max(1, min(TH, LDSF / 6) / items);
  const size_t step = (size_t)a.units * 16 * RS;
  for (int i0 = 0; i0 < items; i0 += TH) {
    const int i = groups > 1 ? tid % items : i0 + tid, grp = groups > 1 ? tid / items : 0;
    const bool here = i < items && grp < groups;
    float M = -FLT_MAX, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    const float* from = part_row(a, sc.slot, unit, min(i, items - 1) / P, DT);
    for (int c0 = grp; here && c0 < sc.n; c0 += 4 * groups) {
      float2 v[4], u[4], ml[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float* p = from + min(c0 + k * groups, sc.n - 1) * step;
        v[k] = published2(p + 4 * (i % P));
        u[k] = published2(p + 4 * (i % P) + 2);
        ml[k] = published2(p + DT);
      }
      const float m = fmaxf(fmaxf(fmaxf(M, ml[0].x), fmaxf(ml[1].x, ml[2].x)), ml[3].x);
      const float f = __builtin_amdgcn_exp2f(M - m);
      L *= f;
      O *= f;
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const float h = c0 + k * groups < sc.n ? __builtin_amdgcn_exp2f(ml[k].x - m) : 0.f;
        L = fmaf(ml[k].y, h, L);
        O[0] = fmaf(v[k].x, h, O[0]);
        O[1] = fmaf(v[k].y, h, O[1]);
        O[2] = fmaf(u[k].x, h, O[2]);
        O[3] = fmaf(u[k].y, h, O[3]);
      }
      M = m;
    }
    if (groups > 1) {
      if (here) {
        float* const mine = lds + 6 * tid;
        mine[0] = M, mine[1] = L;
#pragma unroll
        for (int e = 0; e < 4; e++) mine[2 + e] = O[e];
      }
      __syncthreads();
      for (int x = 1; x < groups && tid < items; x++) {
        const float* y = lds + 6 * (tid + x * items);
        const float m = fmaxf(M, y[0]), f = __builtin_amdgcn_exp2f(M - m), h = __builtin_amdgcn_exp2f(y[0] - m);
        L = L * f + y[1] * h;
#pragma unroll
        for (int e = 0; e < 4; e++) O[e] = O[e] * f + y[2 + e] * h;
        M = m;
      }
    }
    if (here && grp == 0) {
      const float d = L == 0.f ? 0.f : 1.f / L;
      put(r0 + i / P, 4 * (i % P), O[0] * d, O[1] * d);
      put(r0 + i / P, 4 * (i % P) + 2, O[2] * d, O[3] * d);
    }
  }
}

template <typename KT, int DT, int W, bool STREAM>
void launch_attention_of(PagedArgs a, int cus, size_t part_floats, hipStream_t st) {
  using T = PagedTile<KT>;
  // tiles that a sequence may have, as far as the host knows
  int64_t most = a.limit;
  if (a.window > 0) most = std::min<int64_t>(most, (int64_t)a.window + a.tokens);
  const int64_t tiles = most / T::TS + 2;
  a.plan_shift = 0;
  while (a.seqs * ((tiles >> a.plan_shift) + 1) >= ((int64_t)1 << 30)) a.plan_shift++;
  // Sequences of two chunks or more have 2 * chunks at most, each a record and a count.
  // A split costs about 3.5 us (counting, joining), a round of the waves' tiles 0.8: up to
  // 32 tiles a sequence stays whole, and chunks have 16 at least.
  const int64_t record = 16 * (DT + 2);
  a.plan = nullptr;
  if (a.seqs > kPlanInPlace) {  // the plan lies before the records
    const size_t ints = (2 * plan_groups(a.seqs) + 1 + 3) & ~3;
    a.plan = reinterpret_cast<int*>(a.part);
    a.part += ints;
    part_floats -= ints;
  }
  const int64_t fit = std::min<int64_t>((int64_t)part_floats / (2 * a.units * record), kPagedCounters / (2 * a.units));
  a.round = std::max(1, 8 / W * cus / a.units);
  a.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(fit, a.round));
  a.chunk_min = fit < 1 ? INT_MAX / 2 : 16;
  a.whole = 32;
  const int64_t per_seq = fit < 1 || tiles <= a.whole ? 1 : (tiles + a.chunk_min - 1) / a.chunk_min;
  const int64_t blocks = std::min<int64_t>(a.chunks + a.seqs, a.seqs * per_seq) * a.units;
  if (a.plan) hipLaunchKernelGGL((paged_plan_kernel<T::SHIFT>), dim3(1), dim3(kPlanThreads), 0, st, a);
  hipLaunchKernelGGL((paged_attention_kernel<KT, DT, W, STREAM>), dim3((unsigned)blocks), dim3(64 * W), 0, st, a);
}

// Waves a block: four where the sequences' kv heads and row groups alone give a
// block a CU (a short sequence then leaves no waves idle), else eight.  us a call over
// four sets of inputs in turn, sequences of a 16th of the positions named to all of
// them, 8 / 4 waves: 128 x 1 Llama-3.2-1B up to 1000 positions 26.6 / 25.0, 256 x 1 45.6 /
// 41.3, 64 x 1 Llama-3.2-3B 30.0 / 28.6, 16 x 8 up to 2000 20.8 / 18.8; 16 x 5 up to 2500 17.5 /
// 21.9, Qwen2.5-0.5B 1 x 1 at 300 5.6 / 6.4, 16 x 5 up to 2000 10.2 / 11.7.
// Past the last-level cache (256 MB), streaming loads where K and V may exceed it and
// are read once, as nothing of them is still there for the next call: 256 x 1
// Llama-3.2-1B up to 1000 41.3 -> 36.1, 64 x 1 up to 8192 77.9 -> 71.1; what fits it is faster
// kept (64 x 1 up to 1000 13.6, streaming 15.6).
template <typename KT, int DT>
void launch_attention_rows(PagedArgs a, int cus, size_t part_floats, hipStream_t st) {
  const int groups = (a.tokens * a.G + 15) / 16;
  a.units = a.Hkv * groups;
  const int64_t held = std::min<int64_t>(a.limit, a.window > 0 ? (int64_t)a.window + a.tokens : INT_MAX);
  if ((int64_t)a.seqs * a.units < cus)
    launch_attention_of<KT, DT, 8, false>(a, cus, part_floats, st);
  else if (groups > 1 || a.seqs * held * 2 * a.Hkv * DT * (int64_t)sizeof(KT) <= (int64_t)256 << 20)
    launch_attention_of<KT, DT, 4, false>(a, cus, part_floats, st);
  else
    launch_attention_of<KT, DT, 4, true>(a, cus, part_floats, st);
}

}  // namespace

// The row kernel starts one block a row and writes V two bytes at a time; the group
// kernel starts blocks for the positions of whole groups that a sequence may touch.
// us a call, row / group, 64 sequences of 4, 8, 12 and 16 tokens: Llama-3.2-1B heads 4.1 /
// 7.4, 6.0 / 8.0, 7.4 / 8.6, 9.3 / 9.1; Llama-3.2-3B 6.0 / 10.4, 9.6 / 11.5, 11.5 / 11.8, 14.3 / 12.1;
// 2 of up to 2048 (3B) 49.4 / 27.1.
template <typename KT>
static void launch_append_of(const PagedArgs& a, hipStream_t st) {
  const dim3 rows((unsigned)(a.seqs * a.tokens)), block(256);
  if (a.rd % 16) {
    hipLaunchKernelGGL(paged_append_kernel<KT>, rows, block, 0, st, a);
  } else if (a.tokens < 12) {
    hipLaunchKernelGGL(paged_append_row_kernel<KT>, rows, block, 0, st, a);
  } else {
    const int groups = (a.tokens + 30) / 32 + 1;  // aligned groups that `tokens` positions may touch
    const int slices = append_items(a.D, a.rd, 16 / sizeof(KT), a.q != nullptr).slices;
    hipLaunchKernelGGL(paged_append_group_kernel<KT>, dim3((unsigned)(a.seqs * groups * a.Hkv * slices)), block, 0, st,
                       a, groups);
  }
}

bool launch_paged_append(bool kv_f32, const PagedArgs& a, hipStream_t st) {
  if (kv_f32) launch_append_of<float>(a, st);
  else launch_append_of<uint16_t>(a, st);
  return true;
}

bool launch_paged_attention(bool kv_f32, const PagedArgs& a, int cus, size_t part_floats, hipStream_t st) {
#define PAGED_D(DT)                                                                \
  case DT:                                                                         \
    if (kv_f32) launch_attention_rows<float, DT>(a, cus, part_floats, st);         \
    else launch_attention_rows<uint16_t, DT>(a, cus, part_floats, st);             \
    return true;
  switch (a.D) { PAGED_D(32) PAGED_D(64) PAGED_D(96) PAGED_D(128) }
#undef PAGED_D
  return false;
}

}  // namespace tlm
