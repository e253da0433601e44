// Penalties for repeated tokens, biases and grammar masks on logits (tlm_op_adjust_logits).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "tlm_device.h"

namespace tlm {
namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // a row from any 4-byte address
typedef int i32x4 __attribute__((ext_vector_type(4)));

// y = x where token v has not been said, else (x > 0 ? x / rho : x rho) - presence -
// frequency c, c its occurrences in the history and in the drafts before the row; then
// + bias, then -inf where the mask has no bit.  A block counts the tokens of its chunk
// of a row's vocabulary in LDS, where it also has their biases, while its logits are on
// their way to registers, and makes one pass over the chunk; what a mask takes out four
// at a time is not read.  In place it reads and writes the fours that a rule changes.
constexpr int kThreads = 512, kFours = 2, kChunk = 4 * kFours * kThreads;
constexpr int kAhead = 8;  // tokens of the history in flight a thread

// What other lanes of the wave leave in LDS, in the order of its instructions.
template <typename T>
__device__ __forceinline__ T get_lds(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
template <typename T>
__device__ __forceinline__ void put_lds(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

template <bool MASKED, bool BIASED, bool PLACE>
__global__ __launch_bounds__(kThreads) void adjust_kernel(AdjustArgs a, int chunks) {
  constexpr int Q = kFours, C = kChunk;
  __shared__ __align__(16) int times[C];
  __shared__ __align__(16) float bias[BIASED ? C : 4];
  __shared__ int turn[BIASED ? 256 : 1];
  const int row = blockIdx.x / chunks, v0 = blockIdx.x % chunks * C, tid = threadIdx.x;
  const int s = row / a.tokens, j = row % a.tokens;
  const int n = min(C, a.vocab - v0);
  const float* const x = a.logits + (size_t)row * a.vocab + v0;
  float* const y = a.out + (size_t)row * a.vocab + v0;
  // requested before it is known whether the row is there
  uint32_t word[Q];
  if (MASKED) {
    const uint32_t* mask = a.masks + (size_t)row * ((a.vocab + 31) / 32) + v0 / 32;
#pragma unroll
    for (int q = 0; q < Q; q++) word[q] = mask[min(4 * (tid + q * kThreads), n - 1) / 32];
  }
  const int rows = a.counts ? a.counts[s] : a.tokens;
  const int h = !a.history ? 0 : a.history_counts ? min(max(a.history_counts[s], 0), a.history_width) : a.history_width;
  const int32_t* const ids = a.history + (size_t)s * a.history_width;
  const float rho = a.repetition ? a.repetition[s] : 1.f, fr = a.frequency ? a.frequency[s] : 0.f,
              pr = a.presence ? a.presence[s] : 0.f;
#pragma unroll
  for (int q = 0; q < Q; q++) {
    reinterpret_cast<i32x4*>(times)[tid + q * kThreads] = (i32x4){0, 0, 0, 0};
    if (BIASED) reinterpret_cast<f32x4*>(bias)[tid + q * kThreads] = (f32x4){-0.f, -0.f, -0.f, -0.f};
  }
  if (j >= rows) return;
  f32x4 l[Q];
  auto fetch = [&](int q) {
    const int i = 4 * (tid + q * kThreads);
    if (MASKED && !(word[q] >> (i & 31) & 15)) return;
    if (i + 4 <= n) {
      l[q] = *(const TLM_GLOBAL f32x4u*)(x + i);
    } else {
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (i + e < n) l[q][e] = x[i + e];
    }
  };
#pragma unroll
  for (int q = 0; q < Q && !PLACE; q++) fetch(q);
  __syncthreads();
  const bool said = h > 0 || (a.drafts && j > 0);
  for (int i0 = tid; i0 < h; i0 += kAhead * kThreads) {  // h <= kAdjustMaxHistory: no index passes 31 bits
    int id[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; k++) id[k] = i0 + k * kThreads < h ? ids[i0 + k * kThreads] : -1;
#pragma unroll
    for (int k = 0; k < kAhead; k++) {
      const unsigned v = (unsigned)id[k] - (unsigned)v0;
      if (id[k] >= 0 && v < (unsigned)n) atomicAdd(times + v, 1);
    }
  }
  if (a.drafts && tid < j) {
    const int id = a.drafts[(size_t)s * (a.tokens - 1) + tid];
    const unsigned v = (unsigned)id - (unsigned)v0;
    if (id >= 0 && v < (unsigned)n) atomicAdd(times + v, 1);
  }
  if (BIASED && tid < 64) {
    // One wave, 64 of the list at a time, so that a token listed more than once gets its
    // biases in the list's order: the first of the lanes that share a place of `turn` add
    // theirs at once, then the next; what is left after a few turns goes token by token (24
    // rows of 10198 with 151 biases: 10.7 us so from the start, 5.1 with the turns).
    for (int i = 0; i < a.bias_width; i += 64) {
      const bool here = i + tid < a.bias_width;
      const size_t at = (size_t)s * a.bias_width + i + (here ? tid : 0);
      const int id = here ? a.bias_ids[at] : -1;
      const float b = a.biases[at];
      const unsigned v = (unsigned)id - (unsigned)v0;
      bool todo = id >= 0 && v < (unsigned)n;
      for (int k = 0; k < 4 && __ballot(todo); k++) {
        int* const place = turn + (v & 255);
        if (todo) put_lds(place, 64);
        if (todo) __hip_atomic_fetch_min(place, tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        if (todo && get_lds(place) == tid) {
          put_lds(bias + v, get_lds(bias + v) + b);
          todo = false;
        }
      }
      uint64_t left = __ballot(todo);
      while (left) {
        const int first = __builtin_ctzll(left), at_v = __builtin_amdgcn_readlane((int)v, first);
        uint64_t same = __ballot((int)v == at_v) & left;
        left &= ~same;
        float sum = get_lds(bias + at_v);
        while (same) {
          sum += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(b), __builtin_ctzll(same)));
          same &= same - 1;
        }
        put_lds(bias + at_v, sum);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < Q; q++) {
    const int i = 4 * (tid + q * kThreads);
    if (i >= n) continue;
    const i32x4 c = reinterpret_cast<const i32x4*>(times)[tid + q * kThreads];
    f32x4 b = {-0.f, -0.f, -0.f, -0.f};  // x + -0 is x, of every x
    if (BIASED) b = reinterpret_cast<const f32x4*>(bias)[tid + q * kThreads];
    if (PLACE) {
      bool change = MASKED && (word[q] >> (i & 31) & 15) != 15;
#pragma unroll
      for (int e = 0; e < 4; e++) change |= c[e] > 0 || (BIASED && __float_as_uint(b[e]) != 0x80000000u);
      if (!change) continue;
      fetch(q);
    }
    if (said) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (c[e] > 0) l[q][e] = (l[q][e] > 0.f ? l[q][e] / rho : l[q][e] * rho) - pr - fr * (float)c[e];
    }
    if (BIASED) l[q] += b;
    if (MASKED) {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (!(word[q] >> ((i & 31) + e) & 1)) l[q][e] = -INFINITY;
    }
    if (i + 4 <= n) {
      *(TLM_GLOBAL f32x4u*)(y + i) = l[q];
    } else {
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (i + e < n) y[i + e] = l[q][e];
    }
  }
}

template <bool PLACE>
void launch_of(const AdjustArgs& a, hipStream_t st) {
  const int chunks = (a.vocab + kChunk - 1) / kChunk;
  const dim3 grid((unsigned)(a.seqs * a.tokens * chunks)), block(kThreads);
  if (a.masks && a.bias_ids) hipLaunchKernelGGL((adjust_kernel<true, true, PLACE>), grid, block, 0, st, a, chunks);
  else if (a.masks) hipLaunchKernelGGL((adjust_kernel<true, false, PLACE>), grid, block, 0, st, a, chunks);
  else if (a.bias_ids) hipLaunchKernelGGL((adjust_kernel<false, true, PLACE>), grid, block, 0, st, a, chunks);
  else hipLaunchKernelGGL((adjust_kernel<false, false, PLACE>), grid, block, 0, st, a, chunks);
}

}  // namespace

// Chunks of 4096.  Each block reads the whole history, so that larger chunks read less of
// it, but fewer of them fit a CU (16 KB of LDS each, 32 with biases): 62 rows of 128256 with
// everything and histories of 4096, chunks of 4096 / 6144 / 8192: 14.7 / 16.3 / 18.6 us (4.5 TB/s of
// logits); of 2048, 64 x 32000 5.8 against 5.6 and 1 x 5 x 151936 3.7 either way.  64 x 128256 without
// masks 14.7, in place 11.1 (histories of 300: 9.8, the blocks').
void launch_adjust(const AdjustArgs& a, hipStream_t st) {
  if (a.out == a.logits)
    launch_of<true>(a, st);
  else
    launch_of<false>(a, st);
}

}  // namespace tlm
