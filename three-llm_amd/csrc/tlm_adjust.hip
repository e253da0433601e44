// Penalties for repeated tokens, biases and grammar masks on logits (tlm_op_adjust_logits).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "tlm_device.h"

namespace tlm {
namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // a row from any 4-byte address

// y = x where token v has not been said, else (x > 0 ? x / rho : x rho) - presence -
// frequency c, c its occurrences in the history and in the drafts before the row; then
// + bias, then -inf where the mask has no bit.  A block counts the tokens of its chunk
// of a row's vocabulary in LDS and then makes one pass over the chunk.
constexpr int kChunk = 4096, kThreads = 256;

__global__ __launch_bounds__(kThreads) void adjust_kernel(AdjustArgs a, int chunks) {
  __shared__ int times[kChunk];
  __shared__ float bias[kChunk];
  const int row = blockIdx.x / chunks, v0 = blockIdx.x % chunks * kChunk, tid = threadIdx.x;
  const int s = row / a.tokens, j = row % a.tokens;
  if (a.counts && j >= a.counts[s]) return;
  const int n = min(kChunk, a.vocab - v0);
  const bool said = a.history || (a.drafts && j > 0), biased = a.bias_ids != nullptr;
  for (int i = tid; i < kChunk; i += kThreads) {
    times[i] = 0;
    bias[i] = 0.f;
  }
  __syncthreads();
  if (a.history) {
    const int h = a.history_counts ? min(max(a.history_counts[s], 0), a.history_width) : a.history_width;
    const int32_t* ids = a.history + (size_t)s * a.history_width;
    for (int i = tid; i < h; i += kThreads) {
      const unsigned v = (unsigned)ids[i] - (unsigned)v0;
      if (v < (unsigned)n) atomicAdd(times + v, 1);
    }
  }
  if (a.drafts && tid < j) {
    const unsigned v = (unsigned)a.drafts[(size_t)s * (a.tokens - 1) + tid] - (unsigned)v0;
    if (v < (unsigned)n) atomicAdd(times + v, 1);
  }
  if (biased) {
    // a token listed more than once: the first place adds them up, in order
    const int32_t* ids = a.bias_ids + (size_t)s * a.bias_width;
    const float* b = a.biases + (size_t)s * a.bias_width;
    for (int i = tid; i < a.bias_width; i += kThreads) {
      const int id = ids[i];
      const unsigned v = (unsigned)id - (unsigned)v0;
      if (v >= (unsigned)n) continue;
      bool first = true;
      for (int k = 0; k < i && first; k++) first = ids[k] != id;
      if (!first) continue;
      float sum = b[i];
      for (int k = i + 1; k < a.bias_width; k++)
        if (ids[k] == id) sum += b[k];
      bias[v] = sum;
    }
  }
  __syncthreads();
  const float rho = a.repetition ? a.repetition[s] : 1.f, fr = a.frequency ? a.frequency[s] : 0.f,
              pr = a.presence ? a.presence[s] : 0.f;
  const float* x = a.logits + (size_t)row * a.vocab + v0;
  float* y = a.out + (size_t)row * a.vocab + v0;
  const uint32_t* mask = a.masks ? a.masks + (size_t)row * ((a.vocab + 31) / 32) + v0 / 32 : nullptr;
  auto value = [&](float l, int i, uint32_t bits) {
    const int c = said ? times[i] : 0;
    if (c > 0) l = (l > 0.f ? l / rho : l * rho) - pr - fr * (float)c;
    if (biased) l += bias[i];
    return bits >> (i & 31) & 1 ? l : -INFINITY;
  };
  for (int i = 4 * tid; i < n; i += 4 * kThreads) {
    const uint32_t bits = mask ? mask[i / 32] : 0xFFFFFFFFu;
    if (i + 4 <= n) {
      f32x4 l = *(const TLM_GLOBAL f32x4u*)(x + i);
#pragma unroll
      for (int e = 0; e < 4; e++) l[e] = value(l[e], i + e, bits);
      *(TLM_GLOBAL f32x4u*)(y + i) = l;
    } else {
      for (int e = 0; i + e < n; e++) y[i + e] = value(x[i + e], i + e, bits);
    }
  }
}

}  // namespace

void launch_adjust(const AdjustArgs& a, int cus, hipStream_t st) {
  const int chunks = (a.vocab + kChunk - 1) / kChunk;
  hipLaunchKernelGGL(adjust_kernel, dim3((unsigned)(a.seqs * a.tokens * chunks)), dim3(kThreads), 0, st, a, chunks);
}

}  // namespace tlm
