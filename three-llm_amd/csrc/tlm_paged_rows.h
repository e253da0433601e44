// Rows of a step on their way to paged caches: what the append kernels of all cache
// types share.
#pragma once
#include "tlm_device.h"
#include "tlm_paged.h"

namespace tlm {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // a row from any 4-byte address

__device__ __forceinline__ void paged_flag(int* status, int bit) {
  __hip_atomic_fetch_or(status, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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

// Four dims of a token's queries and their partners, head after head of a kv head's
// group: cos and sin are read once for them, a wave covers whole cache lines.  Item of 32
// tokens from p0 on by `quads`; row0 + position: the row.
__device__ __forceinline__ void append_quad(const PagedArgs& a, int hk, int p0, int start, int last, size_t row0, int item,
                                            int quads) {
  const int D = a.D, half = a.rd / 2, N = (a.Hq + 2 * a.Hkv) * D;
  const int f = item % quads, pos = p0 + item / quads, d = 4 * f < half ? 4 * f : 4 * f + half;
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
}

}  // namespace tlm
