// Serving many sequences from a paged cache: the new rows of every sequence
// rotated and appended to its pages (tlm_op_paged_append), and their attention
// over those pages (tlm_op_paged_attention).
#include <float.h>
#include <math.h>

#include "tlm_device.h"
#include "tlm_paged.h"

namespace tlm {
namespace {

__device__ __forceinline__ void paged_flag(int* status, int bit) {
  __hip_atomic_fetch_or(status, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// One block per row: q' = R(p) q, k' = R(p) k (rotate-half over the first rd
// dims) and v, k' and v rounded to the cache's type.
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

// One block per row and query head, 256 positions at a time: scores, their
// softmax carried with a running maximum, the weighted sum of the values.
template <typename KT>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedArgs a) {
  constexpr int E = 16 / sizeof(KT);
  __shared__ float q[128], p[256], red[8];
  const int h = blockIdx.x % a.Hq, row = blockIdx.x / a.Hq, s = row / a.tokens, j = row % a.tokens;
  const int start = a.starts[s], tid = threadIdx.x, D = a.D, hk = h / a.G;
  bool bad;
  const int rows = paged_rows(start, a.counts ? a.counts[s] : a.tokens, a.tokens, a.limit, &bad);
  if (bad && j == 0 && h == 0 && tid == 0) paged_flag(a.status, kPagedStatusRows);
  if (j >= rows) return;
  const int pos = start + j, first = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int* table = a.tables + (size_t)s * a.width;
  if (tid < D) q[tid] = a.x[((size_t)row * a.Hq + h) * D + tid] * a.scale;
  float M = -FLT_MAX, L = 0.f, acc = 0.f;
  for (int t0 = first; t0 <= pos; t0 += 256) {
    __syncthreads();
    const int t = t0 + tid;
    float sc = -INFINITY;
    if (t <= pos) {
      const int page = paged_page(table, t, a.page_shift, a.num_pages);
      if (page < 0) {
        paged_flag(a.status, kPagedStatusPage);
      } else {
        const KT* k = static_cast<const KT*>(a.kc) + paged_head_at(page, hk, a.Hkv, a.page_shift, D);
        sc = 0.f;
        for (int d = 0; d < D; d++)
          sc = fmaf(q[d], kv_load<KT>(k + paged_k_at(t & ((1 << a.page_shift) - 1), d, D, E)), sc);
      }
    }
    const float wm = wave_max(sc);
    if ((tid & 63) == 0) red[tid >> 6] = wm;
    __syncthreads();
    const float m = fmaxf(M, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float corr = __expf(M - m), e = __expf(sc - m);
    p[tid] = e;
    const float ws = wave_sum(e);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = ws;
    __syncthreads();
    L = L * corr + (red[4] + red[5] + red[6] + red[7]);
    M = m;
    acc *= corr;
    if (tid < D)
      for (int i = 0; i < min(256, pos + 1 - t0); i++) {
        const int page = paged_page(table, t0 + i, a.page_shift, a.num_pages);
        if (page < 0) continue;
        const KT* v = static_cast<const KT*>(a.vc) + paged_head_at(page, hk, a.Hkv, a.page_shift, D);
        acc = fmaf(p[i], kv_load<KT>(v + paged_v_at((t0 + i) & ((1 << a.page_shift) - 1), tid, D, E)), acc);
      }
  }
  if (tid >= D) return;
  const float y = L == 0.f ? 0.f : acc / L;  // 0: no position has a page
  const size_t at = ((size_t)row * a.Hq + h) * D + tid;
  if (a.out_f32) static_cast<float*>(a.out)[at] = y;
  else static_cast<uint16_t*>(a.out)[at] = kv_store<uint16_t>(y);
}

}  // namespace

bool launch_paged_append(bool kv_f32, const PagedArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.seqs * a.tokens));
  if (kv_f32) hipLaunchKernelGGL(paged_append_kernel<float>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(paged_append_kernel<uint16_t>, grid, dim3(256), 0, st, a);
  return true;
}

bool launch_paged_attention(bool kv_f32, const PagedArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.seqs * a.tokens * a.Hq));
  if (kv_f32) hipLaunchKernelGGL(paged_attention_kernel<float>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(paged_attention_kernel<uint16_t>, grid, dim3(256), 0, st, a);
  return true;
}

}  // namespace tlm
