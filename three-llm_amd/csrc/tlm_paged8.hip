// The append to a paged cache of 8-bit values (tlm_op_paged_append, TLM_FMT_F8).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "tlm_device.h"
#include "tlm_paged.h"

namespace tlm {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // a row from any 4-byte address

__device__ __forceinline__ void flag(int* status, int bit) {
  __hip_atomic_fetch_or(status, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The magnitude of a value as far as it counts for its block's scale: values that are
// not finite become NaN codes and leave the others' precision alone.
__device__ __forceinline__ float magnitude(float v) { return fabsf(v) < INFINITY ? fabsf(v) : 0.f; }

// A value times 2^-e as its code: rounded to nearest even; past 448 (the largest scale)
// the largest code, NaN where it is not finite.
__device__ __forceinline__ float coded(float v, int e) {
  const float x = ldexpf(v, -e);
  return fabsf(x) <= 448.f ? x : fabsf(v) < INFINITY ? copysignf(448.f, x) : NAN;
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}
// Four codes under a scale 2^by times theirs (by >= 0): exact but for what falls below
// 2^-6 of the code's range.
__device__ __forceinline__ uint32_t recoded(uint32_t c, int by) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  return codes4(ldexpf(lo[0], -by), ldexpf(lo[1], -by), ldexpf(hi[0], -by), ldexpf(hi[1], -by));
}

// Eight dims from 8 o on of a rotated head's row x at a position (cs and sn: its cos and
// sin).  WHOLE: half the rotary dims are a multiple of 8, rows are read 16 bytes at a time.
template <bool WHOLE>
__device__ __forceinline__ void rotated_oct(const float* x, const float* cs, const float* sn, int d, int rd, float* y) {
  const int half = rd / 2;
  if (WHOLE) {
    const f32x4 a = *(const TLM_GLOBAL f32x4u*)(x + d), b = *(const TLM_GLOBAL f32x4u*)(x + d + 4);
    f32x4 ya = a, yb = b;
    if (d < rd) {
      const float sign = d < half ? -1.f : 1.f;
      const int to = d < half ? d + half : d - half, i = d < half ? d : d - half;
      const f32x4 p = *(const TLM_GLOBAL f32x4u*)(x + to), q = *(const TLM_GLOBAL f32x4u*)(x + to + 4);
      const f32x4 ca = *(const TLM_GLOBAL f32x4u*)(cs + i), cb = *(const TLM_GLOBAL f32x4u*)(cs + i + 4);
      const f32x4 sa = *(const TLM_GLOBAL f32x4u*)(sn + i), sb = *(const TLM_GLOBAL f32x4u*)(sn + i + 4);
      ya = a * ca + (sign * p) * sa;
      yb = b * cb + (sign * q) * sb;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = ya[e], y[4 + e] = yb[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int k = d + e;
      float v = x[k];
      if (k < rd) {
        const int i = k < half ? k : k - half;
        v = v * cs[i] + (k < half ? -x[k + half] : x[k - half]) * sn[i];
      }
      y[e] = v;
    }
  }
}

// Per sequence, kv head and aligned block of 32 positions: q' = R(p) q of the head's
// group; k' = R(p) k and v as codes under the block's scale, the larger of what its
// new rows need and, where it has rows before them, of its old one.  Rows before them
// are then coded again.  A block of threads has K and V in registers between the
// maximum and the codes (slice 0); queries are further blocks' (slices 1 ..).
template <bool WHOLE>
__global__ __launch_bounds__(256) void paged_append8_kernel(PagedArgs a, int groups, int slices) {
  __shared__ float top[2][4];
  const int slice = blockIdx.x % slices, block = blockIdx.x / slices, hk = block % a.Hkv;
  const int g = block / a.Hkv % groups, s = block / a.Hkv / groups, tid = threadIdx.x;
  const int start = a.starts[s];
  bool bad;
  const int rows = paged_rows(start, a.counts ? a.counts[s] : a.tokens, a.tokens, a.limit, &bad);
  if (bad && g == 0 && hk == 0 && slice == 0 && tid == 0) flag(a.status, kPagedStatusRows);
  if (rows < 1) return;
  const int p0 = ((start >> 5) + g) << 5, end = min(start + rows, p0 + 32);  // positions from max(start, p0) on
  if (p0 >= end) return;
  const int from = max(start, p0), n = end - from, D = a.D, octs = D / 8, half = a.rd / 2;
  const int N = (a.Hq + 2 * a.Hkv) * D;
  const size_t row0 = (size_t)s * a.tokens - start;  // + position: the row
  const float* const cs = a.rope_cos + (size_t)from * half;
  const float* const sn = a.rope_sin + (size_t)from * half;
  const float* const x0 = a.x + (row0 + from) * N;
  if (slice > 0) {
    const int items = n * a.G * octs;
    for (int i = (slice - 1) * 256 + tid; i < items; i += (slices - 1) * 256) {
      const int o = i % octs, h = i / octs % a.G, j = i / octs / a.G;
      float y[8];
      rotated_oct<WHOLE>(x0 + (size_t)j * N + (hk * a.G + h) * D, cs + j * half, sn + j * half, 8 * o, a.rd, y);
      float* q = a.q + ((row0 + from + j) * a.Hq + hk * a.G + h) * D + 8 * o;
      *(TLM_GLOBAL f32x4u*)(q) = (f32x4){y[0], y[1], y[2], y[3]};
      *(TLM_GLOBAL f32x4u*)(q + 4) = (f32x4){y[4], y[5], y[6], y[7]};
    }
    return;
  }
  const int page = paged_page(a.tables + (size_t)s * a.width, p0, a.page_shift, a.num_pages);
  if (page < 0) {
    if (tid == 0) flag(a.status, kPagedStatusPage);
    return;
  }
  const int tok0 = p0 & ((1 << a.page_shift) - 1);
  const size_t at = (size_t)page * a.page_bytes, head = (size_t)hk * ((size_t)D << a.page_shift);
  uint8_t* const kp = static_cast<uint8_t*>(a.kc) + at;
  uint8_t* const vp = static_cast<uint8_t*>(a.vc) + at;
  const size_t scale_at = paged8_scale_at(hk, a.Hkv, tok0, a.page_shift, D);
  uint32_t* const ks = reinterpret_cast<uint32_t*>(kp + scale_at);
  uint32_t* const vs = reinterpret_cast<uint32_t*>(vp + scale_at);
  const int held = from - p0;  // tokens of the block that it has already
  const uint32_t kold = held ? *ks : 0, vold = held ? *vs : 0;
  // at most 32 * 16 octs of K, and 4 * 128 dims of eight tokens of V (4 q .. of each sixteen)
  constexpr int NI = 2;
  float k[NI][8], v[NI][8];
  float kt = 0.f, vt = 0.f;
#pragma unroll
  for (int m = 0; m < NI; m++) {
    const int i = tid + 256 * m, o = i % octs, j = i / octs;
    if (j >= n) continue;
    rotated_oct<WHOLE>(x0 + (size_t)j * N + (a.Hq + hk) * D, cs + j * half, sn + j * half, 8 * o, a.rd, k[m]);
#pragma unroll
    for (int e = 0; e < 8; e++) kt = fmaxf(kt, magnitude(k[m][e]));
  }
#pragma unroll
  for (int m = 0; m < NI; m++) {
    const int i = tid + 256 * m, d = i % D, q = i / D;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int t = 4 * q + (e & 3) + 16 * (e >> 2) - held;
      v[m][e] = i < 4 * D && t >= 0 && t < n ? x0[(size_t)t * N + (a.Hq + a.Hkv + hk) * D + d] : 0.f;
      vt = fmaxf(vt, magnitude(v[m][e]));
    }
  }
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    kt = fmaxf(kt, __shfl_xor(kt, w));
    vt = fmaxf(vt, __shfl_xor(vt, w));
  }
  if ((tid & 63) == 0) top[0][tid >> 6] = kt, top[1][tid >> 6] = vt;
  __syncthreads();  // also: the old scales have been read
  kt = fmaxf(fmaxf(top[0][0], top[0][1]), fmaxf(top[0][2], top[0][3]));
  vt = fmaxf(fmaxf(top[1][0], top[1][1]), fmaxf(top[1][2], top[1][3]));
  int ke = paged8_exponent(__float_as_uint(kt)), ve = paged8_exponent(__float_as_uint(vt)), kby = 0, vby = 0;
  if (held) {
    const int k0 = paged8_exponent_of(kold), v0 = paged8_exponent_of(vold);
    ke = max(ke, k0), kby = ke - k0;
    ve = max(ve, v0), vby = ve - v0;
  }
  if (tid == 0) {
    *ks = (uint32_t)(ke + 127) << 23;
    *vs = (uint32_t)(ve + 127) << 23;
  }
#pragma unroll
  for (int m = 0; m < NI; m++) {
    const int i = tid + 256 * m, o = i % octs, j = i / octs;
    if (j >= n) continue;
    u32x2 c;
#pragma unroll
    for (int e = 0; e < 2; e++)
      c[e] = codes4(coded(k[m][4 * e], ke), coded(k[m][4 * e + 1], ke), coded(k[m][4 * e + 2], ke),
                    coded(k[m][4 * e + 3], ke));
    *(TLM_GLOBAL u32x2*)(kp + head + paged8_k_at(tok0 + held + j, 8 * o, D)) = c;
  }
  for (int i = tid; kby && i < held * octs; i += 256) {
    TLM_GLOBAL u32x2* p = (TLM_GLOBAL u32x2*)(kp + head + paged8_k_at(tok0 + i / octs, 8 * (i % octs), D));
    u32x2 c = *p;
    c[0] = recoded(c[0], kby), c[1] = recoded(c[1], kby);
    *p = c;
  }
#pragma unroll
  for (int m = 0; m < NI; m++) {
    const int i = tid + 256 * m, d = i % D, q = i / D;
    if (i >= 4 * D) continue;
    uint32_t is_new[2] = {0, 0}, is_held[2] = {0, 0};  // a byte per token
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const int t = 4 * q + (e & 3) + 16 * (e >> 2) - held;
      if (t >= 0 && t < n) is_new[e >> 2] |= 0xFFu << 8 * (e & 3);
      if (t < 0) is_held[e >> 2] |= 0xFFu << 8 * (e & 3);
    }
    if (!(is_new[0] | is_new[1]) && !(vby && (is_held[0] | is_held[1]))) continue;
    TLM_GLOBAL u32x2* p = (TLM_GLOBAL u32x2*)(vp + head + paged8_v_at(tok0 + 4 * q, d, D));
    u32x2 c = {0, 0};
    if ((is_new[0] & is_new[1]) != 0xFFFFFFFFu) c = *p;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (vby && is_held[e]) c[e] = (c[e] & ~is_held[e]) | (recoded(c[e], vby) & is_held[e]);
      const uint32_t y = codes4(coded(v[m][4 * e], ve), coded(v[m][4 * e + 1], ve), coded(v[m][4 * e + 2], ve),
                                coded(v[m][4 * e + 3], ve));
      c[e] = (c[e] & ~is_new[e]) | (y & is_new[e]);
    }
    *p = c;
  }
}

}  // namespace

void launch_paged_append8(const PagedArgs& a, hipStream_t st) {
  const int groups = (a.tokens + 30) / 32 + 1;  // aligned blocks that `tokens` positions may touch
  const int items = std::min(a.tokens, 32) * a.G * (a.D / 8);
  const int slices = 1 + (a.q ? (items + 255) / 256 : 0);
  const dim3 grid((unsigned)((int64_t)a.seqs * groups * a.Hkv * slices)), block(256);
  if (a.rd % 16)
    hipLaunchKernelGGL(paged_append8_kernel<false>, grid, block, 0, st, a, groups, slices);
  else
    hipLaunchKernelGGL(paged_append8_kernel<true>, grid, block, 0, st, a, groups, slices);
}

}  // namespace tlm
