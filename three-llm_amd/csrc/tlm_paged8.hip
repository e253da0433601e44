// The append to a paged cache of 8-bit values (tlm_op_paged_append, TLM_FMT_F8).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "tlm_paged_rows.h"

namespace tlm {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
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
__device__ __forceinline__ u32x2 codes8(const Oct& x, int e) {
  return (u32x2){codes4(coded(x.a[0], e), coded(x.a[1], e), coded(x.a[2], e), coded(x.a[3], e)),
                 codes4(coded(x.b[0], e), coded(x.b[1], e), coded(x.b[2], e), coded(x.b[3], e))};
}
// Four codes under a scale 2^by times theirs (by >= 0): exact but for magnitudes below 2^-6
// of the new scale, the least normal code.
__device__ __forceinline__ uint32_t recoded(uint32_t c, int by) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  return codes4(ldexpf(lo[0], -by), ldexpf(lo[1], -by), ldexpf(hi[0], -by), ldexpf(hi[1], -by));
}

// The bytes of four tokens of which the first n are there.
__device__ __forceinline__ uint32_t held_bytes(int n) { return n >= 4 ? ~0u : n > 0 ? (1u << 8 * n) - 1 : 0u; }

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

// The rows of a sequence that lie in one aligned block of 32 positions.
struct Rows {
  int p0, from, n, held;  // the block, its first new position, how many, those before them in the block
};
__device__ __forceinline__ Rows rows_of(const PagedArgs& a, int s, int g, int start, int count, bool* bad) {
  const int rows = paged_rows(start, count, a.tokens, a.limit, bad);
  Rows r;
  r.p0 = ((start >> 5) + g) << 5;
  r.from = max(start, r.p0);
  r.n = rows < 1 ? 0 : max(0, min(start + rows, r.p0 + 32) - r.from);
  r.held = r.from - r.p0;
  return r;
}

// q' = R(p) q of the block's new rows, items `first`, `first` + `step`, ... of n * Hq * D / 8.
template <bool WHOLE>
__device__ __forceinline__ void append8_queries(const PagedArgs& a, size_t row, const Rows& r, int heads, int h0,
                                                int first, int step) {
  const int D = a.D, octs = D / 8, half = a.rd / 2, N = (a.Hq + 2 * a.Hkv) * D, items = r.n * heads * octs;
  for (int i = first; i < items; i += step) {
    const int o = i % octs, h = h0 + i / octs % heads, j = i / octs / heads;
    float y[8];
    rotated_oct<WHOLE>(a.x + (row + j) * N + h * D, a.rope_cos + (size_t)(r.from + j) * half,
                       a.rope_sin + (size_t)(r.from + j) * half, 8 * o, a.rd, y);
    float* q = a.q + ((row + j) * a.Hq + h) * D + 8 * o;
    *(TLM_GLOBAL f32x4u*)(q) = (f32x4){y[0], y[1], y[2], y[3]};
    *(TLM_GLOBAL f32x4u*)(q + 4) = (f32x4){y[4], y[5], y[6], y[7]};
  }
}

// Two kernels.  Both: k' = R(p) k and v as codes under the scale of the block of 32
// positions, the larger of what its new rows need and, where it has rows before them,
// of its old one; those rows are then coded again.
//
// Few rows: 16 lanes per row, kv head and K or V, a lane per eight dims (of V as many apart
// as there are lanes, so that a store's bytes lie together), in registers between the
// maximum and the codes; a block has the rows of `heads` kv heads, the queries are further
// blocks' (slices from `parts` on).  Latency: loads of the start, then of the table, the old
// scales and the rows, then the stores (64 x 1 Llama-3.2-1B 4.1 us, 0.9 MB read and as much written).
constexpr int kFewHeads = 8;  // that a block has, of one row each
template <bool WHOLE>
__global__ __launch_bounds__(256) void paged_append8_few_kernel(PagedArgs a, int groups, int heads, int parts, int slices) {
  constexpr int NI = 4;  // 2 * 32 rows of one head, where rotations of an odd width bring so many here
  __shared__ unsigned top[2][kFewHeads];
  const int slice = blockIdx.x % slices, block = blockIdx.x / slices, g = block % groups, s = block / groups;
  const int tid = threadIdx.x, D = a.D, octs = D / 8, half = a.rd / 2, N = (a.Hq + 2 * a.Hkv) * D;
  if (tid < 2 * kFewHeads) top[tid / kFewHeads][tid % kFewHeads] = 0;
  const int start = a.starts[s];
  bool bad;
  const Rows r = rows_of(a, s, g, start, a.counts ? a.counts[s] : a.tokens, &bad);
  if (bad && g == 0 && slice == 0 && tid == 0) paged_flag(a.status, kPagedStatusRows);
  if (r.n == 0) return;
  const size_t row = (size_t)s * a.tokens + r.from - start;
  if (slice >= parts) {
    append8_queries<WHOLE>(a, row, r, a.Hq, 0, (slice - parts) * 256 + tid, (slices - parts) * 256);
    return;
  }
  const int page = paged_page(a.tables + (size_t)s * a.width, r.p0, a.page_shift, a.num_pages);
  if (page < 0) {
    if (slice == 0 && tid == 0) paged_flag(a.status, kPagedStatusPage);
    return;
  }
  const int tok0 = r.p0 & ((1 << a.page_shift) - 1), h0 = slice * heads, here = min(heads, a.Hkv - h0);
  const int items = 2 * here * r.n, o = min(tid & 15, octs - 1), d = 8 * o;
  const bool mine = (tid & 15) < octs;
  const float* const cs = a.rope_cos + (size_t)r.from * half;
  const float* const sn = a.rope_sin + (size_t)r.from * half;
  // item i: row j of head h's K, then of its V
  struct Item {
    int j, h;
    bool is_v;
  };
  auto item_of = [&](int i) { return Item{i % r.n, i / r.n % here, i / r.n >= here}; };
  auto page_at = [&](const Item& x) {
    return static_cast<uint8_t*>(x.is_v ? a.vc : a.kc) + (size_t)page * a.page_bytes;
  };
  float y[NI][8];
  uint32_t old[NI];
  __syncthreads();  // the maxima are 0
#pragma unroll
  for (int m = 0; m < NI; m++) {
    if (16 * m >= items) break;
    const int i = 16 * m + (tid >> 4);
    const Item x = item_of(min(i, items - 1));
    old[m] = 0;
    if (r.held) old[m] = *reinterpret_cast<const uint32_t*>(page_at(x) + paged8_scale_at(h0 + x.h, a.Hkv, tok0, a.page_shift, D));
    const float* const p = a.x + (row + x.j) * N + (a.Hq + h0 + x.h) * D;
    if (x.is_v) {
      const float* v = p + a.Hkv * D + o;
#pragma unroll
      for (int e = 0; e < 8; e++) y[m][e] = v[e * octs];
    } else {
      rotated_oct<WHOLE>(p, cs + x.j * half, sn + x.j * half, d, a.rd, y[m]);
    }
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) t = fmaxf(t, magnitude(y[m][e]));
    t = fmaxf(t, dpp<kDppXor1>(t));
    t = fmaxf(t, dpp<kDppXor2>(t));
    t = fmaxf(t, dpp<kDppHalfMirror>(t));
    t = fmaxf(t, dpp<kDppMirror>(t));
    if (i < items && (tid & 15) == 0) atomicMax(&top[x.is_v][x.h], __float_as_uint(t));
  }
  __syncthreads();  // also: the old scales have been read
  int ex[NI];
#pragma unroll
  for (int m = 0; m < NI; m++) {
    if (16 * m >= items) break;
    const int i = 16 * m + (tid >> 4);
    const Item x = item_of(min(i, items - 1));
    ex[m] = paged8_exponent(top[x.is_v][x.h]);
    if (i >= items || !r.held) continue;
    const int was = paged8_exponent_of(old[m]);
    ex[m] = max(ex[m], was);
    const int by = ex[m] - was;
    if (!by || !mine) continue;
    // what the block has is coded again, by the rows' lanes in turn
    uint8_t* const head = page_at(x) + (size_t)(h0 + x.h) * ((size_t)D << a.page_shift);
    for (int t = x.j; !x.is_v && t < r.held; t += r.n) {
      TLM_GLOBAL u32x2* c = (TLM_GLOBAL u32x2*)(head + paged8_k_at(tok0 + t, d, D));
      const u32x2 v = *c;
      *c = (u32x2){recoded(v[0], by), recoded(v[1], by)};
    }
    for (int t = 4 * x.j; x.is_v && t < min(r.held, 16); t += 4 * r.n) {  // tokens t .. t + 3 and 16 further on
      const uint32_t lo = held_bytes(r.held - t), hi = held_bytes(r.held - t - 16);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        TLM_GLOBAL u32x2* c = (TLM_GLOBAL u32x2*)(head + paged8_v_at(tok0 + t, o + e * octs, D));
        const u32x2 v = *c;
        *c = (u32x2){(recoded(v[0], by) & lo) | (v[0] & ~lo), (recoded(v[1], by) & hi) | (v[1] & ~hi)};
      }
    }
  }
  if (r.held) __syncthreads();  // V's words have been written: bytes of them follow
#pragma unroll
  for (int m = 0; m < NI; m++) {
    if (16 * m >= items) break;
    const int i = 16 * m + (tid >> 4);
    if (i >= items || !mine) continue;
    const Item x = item_of(i);
    uint8_t* const p = page_at(x);
    uint8_t* const head = p + (size_t)(h0 + x.h) * ((size_t)D << a.page_shift);
    if (x.j == 0 && o == 0)
      *reinterpret_cast<uint32_t*>(p + paged8_scale_at(h0 + x.h, a.Hkv, tok0, a.page_shift, D)) = (uint32_t)(ex[m] + 127) << 23;
    u32x2 c;
#pragma unroll
    for (int e = 0; e < 2; e++)
      c[e] = codes4(coded(y[m][4 * e], ex[m]), coded(y[m][4 * e + 1], ex[m]), coded(y[m][4 * e + 2], ex[m]),
                    coded(y[m][4 * e + 3], ex[m]));
    const int t = tok0 + r.held + x.j;
    if (!x.is_v) {
      *(TLM_GLOBAL u32x2*)(head + paged8_k_at(t, d, D)) = c;
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) head[paged8_v_at(t, o + e * octs, D)] = (uint8_t)(c[e >> 2] >> 8 * (e & 3));
    }
  }
}

// Many rows: a block of threads per kv head, which has K and V in registers between the
// maximum and the codes (slice 0); the queries of the head's group are further blocks'.
// Half the rotary dims are a multiple of 8 here.
__global__ __launch_bounds__(256) void paged_append8_kernel(PagedArgs a, int groups, int slices) {
  __shared__ float top[2][4];
  const int slice = blockIdx.x % slices, block = blockIdx.x / slices, hk = block % a.Hkv;
  const int g = block / a.Hkv % groups, s = block / a.Hkv / groups, tid = threadIdx.x;
  const int start = a.starts[s];
  bool bad;
  const Rows r = rows_of(a, s, g, start, a.counts ? a.counts[s] : a.tokens, &bad);
  if (bad && g == 0 && hk == 0 && slice == 0 && tid == 0) paged_flag(a.status, kPagedStatusRows);
  if (r.n == 0) return;
  const int p0 = r.p0, from = r.from, n = r.n, held = r.held, D = a.D, octs = D / 8, half = a.rd / 2;
  const int N = (a.Hq + 2 * a.Hkv) * D;
  const size_t row = (size_t)s * a.tokens + from - start;
  const float* const cs = a.rope_cos + (size_t)from * half;
  const float* const sn = a.rope_sin + (size_t)from * half;
  const float* const x0 = a.x + row * N;
  if (slice > 0) {
    const int quads = D / 4 - a.rd / 8, item = (slice - 1) * 256 + tid;
    if (item < 32 * quads) append_quad(a, hk, p0, start, from + n - 1, row - from, item, quads);
    return;
  }
  const int page = paged_page(a.tables + (size_t)s * a.width, p0, a.page_shift, a.num_pages);
  if (page < 0) {
    if (tid == 0) paged_flag(a.status, kPagedStatusPage);
    return;
  }
  const int tok0 = p0 & ((1 << a.page_shift) - 1);
  const size_t at = (size_t)page * a.page_bytes, head = (size_t)hk * ((size_t)D << a.page_shift);
  uint8_t* const kp = static_cast<uint8_t*>(a.kc) + at;
  uint8_t* const vp = static_cast<uint8_t*>(a.vc) + at;
  const size_t scale_at = paged8_scale_at(hk, a.Hkv, tok0, a.page_shift, D);
  uint32_t* const ks = reinterpret_cast<uint32_t*>(kp + scale_at);
  uint32_t* const vs = reinterpret_cast<uint32_t*>(vp + scale_at);
  const uint32_t kold = held ? *ks : 0, vold = held ? *vs : 0;
  // at most 32 * 16 octs of K (with their partners 32 * 8), and 4 * 128 dims of eight
  // tokens of V (4 q .. of each sixteen)
  constexpr int NI = 2;
  const Octs oc(D, a.rd);
  Oct k[NI][2];
  float v[NI][8];
  float kt = 0.f, vt = 0.f;
#pragma unroll
  for (int m = 0; m < NI; m++) {
    const int i = tid + 256 * m, o = i % oc.n, j = i / oc.n, d = oc.dim(o);
    if (j >= n) continue;
    const float* x = x0 + (size_t)j * N + (a.Hq + hk) * D + d;
    k[m][0].load(x);
    if (oc.pair(o)) {
      Oct c, w;
      k[m][1].load(x + half);
      c.load(cs + (size_t)j * half + d);
      w.load(sn + (size_t)j * half + d);
      const Oct y = k[m][0];
      k[m][0].a = rotated(y.a, -k[m][1].a, c.a, w.a), k[m][0].b = rotated(y.b, -k[m][1].b, c.b, w.b);
      k[m][1].a = rotated(k[m][1].a, y.a, c.a, w.a), k[m][1].b = rotated(k[m][1].b, y.b, c.b, w.b);
#pragma unroll
      for (int e = 0; e < 4; e++) kt = fmaxf(kt, fmaxf(magnitude(k[m][1].a[e]), magnitude(k[m][1].b[e])));
    }
#pragma unroll
    for (int e = 0; e < 4; e++) kt = fmaxf(kt, fmaxf(magnitude(k[m][0].a[e]), magnitude(k[m][0].b[e])));
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
  kt = wave_max(kt);
  vt = wave_max(vt);
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
    const int i = tid + 256 * m, o = i % oc.n, j = i / oc.n, d = oc.dim(o);
    if (j >= n) continue;
    *(TLM_GLOBAL u32x2*)(kp + head + paged8_k_at(tok0 + held + j, d, D)) = codes8(k[m][0], ke);
    if (oc.pair(o)) *(TLM_GLOBAL u32x2*)(kp + head + paged8_k_at(tok0 + held + j, d + half, D)) = codes8(k[m][1], ke);
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
  const dim3 block(256);
  // us a call, few-rows / many-rows kernel, 64 sequences of 4, 8, 12 and 16 tokens: Llama-3.2-1B heads
  // 6.1 / 11.7, 9.9 / 12.1, 9.7 / 12.9, 11.8 / 13.0; Llama-3.2-3B 6.0 / 11.4, 8.5 / 12.7, 11.1 / 14.1,
  // 17.1 / 14.7.  2 x up to 2048 (3B, 122 MB) 28.5 us, 4.3 TB/s; of Llama-3.2-1B 14.4, with 20
  // rotated dims, which only the few-rows kernel takes, 43.3.
  if (a.tokens <= 12 || a.rd % 16) {
    const int heads = std::max(1, kFewHeads / a.tokens), parts = (a.Hkv + heads - 1) / heads;
    const int slices = parts + (a.q ? (std::min(a.tokens, 32) * a.Hq * (a.D / 8) + 255) / 256 : 0);
    const dim3 grid((unsigned)((int64_t)a.seqs * groups * slices));
    if (a.rd % 16)
      hipLaunchKernelGGL(paged_append8_few_kernel<false>, grid, block, 0, st, a, groups, heads, parts, slices);
    else
      hipLaunchKernelGGL(paged_append8_few_kernel<true>, grid, block, 0, st, a, groups, heads, parts, slices);
    return;
  }
  const int slices = 1 + (a.q ? (32 * (a.D / 4 - a.rd / 8) + 255) / 256 : 0);
  hipLaunchKernelGGL(paged_append8_kernel, dim3((unsigned)((int64_t)a.seqs * groups * a.Hkv * slices)), block, 0, st, a,
                     groups, slices);
}

}  // namespace tlm
