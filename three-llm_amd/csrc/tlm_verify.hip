// Verification of drafted tokens against the target's logits
// (tlm_op_verify_drafts), greedy or by given random numbers.
//
// Row j of a sequence has the distribution p_j = softmax(logits_j / T); its
// draft x_j came from q_j = softmax(draft logits_j / T), or q_j(x_j) = 1.  The
// draft stands where u_j q_j(x_j) < p_j(x_j); at the first that does not, and
// after the last, a token is drawn: the lowest i with
//   sum_{k <= i} w_k > u sum_k w_k,   w = max(p_j - q_j, 0), or p_j after the last.
// Everything is in 64 bits: which token is drawn hangs on sums over the
// vocabulary, and 32-bit ones (2^-24 a term) would move a border past u once in
// some hundred draws from a flat distribution over 10^5 tokens.
//
// One pass over the logits: a wave takes kVChunk entries of a row into registers
// and leaves their maximum and sum of exponentials (greedy: the best entry).  The
// block that finishes a sequence's last chunk decides from these few numbers and
// reads one more chunk for the token, in the same launch.  With draft logits the
// refused row's max(p - q, 0) takes a second launch.
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "tlm_device.h"

namespace tlm {
namespace {

constexpr int kVW = 8;                    // waves per block, a chunk each
constexpr int kVT = 64 * kVW;             // threads
constexpr int kVChunk = 2048;             // entries: 32 a lane of a wave, 4 a thread of a block
constexpr int kVQuads = kVChunk / 4 / 64;
constexpr int kRestWaves = 2;             // waves that share a chunk of the second launch
constexpr int kVRow = kVerifyMaxVocab / kVChunk / 64;  // chunks of a row that a lane holds
static_assert(kVChunk == 4 * kVT, "a block takes a chunk in one step");

typedef float vf4 __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any 4-byte address

// What the steps pass on.  Cells: per sequence and row (its target rows, then
// its draft rows) and chunk.
struct Decision {
  double s, sq;  // 1 / sum of the row the token is drawn from, of the draft's (0: it has no entry)
  float m, mq;   // their maxima
  int row;       // target row (of all)
  int draft;     // draft row, or -1: the token is known already
};
struct VerifyWork {
  unsigned long long* cell;  // sum of exp((l - max) / T), greedy: the best entry's key
  float* max;
  double* rest;  // per sequence and chunk: the sum of max(p - q, 0)
  Decision* dec;
};
__host__ __device__ inline VerifyWork verify_work(const VerifyArgs& a) {
  const size_t cells = (size_t)a.seqs * a.rows * a.chunks;
  VerifyWork w;
  w.cell = static_cast<unsigned long long*>(a.work);
  w.rest = reinterpret_cast<double*>(w.cell + cells);
  w.dec = reinterpret_cast<Decision*>(w.rest + (size_t)a.seqs * a.chunks);
  w.max = reinterpret_cast<float*>(w.dec + a.seqs);
  return w;
}

// Values that another block of the same launch reads: past the XCD's L2.
template <typename T>
__device__ __forceinline__ void publish(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T published(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// exp((l - m) / T) = 2^((l - m) c), c = log2(e) / T, for a row's maximum m.
// Entries at or below LOWEST_FLOAT (-inf and NaN included) never take part.
// 2^t, t <= 0: t's nearest whole number through the sum with 1.5 * 2^52, and the
// series of 2^f, |f| <= 1/2, up to f^9, its last term spread over f .. f^7 by the
// Chebyshev polynomial T9(2 f) = 0 (2^0 stays 1).  Off by (ln 2 / 2)^10 / 10! = 7e-12
// for what the series leaves out and (ln 2 / 2)^9 / 9! / 256 = 8e-13 for T9, together
// 8.4e-12 of 2^f (a border between tokens moves by so much of what lies below it).  The
// coefficients stay in scalar registers (as literals each took two moves a term).
// No entry is below `floor`, 2^-1100 of the maximum, which is 0: one 32-bit maximum
// for masked entries, NaN and the exponent's range.
constexpr double kLn2 = 0.693147180559945309417232121458;
constexpr double coef(int n) { return n == 0 ? 1.0 : coef(n - 1) * kLn2 / n; }
// f^9 = (576 y^7 - 432 y^5 + 120 y^3 - 9 y) / 256 / 2^9 where T9(y) = 0, y = 2 f
constexpr double spread(int n, double of_y) { return coef(n) + coef(9) * of_y / 256 / (1 << (9 - n)); }
struct Weights {
  double c, m, co[9];
  float mf, floor;
  bool plain;  // else the floor is none: m is infinite, the temperature past 1e35 or so low that m - floor is lost
  __device__ __forceinline__ Weights(float max, double scale) : c(scale), m(max), mf(max) {
    constexpr double k[9] = {1.0,     spread(1, -9),   coef(2), spread(3, 120), coef(4),
                             spread(5, -432), coef(6), spread(7, 576), coef(8)};
#pragma unroll
    for (int i = 0; i < 9; i++) {
      co[i] = k[i];
      asm("" : "+s"(co[i]));
    }
    const double deep = 1100.0 / scale;
    floor = (float)(m - deep);
    plain = floor > kLowest && 1024.0 * deep >= fabs(m);
  }
  static constexpr double kBig = 6755399441055744.0;
  __device__ __forceinline__ double power(double k, double f) const {  // 2^(k - kBig + f)
    double p = co[8];
#pragma unroll
    for (int n = 7; n >= 0; n--) p = fma(p, f, co[n]);
    return ldexp(p, __double2loint(k));
  }
  __device__ __forceinline__ double series(float l) const {
    const double d = (double)fmaxf(l, floor) - m, k = fma(d, c, kBig);
    return power(k, fma(d, c, kBig - k));
  }
  __device__ __forceinline__ double of(float l) const {  // any entry and maximum
    if (plain) return series(l);
    const double t = fmax(((double)l - m) * c, -1100.0), k = t + kBig;
    const double p = power(k, t - (k - kBig));
    return !(l > kLowest) ? 0.0 : l == mf ? 1.0 : p;
  }
};

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ double dpp_f64(double v) {  // lanes without a source: 0
  return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xF, false),
                          __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ double readlane_f64(double v, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v += dpp_f64<kDppXor1>(v);
  v += dpp_f64<kDppXor2>(v);
  v += dpp_f64<kDppHalfMirror>(v);
  v += dpp_f64<kDppMirror>(v);
  return (readlane_f64(v, 0) + readlane_f64(v, 16)) + (readlane_f64(v, 32) + readlane_f64(v, 48));
}
__device__ __forceinline__ double wave_scan_f64(double v) {  // inclusive
  v += dpp_f64<0x111>(v);       // row_shr:1, within 16 lanes
  v += dpp_f64<0x112>(v);
  v += dpp_f64<0x114>(v);
  v += dpp_f64<0x118>(v);
  v += dpp_f64<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp_f64<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long k) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const unsigned long long x = (unsigned long long)__shfl_xor((long long)k, o);
    k = x > k ? x : k;
  }
  return k;
}

__device__ __forceinline__ int row_count(const VerifyArgs& a, int s) {
  return a.counts ? min(a.counts[s], a.tokens) : a.tokens;
}

// Entries 4 lane + 256 k + e from i0 on, k < N; past the end -inf.
template <int N>
__device__ __forceinline__ void load_quads(const float* x, int i0, int n, vf4* v) {
  const int lane = threadIdx.x & 63;
  if (i0 + 256 * N <= n) {
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = *(const TLM_GLOBAL vf4*)(x + i0 + 256 * k + 4 * lane);
  } else {
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int i = i0 + 256 * k + 4 * lane + e;
        v[k][e] = i < n ? x[i] : -INFINITY;
      }
  }
}

struct VerifyShared {
  double red[kVW], s[kVerifyMaxTokens], sq[kVerifyMaxTokens];
  float m[kVerifyMaxTokens], mq[kVerifyMaxTokens], lx[kVerifyMaxTokens];
  int ok[kVerifyMaxTokens], top[kVerifyMaxTokens], x[kVerifyMaxTokens], hit[kVW], last[kVW];
  unsigned long long done;
  unsigned before;
  int chunk, again;  // find_chunk's
  double base, border;
};

// A row's chunks in a wave's registers: chunk lane + 64 k.
struct RowSums {
  float max[kVRow];
  double raw[kVRow], sum[kVRow];  // relative to max; to the row's maximum
};
__device__ __forceinline__ void row_load(const VerifyArgs& a, const VerifyWork& w, size_t row, RowSums& r) {
#pragma unroll
  for (int k = 0; k < kVRow; k++) {
    const int c = (threadIdx.x & 63) + 64 * k;
    r.raw[k] = c < a.chunks ? __longlong_as_double((long long)published(w.cell + row * a.chunks + c)) : 0.0;
    r.max[k] = c < a.chunks ? published(w.max + row * a.chunks + c) : -INFINITY;
  }
}
// The row's maximum and sum, in every lane (a chunk or a row without entries: 0).
__device__ __forceinline__ void row_scale(const VerifyArgs& a, RowSums& r, float* m, double* s) {
  float mx = r.max[0];
#pragma unroll
  for (int k = 1; k < kVRow; k++) mx = fmaxf(mx, r.max[k]);
  mx = wave_max(mx);
  const Weights w(mx, a.scale);
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kVRow; k++) {
    r.sum[k] = 64 * k < a.chunks && r.raw[k] > 0.0 ? r.raw[k] * w.of(r.max[k]) : 0.0;
    sum += r.sum[k];
  }
  *m = mx;
  *s = wave_sum_f64(sum);
}

// One wave: the chunk in which the running sum of the chunks passes u times the
// whole, the sum before it and that border, into sh.  Rounding may leave the last
// border at u: then the last chunk with a weight.  -1: all are zero.
__device__ void find_chunk(const double* v, float u, VerifyShared& sh) {
  const int lane = threadIdx.x & 63;
  double incl[kVRow], total = 0.0;
#pragma unroll
  for (int k = 0; k < kVRow; k++) {
    incl[k] = total + wave_scan_f64(v[k]);
    total = readlane_f64(incl[k], 63);
  }
  const double border = (double)u * total;
  int chunk = -1, last = -1;
  double base = 0.0, last_base = 0.0;
#pragma unroll
  for (int k = 0; k < kVRow; k++) {
    const unsigned long long some = __ballot(v[k] > 0.0), over = __ballot(v[k] > 0.0 && incl[k] > border);
    const double before = incl[k] - v[k];
    if (chunk < 0 && over) {
      const int l = __builtin_ctzll(over);
      chunk = 64 * k + l;
      base = readlane_f64(before, l);
    }
    if (some) {
      const int l = 63 - __builtin_clzll(some);
      last = 64 * k + l;
      last_base = readlane_f64(before, l);
    }
  }
  if (lane == 0) {
    sh.chunk = chunk < 0 ? last : chunk;
    sh.base = chunk < 0 ? last_base : base;
    sh.border = border;
  }
}

// The block: the entry of sh.chunk, at(i, v) an entry's four weights from i on.
template <typename At>
__device__ int find_entry(const VerifyArgs& a, At at, VerifyShared& sh) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int i0 = sh.chunk * kVChunk + 4 * tid;
  double v[4], mine = 0.0;
  at(i0, v);
  int mlast = -1;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    mine += v[e];
    if (v[e] > 0.0) mlast = i0 + e;
  }
  const double incl = wave_scan_f64(mine), border = sh.border;
  double run = sh.base;
  const unsigned long long some = __ballot(mlast >= 0);
  const int wlast = some ? __builtin_amdgcn_readlane(mlast, 63 - __builtin_clzll(some)) : -1;
  if (lane == 63) sh.red[tid >> 6] = incl;
  __syncthreads();
  for (int k = 0; k < tid >> 6; k++) run += sh.red[k];
  run += incl - mine;
  int hit = -1;
#pragma unroll
  for (int e = 0; e < 4; e++) {
    run += v[e];
    if (hit < 0 && v[e] > 0.0 && run > border) hit = i0 + e;
  }
  const unsigned long long over = __ballot(hit >= 0);
  const int whit = over ? __builtin_amdgcn_readlane(hit, __builtin_ctzll(over)) : -1;
  if (lane == 0) sh.hit[tid >> 6] = whit, sh.last[tid >> 6] = wlast;
  __syncthreads();
  int last = -1;
  for (int k = 0; k < kVW; k++) {
    if (sh.hit[k] >= 0) return sh.hit[k];
    if (sh.last[k] >= 0) last = sh.last[k];
  }
  return last;
}

// Four entries of a row from i on; past the end -inf (of no weight).
__device__ __forceinline__ vf4 row_quad(const float* x, int i, int n) {
  if (i + 4 <= n) return *(const TLM_GLOBAL vf4*)(x + i);
  vf4 v;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = i + e < n ? x[i + e] : -INFINITY;
  return v;
}

__device__ double block_sum_f64(double v, VerifyShared& sh) {
  v = wave_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int i = 0; i < kVW; i++) r += sh.red[i];
  __syncthreads();
  return r;
}

// Which drafts of a sequence stand, and the token after them where no draft
// logits are to be subtracted.  The whole block.
template <bool GREEDY>
__device__ void decide(const VerifyArgs& a, int s, VerifyShared& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, T = a.tokens;
  const VerifyWork w = verify_work(a);
  const int n = row_count(a, s);
  __syncthreads();  // sh of the sequence before has been read
  RowSums rp;
  for (int j = wave; j < n; j += kVW) {
    const size_t row = (size_t)s * a.rows + j;
    const bool model = !GREEDY && a.draft_logits && j < n - 1;
    RowSums rq;
    unsigned long long best = 0;
    if (GREEDY) {
#pragma unroll
      for (int i = 0; i < kVRow; i++) {
        const int c = lane + 64 * i;
        const unsigned long long y = c < a.chunks ? published(w.cell + row * a.chunks + c) : 0;
        best = y > best ? y : best;
      }
    } else {
      row_load(a, w, row, rp);
      if (model) row_load(a, w, (size_t)s * a.rows + T + j, rq);
    }
    const int id = j < n - 1 ? a.drafts[s * (T - 1) + j] : -1, x = id < a.vocab ? id : -1;
    if (lane == 0) sh.x[j] = x;
    if (GREEDY) {
      best = wave_max_key(best);
      if (lane == 0) {
        sh.top[j] = best ? greedy_key_id(best) : -1;
        sh.ok[j] = x >= 0 && x == sh.top[j];
      }
      continue;
    }
    const float lx = x >= 0 ? a.logits[((size_t)s * T + j) * a.vocab + x] : -INFINITY;
    const float qx = x >= 0 && model ? a.draft_logits[((size_t)s * (T - 1) + j) * a.vocab + x] : -INFINITY;
    const float u = a.uniforms[s * T + j];
    float m, mq = 0.f;
    double sum, sq = 0.0;
    row_scale(a, rp, &m, &sum);
    if (model) row_scale(a, rq, &mq, &sq);
    const double p = sum > 0.0 ? Weights(m, a.scale).of(lx) / sum : 0.0;
    const double q = !model ? 1.0 : sq > 0.0 ? Weights(mq, a.scale).of(qx) / sq : 0.0;
    if (lane == 0) {
      sh.m[j] = m, sh.s[j] = sum, sh.mq[j] = mq, sh.sq[j] = sq, sh.lx[j] = lx;
      sh.ok[j] = x >= 0 && (double)u * q < p;
    }
  }
  __syncthreads();
  const unsigned long long no = __ballot(lane >= n - 1 || !sh.ok[min(lane, n - 1)]);
  const int taken = __builtin_ctzll(no);  // n - 1 <= 63
  const bool refused = taken < n - 1;
  if (tid < T && tid != taken) a.ids[(size_t)s * T + tid] = tid < taken ? sh.x[tid] : -1;
  if (tid == 0) a.accepted[s] = taken;
  int token;
  if (GREEDY) {
    token = sh.top[taken];
  } else {
    const bool rest = refused && a.draft_logits && sh.s[taken] > 0.0;
    if (a.draft_logits && tid == 0)
      w.dec[s] = Decision{1.0 / sh.s[taken], sh.sq[taken] > 0.0 ? 1.0 / sh.sq[taken] : 0.0, sh.m[taken], sh.mq[taken],
                          s * T + taken, rest ? s * (T - 1) + taken : -1};
    if (rest) return;
    const float* l = a.logits + ((size_t)s * T + taken) * a.vocab;
    const Weights of(sh.m[taken], a.scale);
    const float u = a.uniforms[s * T + T - 1];
    int x = refused && !a.draft_logits ? sh.x[taken] : -1;  // a certain draft's residual is p without it
    auto at = [&](int i, double* v) {
      const vf4 y = row_quad(l, i, a.vocab);
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = i + e == x ? 0.0 : of.of(y[e]);
    };
    const bool mine = wave == taken % kVW;  // this wave has the row's sums, if no row came after it
    double v[kVRow];
    if (mine) {
      if (n > kVW) {
        float dm;
        double ds;
        row_load(a, w, (size_t)s * a.rows + taken, rp);
        row_scale(a, rp, &dm, &ds);
      }
      bool much = false;
#pragma unroll
      for (int k = 0; k < kVRow; k++) {
        v[k] = rp.sum[k];
        if (x >= 0 && lane + 64 * k == x / kVChunk) {  // less the draft's term, as it was added
          const Weights c(rp.max[k], a.scale);
          const double left = rp.raw[k] - c.of(sh.lx[taken]);
          much = !(left >= rp.raw[k] * 0x1p-16);
          v[k] = left * of.of(rp.max[k]);
        }
      }
      const bool again = __ballot(much) != 0;
      if (!again) find_chunk(v, u, sh);
      if (lane == 0) sh.again = again;
    }
    __syncthreads();
    if (sh.again) {  // the difference has lost what is left beside a likely draft: its chunk's sum without it
      double y[4];
      at(x / kVChunk * kVChunk + 4 * tid, y);
      const double without = block_sum_f64((y[0] + y[1]) + (y[2] + y[3]), sh);
      if (mine) {
#pragma unroll
        for (int k = 0; k < kVRow; k++)
          if (lane + 64 * k == x / kVChunk) v[k] = without;
        find_chunk(v, u, sh);
      }
      __syncthreads();
    }
    if (sh.chunk < 0 && x >= 0) {  // nothing beside the draft: p itself
      x = -1;
      __syncthreads();
      if (mine) find_chunk(rp.sum, u, sh);
      __syncthreads();
    }
    token = sh.chunk < 0 ? -1 : find_entry(a, at, sh);
  }
  if (tid == 0) a.ids[(size_t)s * T + taken] = token;
}

// Where the rows that are there lie, a wave's own view: 64 sequences at a time, a
// lane each, their rows (targets, then drafts) numbered through.
struct RowWalk {
  int s0, before, rows, incl, total;  // rows before the 64, this lane's, theirs up to this lane's, all theirs
  __device__ __forceinline__ void group(const VerifyArgs& a, int s) {
    const int l = s + (threadIdx.x & 63), n = l < a.seqs ? row_count(a, l) : 0;
    s0 = s;
    rows = n < 1 ? 0 : a.rows > a.tokens ? 2 * n - 1 : n;
    incl = rows;
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x111, 0xF, 0xF, false);  // as wave_scan_f64
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x112, 0xF, 0xF, false);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x114, 0xF, 0xF, false);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x118, 0xF, 0xF, false);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x142, 0xA, 0xF, false);
    incl += __builtin_amdgcn_update_dpp(0, incl, 0x143, 0xC, 0xF, false);
    total = __builtin_amdgcn_readlane(incl, 63);
  }
  // All rows; the walk then stands at the first 64 sequences.
  __device__ __forceinline__ int start(const VerifyArgs& a) {
    int all = 0;
    for (int s = 0; s < a.seqs; s += 64) {
      group(a, s);
      all += total;
    }
    if (a.seqs > 64) group(a, 0);
    before = 0;
    return all;
  }
  // The lane of the sequence that holds a row, no earlier than the last one asked for.
  __device__ __forceinline__ int seek(const VerifyArgs& a, int row) {
    while (row >= before + total) {
      const int t = total;
      group(a, s0 + 64);
      before += t;
    }
    return __builtin_popcountll(__ballot(before + incl <= row));
  }
};

// All chunks of all rows that are there, shared out evenly: a block takes a run of
// them, its waves in turn.  Having published its results it counts them for their
// sequences; the block that completes a sequence decides it (every value of the
// sequence has then been performed) and clears the count.
template <bool GREEDY>
__global__ __launch_bounds__(kVT, 4) void verify_kernel(VerifyArgs a) {
  __shared__ VerifyShared sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), T = a.tokens;
  const VerifyWork w = verify_work(a);
  RowWalk walk;
  const int cells = walk.start(a) * a.chunks, run = (cells + gridDim.x - 1) / gridDim.x;
  const int c0 = min((int)blockIdx.x * run, cells), c1 = min(c0 + run, cells);
  if (c0 >= c1) return;
  struct Place {
    int s, r, c;  // sequence, row (drafts after the targets), chunk
  };
  auto place = [&](int cell) {
    const int row = cell / a.chunks, l = walk.seek(a, row), rows = __builtin_amdgcn_readlane(walk.rows, l);
    const int k = row - walk.before - (__builtin_amdgcn_readlane(walk.incl, l) - rows);
    const int n = a.rows > T ? (rows + 1) / 2 : rows;
    return Place{walk.s0 + l, k < n ? k : T + k - n, cell - row * a.chunks};
  };
  auto fetch = [&](int cell, vf4* v) {  // past the run's end: its last chunk
    const Place p = place(min(cell, c1 - 1));
    load_quads<kVQuads>(p.r < T ? a.logits + ((size_t)p.s * T + p.r) * a.vocab
                       : a.draft_logits + ((size_t)p.s * (T - 1) + p.r - T) * a.vocab,
               p.c * kVChunk, a.vocab, v);
    return p;
  };
  auto reduce = [&](const Place& p, vf4* v) {
    const size_t at = ((size_t)p.s * a.rows + p.r) * a.chunks + p.c;
    if (GREEDY) {
      const int i0 = p.c * kVChunk + 4 * lane;
      float best = kLowest;
      int id = 0;
#pragma unroll
      for (int k = 0; k < kVQuads; k++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (v[k][e] > best) best = v[k][e], id = i0 + 256 * k + e;  // ids ascend: the lower one stays
      const unsigned long long key = wave_max_key(best > kLowest ? greedy_key(best, id) : 0ull);
      if (lane == 0) publish(w.cell + at, key);
      return;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVQuads; k++)
#pragma unroll
      for (int e = 0; e < 4; e++) mx = fmaxf(mx, v[k][e]);
    mx = wave_max(mx);
    if (!(mx > kLowest)) mx = -INFINITY;  // no entry
    const Weights of(mx, a.scale);
    double sum = 0.0;
    if (of.plain) {
#pragma unroll
      for (int k = 0; k < kVQuads; k++) {
#pragma unroll
        for (int e = 0; e < 4; e++) sum += of.series(v[k][e]);
        __builtin_amdgcn_sched_barrier(0);  // four series at once: 32 would take twice the registers
      }
    } else {
#pragma unroll
      for (int k = 0; k < kVQuads; k++) {
#pragma unroll
        for (int e = 0; e < 4; e++) sum += of.of(v[k][e]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) {
      publish(w.cell + at, (unsigned long long)__double_as_longlong(sum));
      publish(w.max + at, mx);
    }
  };
  // one chunk in work, the next in flight
  if (c0 + wave < c1) {
    vf4 x[kVQuads], y[kVQuads];
    Place px = fetch(c0 + wave, x), py;
    for (int c = c0 + wave;; c += 2 * kVW) {
      py = fetch(c + kVW, y);
      reduce(px, x);
      if (c + kVW >= c1) break;
      px = fetch(c + 2 * kVW, x);
      reduce(py, y);
      if (c + 2 * kVW >= c1) break;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's results are performed
  __syncthreads();                                  // and every wave's
  if (a.seqs > 64) {
    walk.group(a, 0);
    walk.before = 0;
    walk.seek(a, c0 / a.chunks);
  }
  while (true) {  // 64 sequences at a time
    if (wave == 0) {
      const int s = walk.s0 + lane, end = (walk.before + walk.incl) * a.chunks, all = walk.rows * a.chunks;
      const int mine = min(c1, end) - max(c0, end - all);
      bool done = false;
      if (mine > 0) {
        const unsigned count =
            __hip_atomic_fetch_add(a.arrived + s, (unsigned)mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        done = (int)count + mine == all;
        if (done) __hip_atomic_store(a.arrived + s, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      const unsigned long long which = __ballot(done);
      if (lane == 0) sh.done = which;
    }
    __syncthreads();
    for (unsigned long long left = sh.done; left; left &= left - 1)
      decide<GREEDY>(a, walk.s0 + __builtin_ctzll(left), sh);
    const int rows = walk.before + walk.total;
    if (rows * a.chunks >= c1) break;
    walk.seek(a, rows);
    __syncthreads();  // sh.done has been read
  }
}

// kRestWaves waves per chunk of every sequence whose token is still to be drawn: the
// chunk's sum of max(p - q, 0); the last of a sequence's `per` blocks draws.  Two
// share a chunk, as only the refused sequences' blocks have work (32 x 5 over 151936
// tokens with one, two and four 55.6, 55.1 and 56.0 us a call).
__global__ __launch_bounds__(kVT) void verify_rest_kernel(VerifyArgs a, int per) {
  __shared__ VerifyShared sh;
  constexpr int Q = kVQuads / kRestWaves;
  const VerifyWork w = verify_work(a);
  const int s = blockIdx.x / per, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = row_count(a, s);
  const Decision d = w.dec[s];
  if (n < 1 || d.draft < 0) return;
  const float* l = a.logits + (size_t)d.row * a.vocab;
  const float* q = a.draft_logits + (size_t)d.draft * a.vocab;
  const float u = a.uniforms[s * a.tokens + a.tokens - 1];
  const Weights lw(d.m, a.scale), qw(d.mq, a.scale);
  auto residual = [&](float x, float y) { return fmax(lw.of(x) * d.s - (d.sq > 0.0 ? qw.of(y) * d.sq : 0.0), 0.0); };
  const int c0 = blockIdx.x % per * (kVW / kRestWaves), i0 = c0 * kVChunk + wave * (256 * Q);
  double sum = 0.0;
  if (i0 < a.vocab) {
    vf4 x[Q], y[Q];
    load_quads<Q>(l, i0, a.vocab, x);
    load_quads<Q>(q, i0, a.vocab, y);
    if (lw.plain && qw.plain && d.sq > 0.0) {
#pragma unroll
      for (int k = 0; k < Q; k++) {
#pragma unroll
        for (int e = 0; e < 4; e++) sum += fmax(lw.series(x[k][e]) * d.s - qw.series(y[k][e]) * d.sq, 0.0);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int k = 0; k < Q; k++) {
#pragma unroll
        for (int e = 0; e < 4; e++) sum += residual(x[k][e], y[k][e]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    sum = wave_sum_f64(sum);
  }
  if (lane == 0) sh.red[wave] = sum;
  __syncthreads();
  if (wave == 0) {
    if (lane < kVW / kRestWaves && c0 + lane < a.chunks) {
      double v = 0.0;
#pragma unroll
      for (int k = 0; k < kRestWaves; k++) v += sh.red[lane * kRestWaves + k];
      publish(w.rest + (size_t)s * a.chunks + c0 + lane, v);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the block's sums are performed
    if (lane == 0) sh.before = __hip_atomic_fetch_add(a.arrived + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (sh.before != (unsigned)per - 1) return;
  if (threadIdx.x == 0) __hip_atomic_store(a.arrived + s, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (threadIdx.x < 64) {
    double v[kVRow];
#pragma unroll
    for (int i = 0; i < kVRow; i++)
      v[i] = lane + 64 * i < a.chunks ? published(w.rest + (size_t)s * a.chunks + lane + 64 * i) : 0.0;
    find_chunk(v, u, sh);
  }
  __syncthreads();
  const bool same = sh.chunk < 0;  // p and q are: p itself
  if (same) {
    __syncthreads();
    if (threadIdx.x < 64) {
      RowSums r;
      float dm;
      double ds;
      row_load(a, w, (size_t)s * a.rows + d.row % a.tokens, r);
      row_scale(a, r, &dm, &ds);
      find_chunk(r.sum, u, sh);
    }
    __syncthreads();
  }
  const int token = find_entry(a, [&](int i, double* v) {
    const vf4 y = row_quad(l, i, a.vocab), z = row_quad(q, i, a.vocab);
#pragma unroll
    for (int f = 0; f < 4; f++) v[f] = same ? lw.of(y[f]) : residual(y[f], z[f]);
  }, sh);
  if (threadIdx.x == 0) a.ids[d.row] = token;
}

}  // namespace

size_t verify_plan(VerifyArgs& a) {
  a.rows = a.draft_logits && a.scale > 0.0 ? 2 * a.tokens - 1 : a.tokens;
  a.chunks = (a.vocab + kVChunk - 1) / kVChunk;
  const size_t seqs = std::min(a.seqs, kVerifyCounters), cells = seqs * a.rows * a.chunks;
  return cells * (sizeof(unsigned long long) + sizeof(float)) + seqs * (a.chunks * sizeof(double) + sizeof(Decision));
}

// kVerifyCounters sequences at a time.  Two blocks a CU are resident: several
// chunks a wave from there on, so that the next one is in flight during a chunk's
// sum and a block waits for its counts only once.  Up to four chunks a CU: four a
// block, a SIMD each (64 x 1 over 32000 tokens 14.6 -> 12.7 us).
//
// What bounds it: the logits' bytes for many rows (32 x 5 over 151936 tokens with draft
// logits 43 us for 135 MB of live rows and 13 for the second launch; each entry's
// term takes 17 64-bit operations beside 4 bytes), for few a chain of a dozen
// memory round trips and barriers in one block (1 x 5 over 128256: 11.3 us, of which
// 3.7 until the sums are there, 3.5 to publish and count them, 5 to decide and draw).
void launch_verify(const VerifyArgs& all, int cus, hipStream_t st) {
  for (int s0 = 0; s0 < all.seqs; s0 += kVerifyCounters) {
    VerifyArgs a = all;
    const size_t row = (size_t)s0 * a.tokens, draft = (size_t)s0 * (a.tokens - 1);
    a.seqs = std::min(all.seqs - s0, kVerifyCounters);
    a.logits += row * a.vocab;
    if (a.draft_logits) a.draft_logits += draft * a.vocab;
    if (a.drafts) a.drafts += draft;
    if (a.counts) a.counts += s0;
    if (a.uniforms) a.uniforms += row;
    a.accepted += s0;
    a.ids += row;
    const int64_t cells = (int64_t)a.seqs * a.rows * a.chunks;
    const int per_block = cells <= 4 * cus ? kVW / 2 : kVW;
    const dim3 grid((unsigned)std::min<int64_t>(2 * cus, (cells + per_block - 1) / per_block)), block(kVT);
    if (a.scale == 0.0) {
      hipLaunchKernelGGL(verify_kernel<true>, grid, block, 0, st, a);
      continue;
    }
    hipLaunchKernelGGL(verify_kernel<false>, grid, block, 0, st, a);
    const int per = (a.chunks * kRestWaves + kVW - 1) / kVW;
    if (a.rows > a.tokens) hipLaunchKernelGGL(verify_rest_kernel, dim3((unsigned)(a.seqs * per)), block, 0, st, a, per);
  }
}

}  // namespace tlm
