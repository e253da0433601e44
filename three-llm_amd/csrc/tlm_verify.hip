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
#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "tlm_device.h"

namespace tlm {
namespace {

constexpr int kVT = 256;  // threads per block
constexpr int kVE = 8;    // elements of a row a thread takes at a time
constexpr int kVTile = kVT * kVE;

// What the steps pass on: per row of target logits, then of draft logits, and
// chunk of the vocabulary the maximum and the sum of exp((l - max) / T), or the
// greedy key; per sequence the decision and the chunks' sums of max(p - q, 0).
struct Decision {
  double m, s, mq, sq;  // of the row the token is drawn from: maximum and sum, the draft's
  int row;              // target row (of all), or -1: nothing is left to draw
  int draft;            // draft row, or -1
};
struct VerifyWork {
  double* sum;
  float* max;
  unsigned long long* key;
  double* rest;
  Decision* dec;
};
__host__ __device__ inline VerifyWork verify_work(const VerifyArgs& a) {
  const size_t rows = (size_t)a.seqs * (2 * a.tokens - 1), cells = rows * a.chunks;
  VerifyWork w;
  w.sum = static_cast<double*>(a.work);
  w.key = reinterpret_cast<unsigned long long*>(w.sum);  // greedy has no sums
  w.rest = w.sum + cells;
  w.dec = reinterpret_cast<Decision*>(w.rest + (size_t)a.seqs * a.chunks);
  w.max = reinterpret_cast<float*>(w.dec + a.seqs);
  return w;
}

// Entries at or below LOWEST_FLOAT (-inf and NaN included) never take part.
__device__ __forceinline__ double weight(float l, double m, double inv_temp) {
  if (!(l > kLowest)) return 0.0;
  return l == m ? 1.0 : exp(((double)l - m) * inv_temp);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 1; o < 64; o *= 2) v += __shfl_xor(v, o);
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
__device__ double block_sum_f64(double v, double* scratch) {  // scratch: a double per wave
  v = wave_sum_f64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  double r = 0.0;
  for (int i = 0; i < kVT / 64; i++) r += scratch[i];
  return r;
}

__device__ __forceinline__ int row_count(const VerifyArgs& a, int s) {
  return a.counts ? min(a.counts[s], a.tokens) : a.tokens;
}

// A block per chunk of a row.
template <bool GREEDY>
__global__ __launch_bounds__(kVT) void verify_stats_kernel(VerifyArgs a) {
  __shared__ double red[kVT / 64];
  __shared__ float redm[kVT / 64];
  __shared__ unsigned long long redk[kVT / 64];
  const int row = blockIdx.x / a.chunks, c = blockIdx.x % a.chunks, targets = a.seqs * a.tokens;
  const bool target = row < targets;
  const int s = target ? row / a.tokens : (row - targets) / (a.tokens - 1);
  const int j = target ? row % a.tokens : (row - targets) % (a.tokens - 1);
  if (j >= row_count(a, s) - (target ? 0 : 1)) return;
  const float* x = target ? a.logits + (size_t)row * a.vocab : a.draft_logits + (size_t)(row - targets) * a.vocab;
  const int i0 = c * a.chunk, i1 = min(i0 + a.chunk, a.vocab), tid = threadIdx.x;
  const VerifyWork w = verify_work(a);
  const size_t cell = (size_t)row * a.chunks + c;
  if (GREEDY) {
    unsigned long long best = 0;
    for (int i = i0 + tid; i < i1; i += kVT)
      if (x[i] > kLowest) {
        const unsigned long long k = greedy_key(x[i], i);
        best = k > best ? k : best;
      }
    best = wave_max_key(best);
    if ((tid & 63) == 0) redk[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kVT / 64; i++) best = redk[i] > best ? redk[i] : best;
      w.key[cell] = best;
    }
    return;
  }
  float m = -INFINITY;
  for (int i = i0 + tid; i < i1; i += kVT)
    if (x[i] > kLowest) m = fmaxf(m, x[i]);
  m = wave_max(m);
  if ((tid & 63) == 0) redm[tid >> 6] = m;
  __syncthreads();
  for (int i = 0; i < kVT / 64; i++) m = fmaxf(m, redm[i]);
  double sum = 0.0;
  for (int i = i0 + tid; i < i1; i += kVT) sum += weight(x[i], (double)m, a.inv_temp);
  sum = block_sum_f64(sum, red);
  if (tid == 0) {
    w.max[cell] = m;
    w.sum[cell] = sum;
  }
}

// A chunk's sum relative to the row's maximum m (a chunk without entries: 0).
__device__ __forceinline__ double chunk_sum(const VerifyArgs& a, const VerifyWork& w, size_t cell, double m) {
  const double s = w.sum[cell];
  const float cm = w.max[cell];
  return s > 0.0 ? s * (cm == m ? 1.0 : exp(((double)cm - m) * a.inv_temp)) : 0.0;
}

// Maximum and sum of a row, in every lane of the wave.
__device__ void row_stats(const VerifyArgs& a, const VerifyWork& w, size_t row, double* m, double* s) {
  const int lane = threadIdx.x & 63;
  float mx = -INFINITY;
  for (int c = lane; c < a.chunks; c += 64) mx = fmaxf(mx, w.max[row * a.chunks + c]);
  mx = wave_max(mx);
  double sum = 0.0;
  for (int c = lane; c < a.chunks; c += 64) sum += chunk_sum(a, w, row * a.chunks + c, (double)mx);
  *m = (double)mx;
  *s = wave_sum_f64(sum);
}

// The block finds the lowest index whose running sum passes u times the whole:
// `sums(c)` the chunks' sums, `at(i)` an entry's weight.  Rounding may leave the
// last border at u: then it is the last index with a weight.  -1: all are zero.
template <typename Sums, typename At>
__device__ int draw(const VerifyArgs& a, float u, Sums sums, At at, double* red, int* pick) {
  const int tid = threadIdx.x, lane = tid & 63;
  // every wave: the whole, then the chunk
  double total = 0.0;
  for (int c = lane; c < a.chunks; c += 64) total += sums(c);
  total = wave_sum_f64(total);
  if (!(total > 0.0)) return -1;
  const double border = (double)u * total;
  double before = 0.0, found_before = 0.0;
  int chunk = -1, last = -1;
  double last_before = 0.0;
  for (int c0 = 0; c0 < a.chunks && chunk < 0; c0 += 64) {
    const double v = c0 + lane < a.chunks ? sums(c0 + lane) : 0.0;
    double run = v;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const double y = __shfl_up(run, o);
      if (lane >= o) run += y;
    }
    const unsigned long long over = __ballot(v > 0.0 && before + run > border), some = __ballot(v > 0.0);
    const double excl = before + (run - v);
    if (over) {
      const int l = __ffsll(over) - 1;
      chunk = c0 + l;
      found_before = __shfl(excl, l);
    } else if (some) {
      const int l = 63 - __clzll(some);
      last = c0 + l;
      last_before = __shfl(excl, l);
    }
    before += __shfl(run, 63);
  }
  if (chunk < 0) {
    chunk = last;
    found_before = last_before;
  }
  // the block: kVE entries a thread, in order
  const int i1 = min((chunk + 1) * a.chunk, a.vocab);
  double run = found_before;
  int best = -1;
  for (int i0 = chunk * a.chunk; i0 < i1; i0 += kVTile) {
    double v[kVE], mine = 0.0;
    int mlast = -1;
#pragma unroll
    for (int e = 0; e < kVE; e++) {
      const int i = i0 + tid * kVE + e;
      v[e] = i < i1 ? at(i) : 0.0;
      mine += v[e];
      if (v[e] > 0.0) mlast = i;
    }
    double incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const double y = __shfl_up(incl, o);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 63) red[tid >> 6] = incl;
    if (tid == 0) pick[0] = 0x7fffffff, pick[1] = -1;
    __syncthreads();
    double c = run + (incl - mine);
    for (int k = 0; k < tid >> 6; k++) c += red[k];
    int hit = 0x7fffffff;
#pragma unroll
    for (int e = kVE - 1; e >= 0; e--) {
      double upto = c;
      for (int f = 0; f <= e; f++) upto += v[f];
      if (v[e] > 0.0 && upto > border) hit = i0 + tid * kVE + e;
    }
    if (hit != 0x7fffffff) atomicMin(&pick[0], hit);
    if (mlast >= 0) atomicMax(&pick[1], mlast);
    __syncthreads();
    if (pick[0] != 0x7fffffff) return pick[0];
    if (pick[1] >= 0) best = pick[1];
    for (int k = 0; k < kVT / 64; k++) run += red[k];
  }
  return best;
}

// A block per sequence: which drafts stand, and the token after them where no
// draft logits are to be subtracted.
template <bool GREEDY>
__global__ __launch_bounds__(kVT) void verify_decide_kernel(VerifyArgs a) {
  __shared__ double red[kVT / 64], rm[kVerifyMaxTokens], rs[kVerifyMaxTokens], qm[kVerifyMaxTokens],
      qs[kVerifyMaxTokens];
  __shared__ int ok[kVerifyMaxTokens], top[kVerifyMaxTokens], pick[2];
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63, T = a.tokens, targets = a.seqs * T;
  const VerifyWork w = verify_work(a);
  const int n = row_count(a, s);
  if (n < 1) {  // idle: its results stay as they are
    if (!GREEDY && tid == 0) w.dec[s].row = -1, w.dec[s].draft = -1;
    return;
  }
  for (int j = tid >> 6; j < n; j += kVT / 64) {
    const int row = s * T + j, x = j < n - 1 ? a.drafts[s * (T - 1) + j] : -1;
    const bool in = x >= 0 && x < a.vocab;
    if (GREEDY) {
      unsigned long long k = 0;
      for (int c = lane; c < a.chunks; c += 64) {
        const unsigned long long y = w.key[(size_t)row * a.chunks + c];
        k = y > k ? y : k;
      }
      k = wave_max_key(k);
      if (lane == 0) {
        top[j] = k ? greedy_key_id(k) : -1;
        ok[j] = in && x == top[j];
      }
      continue;
    }
    double m, sum, dm = 0.0, ds = 0.0;
    row_stats(a, w, row, &m, &sum);
    if (a.draft_logits && j < n - 1) row_stats(a, w, targets + s * (T - 1) + j, &dm, &ds);
    if (lane == 0) {
      rm[j] = m, rs[j] = sum, qm[j] = dm, qs[j] = ds;
      double p = 0.0, q = 1.0;
      if (in && sum > 0.0) p = weight(a.logits[(size_t)row * a.vocab + x], m, a.inv_temp) / sum;
      if (in && a.draft_logits)
        q = ds > 0.0 ? weight(a.draft_logits[((size_t)s * (T - 1) + j) * a.vocab + x], dm, a.inv_temp) / ds : 0.0;
      ok[j] = in && (double)a.uniforms[s * T + j] * q < p;
    }
  }
  __syncthreads();
  int taken = 0;
  while (taken < n - 1 && ok[taken]) taken++;
  const bool refused = taken < n - 1;
  for (int j = tid; j < T; j += kVT)
    if (j != taken) a.ids[(size_t)s * T + j] = j < taken ? a.drafts[s * (T - 1) + j] : -1;
  if (tid == 0) a.accepted[s] = taken;
  int token;
  if (GREEDY) {
    token = top[taken];
  } else {
    const int row = s * T + taken;
    const double m = rm[taken];
    const bool split = refused && a.draft_logits && rs[taken] > 0.0;
    if (tid == 0) w.dec[s] = Decision{m, rs[taken], qm[taken], qs[taken], row, split ? s * (T - 1) + taken : -1};
    if (split) return;
    const float* l = a.logits + (size_t)row * a.vocab;
    const float u = a.uniforms[s * T + T - 1];
    // a certain draft's residual is p without it
    const int x = refused && !a.draft_logits ? a.drafts[s * (T - 1) + taken] : -1;
    const int cx = x >= 0 && x < a.vocab ? x / a.chunk : -1;
    double without = 0.0;
    if (cx >= 0) {  // its chunk again, as a difference would lose what is left beside a likely draft
      for (int i = cx * a.chunk + tid; i < min((cx + 1) * a.chunk, a.vocab); i += kVT)
        without += i == x ? 0.0 : weight(l[i], m, a.inv_temp);
      without = block_sum_f64(without, red);
    }
    token = draw(a, u, [&](int c) { return c == cx ? without : chunk_sum(a, w, (size_t)row * a.chunks + c, m); },
                 [&](int i) { return i == x ? 0.0 : weight(l[i], m, a.inv_temp); }, red, pick);
    if (token < 0 && x >= 0) {  // nothing beside the draft: p itself
      __syncthreads();
      token = draw(a, u, [&](int c) { return chunk_sum(a, w, (size_t)row * a.chunks + c, m); },
                   [&](int i) { return weight(l[i], m, a.inv_temp); }, red, pick);
    }
  }
  if (tid == 0) a.ids[(size_t)s * T + taken] = token;
}

__device__ __forceinline__ double residual(const VerifyArgs& a, const Decision& d, const float* l, const float* q, int i) {
  const double p = weight(l[i], d.m, a.inv_temp) / d.s;
  const double y = d.sq > 0.0 ? weight(q[i], d.mq, a.inv_temp) / d.sq : 0.0;
  return p > y ? p - y : 0.0;
}

// A block per chunk and sequence: the chunk's sum of max(p - q, 0).
__global__ __launch_bounds__(kVT) void verify_rest_kernel(VerifyArgs a) {
  __shared__ double red[kVT / 64];
  const int s = blockIdx.x / a.chunks, c = blockIdx.x % a.chunks;
  const VerifyWork w = verify_work(a);
  const Decision d = w.dec[s];
  if (d.draft < 0) return;
  const float* l = a.logits + (size_t)d.row * a.vocab;
  const float* q = a.draft_logits + (size_t)d.draft * a.vocab;
  double sum = 0.0;
  for (int i = c * a.chunk + threadIdx.x; i < min((c + 1) * a.chunk, a.vocab); i += kVT) sum += residual(a, d, l, q, i);
  sum = block_sum_f64(sum, red);
  if (threadIdx.x == 0) w.rest[(size_t)s * a.chunks + c] = sum;
}

// A block per sequence: the token from those sums.
__global__ __launch_bounds__(kVT) void verify_draw_kernel(VerifyArgs a) {
  __shared__ double red[kVT / 64];
  __shared__ int pick[2];
  const int s = blockIdx.x;
  const VerifyWork w = verify_work(a);
  const Decision d = w.dec[s];
  if (d.draft < 0) return;
  const float* l = a.logits + (size_t)d.row * a.vocab;
  const float* q = a.draft_logits + (size_t)d.draft * a.vocab;
  const float u = a.uniforms[s * a.tokens + a.tokens - 1];
  int token = draw(a, u, [&](int c) { return w.rest[(size_t)s * a.chunks + c]; },
                   [&](int i) { return residual(a, d, l, q, i); }, red, pick);
  if (token < 0) {  // p and q are the same: p itself
    __syncthreads();
    token = draw(a, u, [&](int c) { return chunk_sum(a, w, (size_t)d.row * a.chunks + c, d.m); },
                 [&](int i) { return weight(l[i], d.m, a.inv_temp); }, red, pick);
  }
  if (threadIdx.x == 0) a.ids[d.row] = token;
}

}  // namespace

static size_t work_bytes(const VerifyArgs& a) {
  const size_t cells = (size_t)a.seqs * (2 * a.tokens - 1) * a.chunks;
  return cells * (sizeof(double) + sizeof(float)) + (size_t)a.seqs * (a.chunks * sizeof(double) + sizeof(Decision));
}

void verify_plan(VerifyArgs& a, int cus, size_t most) {
  const int64_t rows = (int64_t)a.seqs * a.tokens;
  int64_t chunk = kVTile;
  while (chunk < 4 * kVTile && rows * (a.vocab / chunk) > 8 * cus) chunk *= 2;
  for (;; chunk *= 2) {
    a.chunk = (int)std::min<int64_t>(chunk, INT_MAX);
    a.chunks = (int)((a.vocab + (int64_t)a.chunk - 1) / a.chunk);
    if (work_bytes(a) <= most || a.chunks == 1) return;
  }
}

void launch_verify(const VerifyArgs& a, hipStream_t st) {
  const bool greedy = a.inv_temp == 0.0;
  const bool model = !greedy && a.draft_logits && a.tokens > 1;
  const int rows = a.seqs * (model ? 2 * a.tokens - 1 : a.tokens);
  const dim3 grid((unsigned)(rows * a.chunks)), seqs((unsigned)a.seqs), block(kVT);
  if (greedy) {
    hipLaunchKernelGGL(verify_stats_kernel<true>, grid, block, 0, st, a);
    hipLaunchKernelGGL(verify_decide_kernel<true>, seqs, block, 0, st, a);
    return;
  }
  hipLaunchKernelGGL(verify_stats_kernel<false>, grid, block, 0, st, a);
  hipLaunchKernelGGL(verify_decide_kernel<false>, seqs, block, 0, st, a);
  if (!model) return;
  hipLaunchKernelGGL(verify_rest_kernel, dim3((unsigned)(a.seqs * a.chunks)), block, 0, st, a);
  hipLaunchKernelGGL(verify_draw_kernel, seqs, block, 0, st, a);
}

}  // namespace tlm
