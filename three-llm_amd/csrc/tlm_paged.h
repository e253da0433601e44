// Paged key-value caches: where an element lies, and which rows of a batch are
// there.  Host and device share these, so the host tests them.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __HIP__
#define TLM_HD __host__ __device__ __forceinline__
#else
#define TLM_HD inline
#endif

namespace tlm {

// A page holds page_tokens tokens of every kv head, [kv head][page_tokens x D],
// in 16-byte pieces of E elements (8 of fp16, 4 of fp32) that lie in the order
// in which the matrix cores' lanes take them: a wave's load of 64 pieces is 1 KB
// in a row and an operand register, without a pass through LDS.
//   K: operand row = token, contraction = dim:
//      [token / 16][dim / E][token % 16][dim % E]
//   V: operand row = dim, contraction = token, in the order in which the scores
//      leave the matrix cores (lane group q holds tokens 4 q .. 4 q + 3 of each 16):
//      [token / (4 E)][dim / 16][token % 16 / 4][dim % 16][token % (4 E) / 16][token % 4]
// token: position within the page.  The offsets are within one head of a page.
TLM_HD int paged_k_at(int token, int dim, int D, int E) {
  return ((token >> 4) * (D / E) + dim / E) * (16 * E) + (token & 15) * E + dim % E;
}
TLM_HD int paged_v_at(int token, int dim, int D, int E) {
  const int g = 4 * E;
  return ((token / g) * (D >> 4) + (dim >> 4)) * (64 * E) + (((token & 15) >> 2) * 16 + (dim & 15)) * E +
         (token % g >> 4) * 4 + (token & 3);
}

// Caches of 8-bit values (e4m3 codes): a page is [kv head][page_tokens x D] codes,
// then fp32 scales [kv head][page_tokens / 32], up to a multiple of 128 bytes, so that
// a page is whole by itself and its codes start on a cache line.  Codes lie in the
// order of the operands again, 32 tokens by 32 dims a kilobyte: a lane's 16 bytes are
// the operands of two 16-row products.
//   K: [token / 32][dim / 32][dim % 32 / 8][token % 16][token % 32 / 16][dim % 8]
//   V: [token / 32][dim / 32][token % 16 / 4][dim % 16][dim % 32 / 16][token % 32 / 16][token % 4]
constexpr int kPagedScaleTokens = 32;  // tokens of a kv head that share a scale
TLM_HD int paged8_k_at(int token, int dim, int D) {
  return ((token >> 5) * (D >> 5) + (dim >> 5)) * 1024 + ((dim & 31) >> 3) * 256 + (token & 15) * 16 +
         ((token & 31) >> 4) * 8 + (dim & 7);
}
TLM_HD int paged8_v_at(int token, int dim, int D) {
  return ((token >> 5) * (D >> 5) + (dim >> 5)) * 1024 + ((token & 15) >> 2) * 256 + (dim & 15) * 16 +
         ((dim & 31) >> 4) * 8 + ((token & 31) >> 4) * 4 + (token & 3);
}
TLM_HD size_t paged8_codes(int heads, int page_shift, int D) { return (size_t)heads * ((size_t)D << page_shift); }
TLM_HD size_t paged8_page(int heads, int page_shift, int D) {
  return paged8_codes(heads, page_shift, D) + (((size_t)heads * 4 << (page_shift - 5)) + 127) / 128 * 128;
}
// Where the scale of a token of a page's head lies, in bytes from the page's start.
TLM_HD size_t paged8_scale_at(int head, int heads, int token, int page_shift, int D) {
  return paged8_codes(heads, page_shift, D) + 4 * (((size_t)head << (page_shift - 5)) + (token >> 5));
}

// A scale is 2^e, the least that takes magnitudes up to `top` (the bits of a finite
// fp32 >= 0) to at most 448 = 1.75 * 2^8, the largest code: e from -32 to 31.
constexpr int kPagedScaleMin = -32, kPagedScaleMax = 31;
TLM_HD int paged8_exponent(uint32_t top) {
  const int e = (int)((top + 0x1FFFFFu) >> 23) - 127 - 8;  // the next power where the mantissa is above 1.75
  return e < kPagedScaleMin ? kPagedScaleMin : e > kPagedScaleMax ? kPagedScaleMax : e;
}
// The exponent of a scale that lies in a pool (the kernels take no other scales).
TLM_HD int paged8_exponent_of(uint32_t scale) {
  const int e = (int)(scale >> 23 & 0xFF) - 127;
  return e < kPagedScaleMin ? kPagedScaleMin : e > kPagedScaleMax ? kPagedScaleMax : e;
}

// The first element of a page's head in its pool.
TLM_HD size_t paged_head_at(int page, int head, int heads, int page_shift, int D) {
  return ((size_t)page * heads + head) * ((size_t)D << page_shift);
}

// Positions that a sequence can have: its table's pages, its RoPE table's rows.
TLM_HD int paged_limit(int max_tokens, int width, int page_shift) {
  const int64_t held = (int64_t)width << page_shift;
  return held < max_tokens ? (int)held : max_tokens;
}

// Rows of a sequence that a call computes: none of an idle one (start < 0 or
// count < 1), else `count` of its `tokens` rows as far as its positions are
// below `limit`; *bad: some row was left out for the limit or there are more
// than `tokens`.
TLM_HD int paged_rows(int start, int count, int tokens, int limit, bool* bad) {
  *bad = false;
  if (start < 0 || count < 1) return 0;
  const int want = count < tokens ? count : tokens;
  const int room = start < limit ? limit - start : 0;
  const int rows = want < room ? want : room;
  *bad = count > tokens || rows < want;
  return rows;
}

// The pages that a sequence with rows at start, start + 1, ... has in use: those of
// its sinks [0, sink), then [first, end) from its first row's window on.
struct PagedUse {
  int sink, first, end;
};
TLM_HD PagedUse paged_use(int start, int rows, int window, int sinks, int page_shift) {
  PagedUse u;
  const int from = window > 0 && start >= window ? start - window + 1 : 0;
  u.end = (int)(((int64_t)start + rows + (1 << page_shift) - 1) >> page_shift);
  u.first = from >> page_shift;
  if (u.first > u.end) u.first = u.end;
  u.sink = (int)(((int64_t)sinks + (1 << page_shift) - 1) >> page_shift);
  if (window <= 0) u.sink = 0;
  if (u.sink > u.first) u.sink = u.first;
  return u;
}

// The page of a position in its sequence's table, or -1 where the entry is none
// of the pool's.
TLM_HD int paged_page(const int32_t* table, int position, int page_shift, int num_pages) {
  const int p = table[position >> page_shift];
  return p >= 0 && p < num_pages ? p : -1;
}

}  // namespace tlm
