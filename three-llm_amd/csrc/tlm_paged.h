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

// The page of a position in its sequence's table, or -1 where the entry is none
// of the pool's.
TLM_HD int paged_page(const int32_t* table, int position, int page_shift, int num_pages) {
  const int p = table[position >> page_shift];
  return p >= 0 && p < num_pages ? p : -1;
}

}  // namespace tlm
