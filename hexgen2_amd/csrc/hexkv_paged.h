// Device helpers and argument checks of the paged caches (hexkv_paged.hip,
// hexkv_paged_attend.hip).
#pragma once

#include "hexkv_common.h"

namespace hexkv {

// A call's sequences, and their pages, as its kernels take them.
struct PageTables {
  const int32_t *tables;
  int64_t table_stride;
  const int32_t *starts, *cu;  // cu: nullptr where every sequence has `each` tokens
  int32_t width, batch, tokens, each;
  int32_t n_pages, shift;  // positions of a page: 2^shift
  int64_t page_stride, pos_stride, kv_stride, head_stride;  // elements
};

// Tokens of one sequence: [first, first + count), the first at position
// start.  What cu_tokens holds is taken for what it is only inside [0, tokens]; a
// sequence it puts elsewhere has no tokens.
struct Sequence {
  int32_t first, count, start;
};

__device__ __forceinline__ Sequence sequence_of(const PageTables &p, int b) {
  Sequence s;
  s.start = p.starts[b];
  if (p.cu) {
    const int lo = p.cu[b], hi = p.cu[b + 1];
    const bool fits = lo >= 0 && hi >= lo && hi <= p.tokens;
    s.first = fits ? lo : 0;
    s.count = fits ? hi - lo : 0;
  } else {
    s.first = b * p.each;
    s.count = p.each;
  }
  return s;
}

// The sequence that token t belongs to, or -1: a wave looks at 64 at a time.
__device__ __forceinline__ int token_sequence(const PageTables &p, int t) {
  const int lane = threadIdx.x & 63;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const int b = min(b0 + lane, p.batch - 1), lo = p.cu[b], hi = p.cu[b + 1];
    const uint64_t in = __ballot(lo >= 0 && lo <= t && t < hi && hi <= p.tokens);
    if (in) return min(b0 + __builtin_ctzll(in), p.batch - 1);
  }
  return -1;
}

// Checks a pool and a call's sequences and fills `p`; the library's status.
int check_pool(const hexkv_pool &pool, const char *what);
int fill_tables(const hexkv_pool &pool, const hexkv_paged_batch &seqs, PageTables *p, const char *what);

inline int elem_bytes(int dtype) { return dtype == HEXKV_F32 ? 4 : 2; }

// Bytes from the pool's base to the end of its last element.
int64_t pool_bytes(const hexkv_pool &pool);

// Whether [a, a + a_bytes) and [b, b + b_bytes) share a byte.
inline bool overlap(const void *a, int64_t a_bytes, const void *b, int64_t b_bytes) {
  const intptr_t x = reinterpret_cast<intptr_t>(a), y = reinterpret_cast<intptr_t>(b);
  return a_bytes > 0 && b_bytes > 0 && x < y + b_bytes && y < x + a_bytes;
}

}  // namespace hexkv
