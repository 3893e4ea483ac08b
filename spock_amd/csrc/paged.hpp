// paged.hpp -- where the tokens of a step and the positions of a paged cache
// lie: the index arithmetic of spk_mrope_append and spk_paged_attention, with
// every value that comes from device memory (offsets, lengths, page ids)
// brought into the caller's buffers.  Plain C++ on host and device.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define SPK_HD __host__ __device__ __forceinline__
#else
#define SPK_HD inline
#endif

namespace spk_paged {

// p / d for 0 <= p < 2^31 as the high half of a 32-bit product and a shift:
// with 2^(s-1) < d <= 2^s and mul = floor(2^(31+s) / d) + 1 the product p mul /
// 2^(31+s) is at most p / 2^(31+s) < 1 / d too large, which never reaches the
// next integer.
struct PageDiv {
  uint32_t mul, shift;
};

SPK_HD PageDiv page_div(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < d) ++s;
  return {(uint32_t)((uint64_t(1) << (31 + s)) / d + 1), s};
}

SPK_HD uint32_t divide(PageDiv v, uint32_t p) { return (uint32_t)(((uint64_t)(2 * p) * v.mul) >> 32) >> v.shift; }

struct Cache {
  const int32_t* table;  // [num_seqs][table_stride]
  const int32_t* cu;     // [num_seqs + 1]
  const int32_t* ctx;    // [num_seqs]
  int64_t table_stride;
  int64_t head_stride;                  // elements, as all strides
  uint32_t page_stride, token_stride;
  int32_t num_seqs, total_tokens, page_size, num_pages, max_pages;
  PageDiv div;
};

// Tokens [first, first + n) of the step, after which the cache holds `ctx`.
struct Seq {
  int32_t first, n, ctx;
};

SPK_HD Seq make_seq(const Cache& c, int32_t begin, int32_t end, int32_t ctx) {
  Seq s;
  s.first = begin < 0 ? 0 : begin > c.total_tokens ? c.total_tokens : begin;
  const int32_t last = end < s.first ? s.first : end > c.total_tokens ? c.total_tokens : end;
  s.n = last - s.first;
  const int64_t room = (int64_t)c.max_pages * c.page_size;
  s.ctx = ctx < 0 ? 0 : (int64_t)ctx > room ? (int32_t)room : ctx;
  return s;
}

SPK_HD Seq seq_at(const Cache& c, int32_t s) { return make_seq(c, c.cu[s], c.cu[s + 1], c.ctx[s]); }

// Element offset of position `pos` (0 <= pos < ctx) of KV head 0 in a page
// that the table named, or -1 where that is no page of the pool.
SPK_HD int64_t offset_in(const Cache& c, int32_t page, int32_t pos) {
  if ((uint32_t)page >= (uint32_t)c.num_pages) return -1;
  const int32_t at = pos - (int32_t)(divide(c.div, (uint32_t)pos) * (uint32_t)c.page_size);
  return (int64_t)((uint64_t)(uint32_t)page * c.page_stride + (uint64_t)(uint32_t)at * c.token_stride);
}

SPK_HD int64_t offset_of(const Cache& c, int32_t s, int32_t pos) {
  return offset_in(c, c.table[(int64_t)s * c.table_stride + divide(c.div, (uint32_t)pos)], pos);
}

// Keys [lo, hi) that the query at step index i of a sequence sees: up to its
// own position, the last `window` of them where window > 0.  Empty (0, 0)
// where the position lies before the cache's first.
SPK_HD void visible(const Seq& s, int32_t i, int32_t window, int32_t* lo, int32_t* hi) {
  const int32_t pos = s.ctx - s.n + i;
  *hi = pos < 0 ? 0 : pos + 1;
  *lo = window > 0 && *hi > window ? *hi - window : 0;
}

#if defined(__HIPCC__)
// The sequence of row t: how many sequences end at or before it.  One load
// per lane and a ballot for 64 sequences; every lane returns the same.
__device__ __forceinline__ int seq_of_token(const int32_t* cu, int num_seqs, int t, int lane) {
  int s = 0;
  for (int s0 = 0; s0 < num_seqs; s0 += 64) {
    const bool ended = s0 + lane < num_seqs && cu[s0 + lane + 1] <= t;
    const int n = __popcll(__ballot(ended));
    s += n;
    if (n < 64) break;
  }
  return s;
}
#endif

}  // namespace spk_paged
