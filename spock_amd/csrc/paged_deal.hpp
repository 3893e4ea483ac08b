// paged_deal.hpp -- how the rows and keys of a call of spk_paged_attention are
// dealt to workgroups: the host's plan from its bounds, and the device's choice
// from the lengths there.  Plain C++ on host and device; what a wave does
// together comes as W: first (the first lane's value), at (a lane's), count (of
// lanes where a condition holds), sum, max and scan (inclusive sum) over lanes.
#pragma once

#include <stddef.h>

#include <algorithm>

#include "../../include/spock_hip.h"
#include "paged.hpp"

namespace spk_paged {

SPK_HD int lesser(int a, int b) { return a < b ? a : b; }
SPK_HD int larger(int a, int b) { return a > b ? a : b; }
SPK_HD long long lesser(long long a, long long b) { return a < b ? a : b; }

struct Deal {
  Cache c;
  int32_t kv_heads, group, window;
  int32_t many;                // a sequence has many rows from this on
  int32_t shares, share_rows;  // few rows: workgroups, and rows of one
  int32_t alone;               // few rows: no ranges
  int32_t splits, chunk;       // many rows: key ranges of a tile and the least keys of one
};

// The work of the sequences of few rows, dealt to the workgroups of a launch:
// each takes the rows of one sequence, tile of rows and KV head over one range
// of its keys.  The ranges' length follows from the lengths on the device, so
// that they fill the launch once and are nearly equal: with pieces = (sequence,
// tile, head) the number of shares for ranges of c keys is the sum of
// ceil(keys / c) over the pieces, and c the smallest tried with no more shares
// than workgroups.  Every workgroup finds c and its share by itself.
struct Share {
  int seq, tile, kvh;
  int range, ranges, keys;  // this one of the piece's, and the keys of each
  int lo;                   // where the first range begins
  int first;                // the piece's first share
};

struct Load {
  int tiles, span;  // tiles of rows, keys that they see
};

// Of sequence s; nothing past the last.  No branch before the loads: those of
// several sequences are under way together.
SPK_HD Load load_of(const Deal& a, int s) {
  const Seq sq = seq_at(a.c, lesser(s, a.c.num_seqs - 1));
  const int rows = s < a.c.num_seqs ? sq.n * a.group : 0;
  int lo, hi, x;
  visible(sq, 0, a.window, &lo, &x);
  visible(sq, sq.n - 1, a.window, &x, &hi);
  const bool few = rows > 0 && rows < a.many;
  return {few ? (rows + a.share_rows - 1) / a.share_rows : 0, few ? larger(hi - (lo & ~31), 1) : 0};
}

SPK_HD int ranges_of(const Load& l, int c) { return (l.span - 1) / c + (l.span > 0); }

// The share numbered `at`.  false: there is none.
template <class W>
SPK_HD bool find_share(const Deal& a, int at, int lane, Share* out) {
  constexpr int N = 4;  // sequences of a lane at a time
  Load mine[N];
  long long keys = 0;
  int pieces = 0, low = 0, high = 0;  // keys = high * 2^16 + low
  for (int s0 = 0; s0 < a.c.num_seqs; s0 += 64 * N)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      mine[j] = load_of(a, s0 + N * lane + j);
      keys += (long long)mine[j].tiles * mine[j].span;
      pieces += mine[j].tiles;
    }
  low = (int)(keys & 0xffff);
  high = (int)(keys >> 16);
  keys = (((long long)W::first(W::sum(high)) << 16) + W::first(W::sum(low))) * a.kv_heads;
  pieces = W::first(W::sum(pieces)) * a.kv_heads;
  if (pieces == 0) return false;
  // enough for any lengths: each piece's last range may be short
  auto whole = [](long long k) { return (int)((lesser(k, (long long)INT32_MAX - 128) + 127) & ~127ll); };
  int c = INT32_MAX;
  if (!a.alone) {
    const int room = larger(a.shares - pieces, 1);
    c = W::first(whole((keys + room - 1) / room));
  }
  if (!a.alone && a.c.num_seqs <= 64 * N) {
    // unsigned: the next t may pass 2^31
    for (uint32_t t = W::first(whole((keys + a.shares - 1) / a.shares)); t < (uint32_t)c; t += larger(128, (int)(t >> 4) & ~127)) {
      int n = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) n += mine[j].tiles * ranges_of(mine[j], (int)t);
      if (W::first(W::sum(n)) * a.kv_heads <= a.shares) c = (int)t;
    }
  }
  int before = 0;
  for (int s0 = 0; s0 < a.c.num_seqs; s0 += 64 * N) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (a.c.num_seqs > 64 * N) mine[j] = load_of(a, s0 + N * lane + j);
      n += mine[j].tiles * a.kv_heads * ranges_of(mine[j], c);
    }
    const int sum = W::scan(n), total = W::at(sum, 63);
    if (at < before + total) {
      // the lane that holds it, then the one of its sequences
      const int l = W::first(W::count(before + sum <= at));
      int first = before + sum - n;
      Load found{0, 0};
      int s = -1;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int count = mine[j].tiles * a.kv_heads * ranges_of(mine[j], c);
        const bool here = at >= first && at < first + count;
        if (s < 0) {
          if (here) {
            s = s0 + N * lane + j;
            found = mine[j];
          } else {
            first += count;
          }
        }
      }
      s = W::at(s, l);
      first = W::at(first, l);
      found.tiles = W::at(found.tiles, l);
      found.span = W::at(found.span, l);
      if (s < 0 || found.tiles == 0) return false;
      out->seq = s;
      out->ranges = ranges_of(found, c);
      out->keys = ((int)(((uint32_t)found.span + out->ranges - 1) / out->ranges) + 127) & ~127;
      const int rest = at - first, piece = rest / out->ranges;
      out->range = rest - piece * out->ranges;
      out->tile = piece / a.kv_heads;
      out->kvh = piece - out->tile * a.kv_heads;
      out->first = first + (out->tile * a.kv_heads + out->kvh) * out->ranges;
      int x;
      visible(seq_at(a.c, out->seq), 0, a.window, &out->lo, &x);
      out->lo &= ~31;
      return true;
    }
    before += total;
  }
  return false;
}

// Keys in one range of a tile of many rows that sees [lo, hi): the plan's, or
// more where the lengths pass the host's bound.
SPK_HD int range_keys(const Deal& a, int lo, int hi) {
  const int span = larger(hi - (lo & ~31), 0);
  return larger(a.chunk, (int)((((int64_t)span + a.splits - 1) / a.splits + 127) & ~127));
}

// Tile `at` of the tiles of 256 of the n * group rows of the sequences of many:
// its sequence and its index there.  false past the last of them.  Those that
// see the most keys come first, to within 128 keys, so that the last that
// workgroups take are short (six prompts of 16 heads over 4: 180 us, 185 with
// the last sequence's last tile first).
template <class W>
SPK_HD bool find_tile(const Deal& a, int at, int last, int lane, int* seq, int* tile) {
  constexpr int N = 4;  // sequences of a lane
  if (a.c.num_seqs > 64 * N) {  // more than are looked at together: by sequence, the last tiles first
    at = last - at;
    for (int s0 = 0; s0 < a.c.num_seqs; s0 += 64) {
      int mine = 0;
      if (s0 + lane < a.c.num_seqs) {
        const int n = make_seq(a.c, a.c.cu[s0 + lane], a.c.cu[s0 + lane + 1], 0).n * a.group;
        if (n >= a.many) mine = (n + 255) / 256;
      }
      const int sum = W::scan(mine), total = W::at(sum, 63);
      if (at < total) {
        const int l = W::count(sum <= at);
        *seq = s0 + l;
        *tile = at - W::at(sum - mine, l);
        return true;
      }
      at -= total;
    }
    return false;
  }
  Seq sq[N];
  int tiles[N], total = 0, top = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) sq[j] = seq_at(a.c, lesser(N * lane + j, a.c.num_seqs - 1));
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int rows = N * lane + j < a.c.num_seqs ? sq[j].n * a.group : 0;
    tiles[j] = rows >= a.many ? (rows + 255) / 256 : 0;
    if (tiles[j] == 0) sq[j] = {0, 0, 0};  // no tokens: past() is 0
    total += tiles[j];
    top = larger(top, sq[j].ctx);
  }
  if (at >= W::first(W::sum(total))) return false;
  // tiles of the lane's sequence j that see past key 128 * level; all for -1
  auto past = [&](int j, int level) {
    const int64_t d = 128ll * level - sq[j].ctx + sq[j].n;  // its tokens that do not
    return level < 0 || d <= 0 ? tiles[j] : d >= sq[j].n ? 0 : tiles[j] - ((int)d * a.group >> 8);
  };
  int low = -1, high = W::first(W::max(top)) / 128 + 1;
  int before = 0;  // tiles past high
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    int n = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) n += past(j, mid);
    n = W::first(W::sum(n));
    if (n > at) {
      low = mid;
    } else {
      high = mid;
      before = n;
    }
  }
  at -= before;
  int n = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) n += past(j, low) - past(j, high);
  const int sum = W::scan(n), l = W::count(sum <= at);
  int first = sum - n, found = -1, its = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int m = past(j, low) - past(j, high);
    if (found < 0 && at < first + m) {
      found = N * lane + j;
      its = tiles[j] - 1 - past(j, high) - (at - first);
    }
    first += m;
  }
  *seq = W::at(found, l);
  *tile = W::at(its, l);
  return true;
}

// ---------------------------------------------------------------------------
// The host's plan.
// ---------------------------------------------------------------------------

constexpr int kFew = 128;  // rows of a sequence that are not many
constexpr int64_t kMostGroups = 16777215;  // workgroups of 256 in a launch: below 2^32 threads

// How a call's rows and keys are dealt to the kernels.
struct Plan {
  int many, shares, share_rows, tiles, splits, chunk;
  bool join, join_few;
  int64_t join_rows;
  int64_t longest, steps;  // rows of a sequence, and steps of 128 keys, by the bounds
};

// Workgroups of the sequences of few rows.  As many as the chip holds at once (2 to
// a CU; with 4, 32 sequences of one token at 4000 keys take 36 us for 33), more
// only where the pieces alone are more, and no more than ranges of 128 keys.
inline int64_t shares_of(int64_t pieces, int64_t steps) {
  const int64_t slots = 512;
  return std::min<int64_t>(std::min<int64_t>(2 * pieces <= slots ? slots : pieces + slots, pieces * (steps + 1)), INT32_MAX);
}

inline Plan plan_of(const SpkPagedAttnArgs& p) {
  const SpkPagedCache& c = p.cache;
  const int group = p.num_q_heads / c.num_kv_heads;
  const int64_t tokens = std::min(p.max_query_len, c.total_tokens);
  const int64_t longest = tokens * group, all = (int64_t)c.total_tokens * group;
  Plan r;
  r.longest = longest;
  // a call of one sequence that may have many rows goes to their kernel
  // whatever it has; one that has none to the others
  // Many are more than 128, two pieces of 64 (16 sequences at 4000 keys, heads of
  // 128: 128 rows 68 us, 83 as many; 192 rows 88 as many, 118 in three pieces).
  const bool any_many = longest > kFew;
  r.many = !any_many ? INT32_MAX : c.num_seqs == 1 ? 1 : kFew + 1;
  // pieces of 16 rows where none has more (16 rows: 35 us, 38 in pieces of 64;
  // 36 rows: 42 in one of 64, 68 in three of 16)
  r.share_rows = longest <= 16 ? 16 : 64;
  int64_t span = std::min<int64_t>(p.max_context_len, (int64_t)c.max_pages * c.page_size);
  if (p.window > 0) span = std::min<int64_t>(span, (int64_t)p.window + tokens + 31);
  const int64_t steps = std::max<int64_t>(1, (span + 127) / 128);  // of 128 keys
  r.steps = steps;

  // sequences of few rows: all of them, unless the one there is has many.
  // Next to many rows a sequence of few is two pieces; else the bound may be low.
  const int64_t some = all / r.share_rows + c.num_seqs;
  const int64_t pieces = c.num_kv_heads * (!any_many ? some : c.num_seqs > 1 ? std::min<int64_t>(2 * (int64_t)c.num_seqs, some) : 0);
  r.shares = (int)shares_of(pieces, steps);

  // sequences of many rows: one workgroup to a CU.  A tile's keys are split into
  // the number of ranges that takes the fewest rounds of 256 workgroups times
  // steps in each; a range's share of the join costs as much as some 4 steps
  // (2048 tokens at 16384 keys, 64 workgroups: 347 us in 3 ranges, 322 in the 4 that
  // fill the chip; six prompts in 500 workgroups: 184 us, 210 in 2 ranges each).
  const int64_t seqs = std::min<int64_t>(c.num_seqs, all / (kFew + 1) + 1);
  r.tiles = any_many ? (int)std::min<int64_t>((all + 255 * seqs) / 256, INT32_MAX) : 0;
  const int64_t groups = std::max<int64_t>(1, (int64_t)r.tiles * c.num_kv_heads);
  int64_t per = steps, least = (groups + 255) / 256 * steps;
  for (int64_t n = 2; n <= std::min<int64_t>(512 / groups + 1, steps / 4); ++n) {
    const int64_t in = (steps + n - 1) / n, cost = (groups * n + 255) / 256 * (in + 4);
    if (cost < least) per = in, least = cost;
  }
  r.chunk = (int)(128 * per);
  r.splits = r.tiles ? (int)((steps + per - 1) / per) : 1;
  r.join = r.splits > 1 || (r.shares && steps > 1);
  // rows to join: all tokens', or of each sequence those that few can be
  const int64_t every = (int64_t)c.total_tokens * p.num_q_heads, of_few = (int64_t)c.num_seqs * c.num_kv_heads * kFew;
  r.join_few = any_many && r.splits == 1 && of_few < every;
  r.join_rows = r.join_few ? of_few : every;
  return r;
}

inline size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// Of one row's part: its maximum, its sum and its output.
inline size_t part_bytes(const SpkPagedAttnArgs& p) { return (p.cache.head_dim + 2) * sizeof(float); }

inline size_t shared_bytes(const SpkPagedAttnArgs& p, const Plan& r) {
  return r.join ? up((size_t)r.shares * r.share_rows * part_bytes(p)) : 0;
}

inline size_t ranges_bytes(const SpkPagedAttnArgs& p, const Plan& r) {
  return r.join ? up((size_t)p.cache.total_tokens * p.num_q_heads * 2 * sizeof(int32_t)) : 0;
}

inline size_t workspace_of(const SpkPagedAttnArgs& p, const Plan& r) {
  const size_t part = r.splits <= 1 ? 0 : (size_t)r.splits * p.cache.total_tokens * p.num_q_heads * part_bytes(p);
  return shared_bytes(p, r) + ranges_bytes(p, r) + part;
}

// Bytes that no call exceeds whose tokens, sequences, bounds, window and table are
// at most these.  What a plan needs is not monotone in them: more rows leave fewer
// ranges and pieces of other sizes (one sequence of up to 32,768 keys, 8 heads of 256
// over 2: 8 MB for one token, 34 for 9, none for 8,192).  So the largest of each
// part: shares of either size; and with groups = tiles * KV heads, of at most 256
// rows each, up to 512 / groups + 1 ranges of at least 4 steps while that is more
// than one.
inline size_t workspace_bound(const SpkPagedAttnArgs& p) {
  const SpkPagedCache& c = p.cache;
  const Plan r = plan_of(p);
  const int64_t all = (int64_t)c.total_tokens * (p.num_q_heads / c.num_kv_heads), rows = (int64_t)c.total_tokens * p.num_q_heads;
  if (r.steps <= 1) return 0;
  auto shared = [&](int64_t share_rows) { return share_rows * shares_of(c.num_kv_heads * (all / share_rows + c.num_seqs), r.steps); };
  int64_t parts = shared(16);
  if (r.longest > 16) parts = std::max(parts, shared(64));
  int64_t split = 0;
  if (r.longest > kFew && r.steps >= 8)
    split = std::min(131072 + 256 * std::min<int64_t>(512, (all + 255) / 256 * c.num_kv_heads), rows * (r.steps / 4));
  return up(parts * part_bytes(p)) + up(rows * 2 * sizeof(int32_t)) + split * part_bytes(p);
}

// What the kernels know of it.
inline Deal deal_of(const SpkPagedAttnArgs& p, const Plan& r, const Cache& c) {
  Deal d{};
  d.c = c;
  d.kv_heads = p.cache.num_kv_heads;
  d.group = p.num_q_heads / p.cache.num_kv_heads;
  d.window = p.window;
  d.many = r.many;
  d.shares = r.shares;
  d.share_rows = r.share_rows;
  d.alone = !r.join;
  d.splits = r.splits;
  d.chunk = r.chunk;
  return d;
}

}  // namespace spk_paged
