// How ls_paged_attn cuts its work, from the sizes alone (host code, no CUDA).
#pragma once

#include <algorithm>
#include <cstdint>

#include "../../include/leanselect_b200.h"

namespace ls {

constexpr int kPagedMaxRanges = 2 * 148;  // work ranges: two on each of the B200's SMs

// Units of work a row counts for besides its pages.
constexpr int kPagedRowCost = 4;
// Most pages of a request whose tokens' page lists are joined in one tile.
constexpr int kPagedMaxUnion = 512;
// The kernels add up units in 32 bits.
constexpr int64_t kPagedMaxWork = int64_t{1} << 31;

struct PagedSizes {
  int64_t total_q;
  int batch;
  int num_kv_heads;
  int heads_per_group;
  int topk;              // 0: every page
  int max_blocks;
  int max_seqlen_q;
  int max_seqlen_k;
};

struct PagedSchedule {
  int units;   // lists of single tokens: pages a row is scheduled with
  int pack;    // tokens of one request in a 16-row tile
  int ranges;  // most ranges of work
};

// Whether rows that each stand alone stay within the kernels' sums: the limit
// callers are held to.
inline bool paged_rows_fit(const PagedSizes& s) {
  return s.total_q * s.num_kv_heads * ((s.topk > 0 ? s.topk : s.max_blocks) + kPagedRowCost) <
         kPagedMaxWork;
}

// The same for tiles of `tokens` tokens with joined lists: a tile is scheduled
// with all the pages its tokens can list, also where its request has one token
// only.  Every request fills at most one tile partly.
inline bool paged_joined_tiles_fit(const PagedSizes& s, int tokens) {
  const int64_t tiles = std::min<int64_t>(s.total_q, s.total_q / tokens + s.batch);
  const int64_t pages = std::min<int64_t>(int64_t{tokens} * s.topk, s.max_blocks);
  return tiles * s.num_kv_heads * (pages + kPagedRowCost) < kPagedMaxWork;
}

inline PagedSchedule paged_schedule(const PagedSizes& s, int sms) {
  PagedSchedule r{0, 1, 1};
  // At most one range per scheduled page: the caller's max_seqlen_k bounds the
  // pages of a dense row (a longer request only gets fewer ranges).
  const int64_t most_pages = std::max<int64_t>(1, (int64_t{s.max_seqlen_k} + LS_PAGE_TOKENS - 1) /
                                                      LS_PAGE_TOKENS);
  const int64_t rows = s.total_q * s.num_kv_heads;
  if (s.topk > 0) r.units = static_cast<int>(std::min<int64_t>(s.topk, most_pages));
  // A tile of 16 rows takes as many tokens of a request as their heads fit, so
  // that a draft or a chunk reads each page once for all of them: 8 tokens over
  // 131072 keys, 2 x 8 heads, take 55 us against 87 one by one.  Page lists are
  // joined for that where a table of the request's pages fits on chip, where
  // they must overlap threefold (one visit for several tokens masks per page
  // and costs twice as much: 512 tokens of 2 x 2 heads with 96 of 256 pages
  // each 156 us against 204, with 96 of 384 pages 220 against 212), where 30
  // pages per range, rows' own cost included, hide the joining (512 tokens of 2
  // x 4 heads over 5 pages 19 us against 27; 128 of 2 x 1 heads with 16 of 16
  // pages 20 against 18, 32 of 2 x 4 with 32 of 42 pages 19 against 14) and
  // where the tiles' units can be added up (millions of requests of a token or
  // two do not get there: they stay rows of their own).
  if (s.max_seqlen_q > 1) {
    const int tokens = std::min(16 / s.heads_per_group, s.max_seqlen_q);
    if (s.topk == 0 ||
        (most_pages <= kPagedMaxUnion && int64_t{tokens} * r.units >= 3 * most_pages &&
         rows * (r.units + kPagedRowCost) >= int64_t{30} * 2 * sms &&
         paged_joined_tiles_fit(s, tokens)))
      r.pack = tokens;
  }
  const int64_t per_row = s.topk > 0 ? r.units : most_pages;
  r.ranges = static_cast<int>(
      std::min<int64_t>({rows * per_row, int64_t{2} * sms, int64_t{kPagedMaxRanges}}));
  return r;
}

}  // namespace ls
