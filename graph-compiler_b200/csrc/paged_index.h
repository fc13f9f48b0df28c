// Index arithmetic of the paged cache that decides which memory a kernel touches.  Plain C++, for the device and the host alike,
// so that it can be checked without a device.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define GCB_HD __host__ __device__ __forceinline__
#else
#define GCB_HD inline
#endif

namespace gcb {

struct PageTable {
  const int32_t *entries;
  int64_t stride;                             // entries between the rows of two sequences
  int sequences, max_pages, page_size, pages; // rows, entries of a row, tokens of a page, pages of the cache
};

// Page in entry `entry` of sequence `seq`, or -1 when there is no such entry or it is outside the cache.
GCB_HD int page_at(const PageTable &t, int seq, int entry) {
  if (seq < 0 || seq >= t.sequences || entry < 0 || entry >= t.max_pages) return -1;
  const int page = t.entries[int64_t(seq) * t.stride + entry];
  return page >= 0 && page < t.pages ? page : -1;
}
// Page that holds position `pos`.
GCB_HD int page_of(const PageTable &t, int seq, int pos) { return pos < 0 ? -1 : page_at(t, seq, pos / t.page_size); }

// Whether two of the rows of `dim` elements at i a + j b overlap (0 <= i < na, 0 <= j < nb).
inline bool rows_overlap(int64_t na, int64_t a, int64_t nb, int64_t b, int64_t dim) {
  if (na < 1 || nb < 1) return false;
  if (na == 1) na = nb, a = b, nb = 1;
  if (na == 1) return false;
  a = a < 0 ? -a : a;   // the same rows, counted from the other end
  b = b < 0 ? -b : b;
  if (nb > 1 && a > b) {
    int64_t t = a; a = b; b = t;
    t = na; na = nb; nb = t;
  }
  if (a < dim) return true;
  // rows i and j steps away: the nearest ones before and behind every j b
  for (int64_t j = 1; j < nb; ++j) {
    const int64_t i = j * b / a, rest = j * b - i * a;
    if (i >= na) return false;
    if (rest < dim || (i + 1 < na && a - rest < dim)) return true;
  }
  return false;
}

// Positions [first, end) that a query sees in a sequence said to hold `length` tokens; window 0: all.  `cut`: length was more than
// the table has room for.
struct Seen {
  int first, end;
  bool cut;
};
GCB_HD Seen seen_of(const PageTable &t, int length, int window) {
  const int room = t.max_pages * t.page_size;   // below 2^31, checked by the launchers
  Seen s;
  s.cut = length > room;
  s.end = length < 0 ? 0 : s.cut ? room : length;
  s.first = window > 0 && s.end > window ? s.end - window : 0;
  return s;
}

// How the tokens that all queries see are shared out among `blocks` thread blocks.  A unit is what one set of query heads of one
// KV head does for one sequence; its tokens are cut into tiles, and the tiles of all units, sequence by sequence and unit by unit
// inside, are one row of `total` that is cut into equal parts: block i takes [i per, (i + 1) per).  A unit may be cut by the borders
// of several blocks; each then keeps a part of its softmax, and the parts are joined in the order of the blocks.
GCB_HD int tiles_of(const Seen &s, int tile) { return (s.end - s.first + tile - 1) / tile; }
// Large shares are rounded up to fours (never by more than an eighth): where units have 2^n tiles, odd shares leave the blocks at as
// many different places of a sequence at a time.  Without and with, 32 heads of their own: 16 x 2048 tokens 110 and 90 us, 32 x 1024
// 112 and 90, 16 x 4096 208 and 176, 8 x 5000 109 and 108.  The blocks that it leaves idle cost less than it gives elsewhere too: 64 x
// 512..4096 tokens of eight KV heads 102.5 and 103.0, 128 x 1024..8192 in 8 bits 201.8 and 199.2, 2 x 131071 167.9 and 168.6, 8 x 30000
// 156.0 and 156.4.
GCB_HD int64_t share_of(int64_t total, int blocks, int least) {
  int64_t per = (total + blocks - 1) / blocks;
  if (per >= 32) per = (per + 3) / 4 * 4;
  return per < least ? least : per;
}
// A block keeps at most two parts: of the unit that it continues (0) and of one that it begins and does not end (1).
GCB_HD int64_t part_slot(int64_t block, int64_t per, int64_t unit_begin) { return 2 * block + (unit_begin >= block * per ? 1 : 0); }
// Whether border number `i` (the tile i per) is the first one inside the unit [begin, end): the join of its parts belongs to it.
GCB_HD bool first_cut(int64_t i, int64_t per, int64_t begin, int64_t end) {
  return begin < i * per && i * per < end && begin >= (i - 1) * per;
}

} // namespace gcb
