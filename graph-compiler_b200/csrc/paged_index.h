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

// Page that holds position `pos` of sequence `seq`, or -1 when the table has no entry for it or the entry is outside the cache.
GCB_HD int page_of(const PageTable &t, int seq, int pos) {
  if (seq < 0 || seq >= t.sequences || pos < 0) return -1;
  const int entry = pos / t.page_size;
  if (entry >= t.max_pages) return -1;
  const int page = t.entries[int64_t(seq) * t.stride + entry];
  return page >= 0 && page < t.pages ? page : -1;
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

} // namespace gcb
