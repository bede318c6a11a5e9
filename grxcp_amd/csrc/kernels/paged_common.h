// The paged key-value cache as the kernels see it: which page and which row of it
// a sequence's slot is, with every index checked before it is followed. Host and
// device code (the arithmetic is tested on the CPU).
#ifndef GRXCP_PAGED_COMMON_H
#define GRXCP_PAGED_COMMON_H

#include <stdint.h>

#ifdef __HIPCC__
#define GRX_HD __host__ __device__ __forceinline__
#else
#define GRX_HD inline
#endif

namespace grxk {

// n / d for 0 <= n < 2^31 by one multiplication. With l = ceil(log2 d) and
// m = ceil(2^(31+l) / d): m d = 2^(31+l) + e with 0 <= e < d <= 2^l, so n m /
// 2^(31+l) exceeds n / d by n e / (d 2^(31+l)) < 1 / d, too little to reach the
// next integer. m <= 2^32 / 2 * 2^l / d < 2^32.
struct PageDiv {
  uint32_t mul;
  int shift;
};
inline PageDiv page_div(int d) {
  int l = 0;
  while ((1ll << l) < d) ++l;
  const uint64_t top = 1ull << (31 + l);
  return {(uint32_t)((top + (uint64_t)d - 1) / (uint64_t)d), 31 + l};
}
GRX_HD int div_page(PageDiv d, int n) { return (int)(((uint64_t)(uint32_t)n * d.mul) >> d.shift); }

struct PagedView {
  const int* table;      // [B, W], rows table_rs apart
  int64_t table_rs;
  const int* lengths;    // [B]
  int pages;             // pages of the pools
  int page;              // slots per page
  int room;              // W * page: slots that a table row has room for
  PageDiv div;
};

GRX_HD int clamp_length(int n, int room) { return n < 0 ? 0 : n > room ? room : n; }

// The page that a table entry names, or -1 for one that no pool has.
GRX_HD int checked_page(int entry, int pages) { return (uint32_t)entry < (uint32_t)pages ? entry : -1; }

// Slot `slot` (>= 0) of sequence b: its page and row in it. False, and page -1, where
// the sequence has no room for it or its entry names no page. Without a branch (a slot
// without room reads the row's last entry): the compiler (ROCm 7.2) lost the assignment
// in "if (!find_slot(a) || !find_slot(b)) x[u] = -1" over an unrolled array when this was
// one, and rows went to page -1. Callers join its results with & and selects.
GRX_HD bool find_slot(const PagedView& v, int b, int slot, int* page, int* row) {
  const int in = slot < v.room ? slot : v.room - 1;
  const int i = div_page(v.div, in);
  const int at = checked_page(v.table[b * v.table_rs + i], v.pages);
  *page = slot < v.room ? at : -1;
  *row = in - i * v.page;
  return *page >= 0;
}

// A weight as a key whose unsigned order is the eviction's: NaN above all, -0 as 0.
GRX_HD uint32_t order_key(uint32_t bits) {
  const uint32_t mag = bits & 0x7fffffffu;
  if (mag > 0x7f800000u) return 0xffffffffu;
  if (mag == 0) return 0x80000000u;
  return (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}

}  // namespace grxk

#endif  // GRXCP_PAGED_COMMON_H
