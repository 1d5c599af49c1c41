// The paged cache as the kernels see it: where a row is, and the checks of a caller's description.
#pragma once

#include "common.cuh"

namespace rab {

inline int page_shift(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

// Index of row `slot` of a sequence among the rows of KV head 0 of its page (of kv_heads << shift rows a page), -1 where the
// sequence has no such row: before its first one, behind its table, or in a page whose number is out of range.
__host__ __device__ inline long long paged_row(const int* table, int max_pages, int num_pages, int shift, int kv_heads,
                                               long long slot) {
  if (slot < 0 || slot >> shift >= max_pages) return -1;
  const int page = table[slot >> shift];
  if (page < 0 || page >= num_pages) return -1;
  return (static_cast<long long>(page) * kv_heads << shift) + (slot & ((1ll << shift) - 1));
}

inline int check_paged(const ra_paged_kv& c, const char* what) {
  RAB_REQUIRE(c.kv_heads > 0 && c.num_pages >= 0 && c.batch >= 0 && c.max_pages >= 0, RA_ERR_INVALID, "%s: bad cache", what);
  RAB_REQUIRE(c.page_size == 16 || c.page_size == 32 || c.page_size == 64 || c.page_size == 128 || c.page_size == 256,
              RA_ERR_UNSUPPORTED, "%s: unsupported page_size=%d (supported: 16, 32, 64, 128, 256)", what, c.page_size);
  RAB_REQUIRE(c.num_pages == 0 || (c.k && c.v), RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & 15u) == 0, RA_ERR_INVALID,
              "%s: the pages must be 16-byte aligned", what);
  RAB_REQUIRE(c.batch == 0 || (c.lens && (c.page_table || c.max_pages == 0)), RA_ERR_INVALID, "%s: null argument", what);
  RAB_REQUIRE(c.batch <= 1 || c.table_stride >= 0, RA_ERR_INVALID, "%s: bad stride of the page table", what);
  return RA_OK;
}

// (of a call that reads them; the size of a workspace does not depend on where they are)
inline int check_lists(const ra_paged_kv& c, const char* what) {
  RAB_REQUIRE(((reinterpret_cast<uintptr_t>(c.lens) | reinterpret_cast<uintptr_t>(c.page_table)) & 3u) == 0, RA_ERR_INVALID,
              "%s: lens or page_table is not aligned to its elements", what);
  return RA_OK;
}

}  // namespace rab
