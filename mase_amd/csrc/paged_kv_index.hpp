// Where a slot of a paged key-value cache lies.  Plain C++ (no device types), so that the bounds that keep a kernel inside
// the pool can be checked by a host program too.
//
// Slot t of a sequence is row t % page_size of page table[t / page_size].  Lengths and page numbers come from device
// memory, so no host check sees them: a length is cut to what the call and the table can hold, and a page number outside
// the pool is never followed (its slots count as absent).
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define MASE_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define MASE_HOST_DEVICE inline
#endif

namespace mase {

// slots of a sequence that a kernel looks at, from the length in memory
MASE_HOST_DEVICE int kv_length(int given, int max_length, int table_pages, int page_shift) {
  const long long room = (long long)table_pages << page_shift;
  long long n = given < max_length ? given : max_length;
  n = n < room ? n : room;
  return n > 0 ? (int)n : 0;
}

// page number of a slot, or -1 when the slot lies outside the table or the table's entry outside the pool
MASE_HOST_DEVICE int kv_page(const int32_t* table_row, int table_pages, int page_shift, int num_pages, int slot) {
  if (slot < 0) return -1;
  const int at = slot >> page_shift;
  if (at >= table_pages) return -1;
  const int page = table_row[at];
  return page >= 0 && page < num_pages ? page : -1;
}

// slot of new token j of a sequence whose tokens go to start, start + 1, ..., or -1 when it does not exist or fit
MASE_HOST_DEVICE int kv_new_slot(int start, int count, int j, int table_pages, int page_shift) {
  if (j >= count || start < 0) return -1;
  const long long slot = (long long)start + j;
  return slot < ((long long)table_pages << page_shift) ? (int)slot : -1;
}

}  // namespace mase
