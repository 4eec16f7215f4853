// A key-value cache in pages, as the kernels see it (passed by value), and
// the one place where a slot of a row becomes an address.  Plain C++: the
// host fills the struct, and a CPU test calls the same functions.
//
// k, v: [num_pages][kv_heads][1 << page_shift][head_dim] bf16, table:
// [rows][max_pages] page numbers.  Slot j of a row lives in page
// table[row][j >> page_shift].  A page number that the pool does not have
// gives no address: readers treat its slots as absent, writers skip them.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define CATENA_HD __host__ __device__ __forceinline__
#else
#define CATENA_HD inline
#endif

struct PagedKv {
  uint16_t* k;
  uint16_t* v;
  const uint32_t* table;
  uint32_t num_pages, page_shift, rows, max_pages, kv_heads, head_dim;
};

CATENA_HD uint32_t paged_slots(const PagedKv& kv) { return kv.max_pages << kv.page_shift; }

// Slots in use: a length past the table's end is cut to it.
CATENA_HD uint32_t paged_len(const PagedKv& kv, uint32_t len) {
  const uint32_t slots = paged_slots(kv);
  return len < slots ? len : slots;
}

// Elements in front of place `place` of (page, head), in 64 bits: a pool of
// 2^31 bytes is passed long before the page numbers run out.
CATENA_HD uint64_t paged_offset(const PagedKv& kv, uint32_t page, uint32_t head, uint32_t place) {
  return ((((uint64_t)page * kv.kv_heads + head) << kv.page_shift) + place) * kv.head_dim;
}

// Where slot `slot` of `row` lives for `head`; false where it has no place:
// past the table or in a page that the pool does not have.
CATENA_HD bool paged_place(const PagedKv& kv, uint32_t row, uint32_t head, uint32_t slot, uint64_t* at) {
  if (slot >= paged_slots(kv)) return false;
  const uint32_t page = kv.table[(uint64_t)row * kv.max_pages + (slot >> kv.page_shift)];
  if (page >= kv.num_pages) return false;
  *at = paged_offset(kv, page, head, slot & ((1u << kv.page_shift) - 1u));
  return true;
}
