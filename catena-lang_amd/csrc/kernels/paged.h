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

// The kernels' arguments, which the host fills.

// attn_paged.hip
struct AttnPagedArgs {
  PagedKv kv;
  const uint16_t* q;      // [rows][heads][D]
  const uint32_t* lens;   // [rows]
  void* o;                // [rows][heads][D]
  float* part_o;          // [blocks][2][min(group, 16)][D]
  float* part_ml;         // [blocks][2][min(group, 16)][2]: maximum (base 2), sum
  float* whole_ml;        // [rows][heads][2]: of units that were not cut, with weights that the join adds
  float* scores;          // [rows][heads][slots] base-2 scores, with weights only
  const float* acc_in;    // [rows][kv_heads][slots]
  float* acc_out;
  uint32_t group, head_tiles;
  uint32_t blocks;        // workgroups; 0: one a unit
  uint32_t short_slots;   // whole units while no row is longer
  float scale_log2;       // scale * log2(e)
};

// kv_paged.hip: eviction, reordering
struct EvictArgs {
  PagedKv kv;
  const uint32_t* lens;
  const uint32_t* seen;
  const float* acc_in;
  const uint32_t* pos_in;
  uint32_t* lens_out;
  float* acc_out;
  uint32_t* pos_out;
  uint32_t* count;    // [pairs]
  uint32_t* holes;    // [pairs][most]
  uint32_t* sources;  // [pairs][most]
  uint32_t most, budget, recent;
  uint32_t at_once;   // the choosing workgroup makes the moves itself
};

struct ReorderArgs {
  PagedKv kv;
  const uint32_t* lens;
  const uint32_t* parents;
  const uint32_t* spare;
  uint32_t* table_out;
  uint32_t* lens_out;
  uint32_t* spare_out;
  uint32_t n_pools, tables;
};
template <int MOST>
struct ReorderPools {
  uint16_t* p[MOST];
};
