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

// The same cache in 4 bits (e2m1, two values a byte, the first in the lower half):
//   k [num_pages][kv_heads][page][head_dim / 2], k_scale [..][head_dim / 32][page]:
//     32 values of a slot share the power of two 2^(byte - 127)
//   v [num_pages][kv_heads][head_dim / 2][page], v_scale [..][page]: one bf16 scale
//     a (slot, head)
struct PagedKv4 {
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_scale;
  uint16_t* v_scale;
  const uint32_t* table;
  uint32_t num_pages, page_shift, rows, max_pages, kv_heads, head_dim;
};

// Slots in front of (page, head) in a pool, in 64 bits
CATENA_HD uint64_t paged_cells(uint32_t kv_heads, uint32_t page_shift, uint32_t page, uint32_t head) {
  return ((uint64_t)page * kv_heads + head) << page_shift;
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

// attn_paged_q4.hip.  Units (a row, kv head and up to 16 query heads) are cut into tiles of
// kAttnQ4Slots slots for two workgroups a CU, or three where these hold them (64 columns) and there are kAttnQ4TwoACu
// tiles (64 ragged rows up to 8192 slots 46 us against 52, up to 16384 76 / 83; 4 x 32768, 2048 tiles, 30.5 / 22.8).  Not where the longest row, which one workgroup
// reads at about 2.2 us a tile, ends with the others: all of them take 7.1 us for 512 tiles
// of 128 columns, cutting about 6; nor is it long beside the others, which would leave CUs
// idle at the end.  Rows x slots of 8 kv heads, whole / cut, us: 2 x 1024 9.2 / 11.0, x 2048
// 13.5 / 11.1, x 4096 22.4 / 11.6; 8 x 1024 9.3 / 11.5, x 2048 14.5 / 12.8, x 4096 23.2 /
// 16.5; 16 x 2048 14.9 / 16.6, x 4096 23.6 / 21.1; 32 x 2048 17.3 / 21, x 4096 31 / 34.5;
// 64 x 4096 55 / 57; ragged 32 up to 4096 25 / 29, 64 up to 2048 24 / 29, up to 8192 76 / 70,
// up to 16384 147 / 122, 256 up to 4096 128 / 144.
constexpr uint32_t kAttnQ4Slots = 512, kAttnQ4WholeShare = 200, kAttnQ4WholeMost = 12, kAttnQ4TwoACu = 4096;
// The pools, in place of AttnPagedArgs' own
struct AttnQ4Pools {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* k_scale;
  const uint16_t* v_scale;
  uint32_t flip;  // the signs of q, so that scale_log2 > 0
};

// Workgroup `block`'s stretch [beg, end) of a line of tiles (below 2^31), `per` to each of its `blocks` workgroups.  A
// grid may have more, whose place would pass 32 bits: they have none, beg = end.
struct Stretch {
  uint32_t beg, end;
};
CATENA_HD Stretch stretch_of(uint32_t tiles, uint32_t per, uint32_t blocks, uint32_t block) {
  const uint32_t beg = block < blocks ? block * per : tiles;
  if (beg >= tiles) return Stretch{tiles, tiles};
  return Stretch{beg, tiles - beg < per ? tiles : beg + per};
}

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

// kv_admit.hip
struct AdmitArgs {
  uint32_t rows, max_pages, page_shift, num_pages;
  uint32_t* table;
  const uint32_t* lens;
  const uint32_t* held;
  const uint32_t* want;
  const uint32_t* seen;  // may be null, then seen_out is
  const uint32_t* free_pages;
  const uint32_t* free_count;
  uint32_t* lens_out;
  uint32_t* held_out;
  uint32_t* seen_out;
  uint32_t* starts;
  uint32_t* free_count_out;
  uint32_t* token_pos;
  uint64_t* slot_map;
  uint32_t max_tokens;
};

struct ReleaseArgs {
  uint32_t rows, max_pages, num_pages;
  uint32_t* table;
  const uint32_t* lens;
  const uint32_t* held;
  const uint32_t* finished;
  uint32_t* free_pages;
  const uint32_t* free_count;
  uint32_t* lens_out;
  uint32_t* held_out;
  uint32_t* free_count_out;
};

// rope_packed.hip
struct RopePackedArgs {
  const void* qkv;
  const float* tab;         // [positions][rot / 2] (cos, sin)
  const uint32_t* pos;      // [tokens]
  const uint64_t* slots;    // [tokens] page * page_size + place; may be null
  uint16_t* q;
  uint16_t* k_out;          // [tokens][kv_heads][head_dim], may be null
  uint16_t* v_out;
  uint32_t positions, rot, interleaved, heads;
};

// attn_prompt.hip
constexpr uint32_t kPromptWhole = 0xFFFFFFFFu;  // an item that is all of its unit
constexpr uint32_t kPromptQueues = 8;           // one an XCD
constexpr uint32_t kPromptCus = 256;
constexpr uint32_t kPromptRows = 256, kPromptNarrow = 64;  // query rows of a unit; of so many a narrow one
constexpr uint32_t kPromptLeast = 32;              // what a unit costs that is not cut (two a tile of 64 slots)
constexpr uint32_t kPromptParts = 16 * kPromptCus;  // places of kPromptNarrow query rows for the parts of all kv heads
// What a unit costs that is not cut, in half tiles for a wide one (its tiles twice) and tiles for a narrow one: three
// quarters of a CU's share of all the work, a quarter of that for a narrow one, whose parts have next to nothing to join.
struct PromptCut {
  uint32_t most, most_narrow;
  float share, share_narrow;  // 1 / most
};
// work: the units' costs of all kv heads
CATENA_HD PromptCut prompt_cut(uint64_t work) {
  const uint64_t even = 3 * work / (4 * kPromptCus) + 1;
  PromptCut c;
  c.most = even < kPromptLeast ? kPromptLeast : even < 0x7FFFFFFFull ? (uint32_t)even : 0x7FFFFFFFu;
  c.most_narrow = c.most / 4 < kPromptLeast / 2 ? kPromptLeast / 2 : c.most / 4;
  c.share = 1.0f / (float)c.most;
  c.share_narrow = 1.0f / (float)c.most_narrow;
  return c;
}
// (a rounding may make a part a little larger or smaller, the same for all who ask)
CATENA_HD uint32_t prompt_parts(const PromptCut& c, uint32_t cost, bool narrow) {
  if (cost <= (narrow ? c.most_narrow : c.most)) return 1;
  return (uint32_t)((float)(cost - 1) * (narrow ? c.share_narrow : c.share)) + 1;
}
// Places that one part takes for each kv head
CATENA_HD uint32_t prompt_places(bool narrow) { return narrow ? 1 : kPromptRows / kPromptNarrow; }
// Why kPromptParts places are enough.  A unit that is cut costs more than the most of its kind, so its parts are fewer
// than 2 cost / most (both up to roundings of 2^-22).  With W the costs of all kv heads, most > 3 W / (4 CUs): wide
// units take 4 places a part, so fewer than 8 W / most < 32 / 3 a CU; narrow ones one place, and most_narrow >= (most
// - 3) / 4 >= 29 / 128 most, so fewer than 2 * 128 / 29 W / most < 11.8 a CU.  Whatever the mixture, no more than 12.
static_assert(kPromptParts >= 12 * kPromptCus && kPromptRows == 4 * kPromptNarrow && kPromptLeast >= 32, "places for parts");

// 256 query rows (unit `unit`) of a row's n new tokens, `old` slots in front of them: tiles [beg, end) of what they
// see.  In the list of cut units: beg is the number of parts, `part` the first one.
struct PromptItem {
  uint32_t row, unit, first, n;
  int32_t old;
  uint32_t beg, end, part;
};
struct PromptCounts {
  uint32_t items, wide;   // of the list; of them, in front, those of rows with wide units
  uint32_t splits;
  uint32_t narrow_first;  // of a queue's workgroups so many begin with the others
  uint32_t narrow_waves;  // so many waves to one of their units
  uint32_t tickets[2][kPromptQueues];  // taken of each kind
};
constexpr uint32_t kPromptCountBytes = 128;  // in the workspace, in front of the list
struct AttnPromptArgs {
  PagedKv kv;               // table null: k, v [tokens][kv_heads][head_dim], stride apart
  const uint16_t* q;        // [tokens][heads][D]
  const uint32_t* starts;   // [rows + 1]
  const uint32_t* lens;     // [rows]; null: as many as new tokens
  uint16_t* o;              // [tokens][heads][D]
  uint64_t stride;          // elements from a token's k to the next one's, without a table
  PromptItem* items;        // the list; null: a workgroup a unit
  PromptItem* splits;       // units that were cut
  PromptCounts* counts;
  // part_rows query rows a place, as many as there may be up to kPromptNarrow; a part has one for each kv head, or, of
  // a wide unit, kPromptRows / kPromptNarrow
  float* part_o;            // [place][part_rows][D]
  float* part_ml;           // [place][part_rows][2]: reference point (base 2), sum
  uint32_t part_rows;
  uint32_t max_items, max_splits;
  uint32_t tokens, group;
  float scale_log2;         // |scale| log2(e)
  uint32_t flip;            // 0x80008000 where the scale is negative: q's signs
};
