// Checks and plans that the calls over a cache in pages share (paged.cpp,
// requests.cpp).
#pragma once

#include <algorithm>
#include <cstdint>

#include "../kernels/paged.h"
#include "internal.h"

namespace catena {

inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
inline uint64_t round_up(uint64_t a, uint64_t to) { return ceil_div(a, to) * to; }
// a grid's first side, whose threads may not pass 32 bits
constexpr uint64_t grid_most(uint32_t threads) { return 0xFFFFFFFFull / threads; }

// The cache's sizes (and with `pools` its pointers) checked, as the kernels
// take them.
inline int paged_check(const catena_paged_kv_t* kv, bool pools, PagedKv* out) {
  if (!kv) return fail(CATENA_ERR_INVALID_ARGUMENT, "null cache");
  const uint32_t ps = kv->page_size;
  if (ps < 16 || ps > 1024 || (ps & (ps - 1)) != 0)
    return fail(CATENA_ERR_UNSUPPORTED, "page_size %u is not a power of two from 16 to 1024", ps);
  if (kv->head_dim != 64 && kv->head_dim != 128)
    return fail(CATENA_ERR_UNSUPPORTED, "paged cache head_dim %u unsupported (64 or 128)", kv->head_dim);
  if (kv->kv_heads == 0 || kv->num_pages == 0 || kv->max_pages == 0)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "paged cache of %u heads, %u pages, %u table entries a row",
                kv->kv_heads, kv->num_pages, kv->max_pages);
  if (kv->kv_heads > 65535 || (uint64_t)kv->max_pages * ps > 0x7FFFFFFFull)
    return fail(CATENA_ERR_UNSUPPORTED, "paged cache too large");
  // bytes of a pool, so that no offset passes 64 bits
  if ((uint64_t)kv->num_pages * kv->kv_heads > (1ull << 44))
    return fail(CATENA_ERR_UNSUPPORTED, "paged cache too large");
  if (pools && kv->rows > 0) {
    if (!kv->k || !kv->v || !kv->table) return fail(CATENA_ERR_INVALID_ARGUMENT, "null page pool or table");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->table, 4))
      return fail(CATENA_ERR_INVALID_ARGUMENT, "page pools must be 16-byte aligned");
  }
  uint32_t shift = 0;
  while ((1u << shift) < ps) ++shift;
  *out = PagedKv{kv->k, kv->v, kv->table, kv->num_pages, shift, kv->rows, kv->max_pages, kv->kv_heads, kv->head_dim};
  return CATENA_OK;
}

constexpr uint64_t kJoinBlocks = 2048;  // eight a CU; they take several rows each
struct AttnPagedPlan {
  uint32_t group, head_tiles, blocks, short_slots, pieces;
  uint64_t part_ml, whole_ml, scores, bytes;  // offsets and the sum; part_o comes first
};

inline int attn_paged_plan(const PagedKv& kv, uint32_t heads, bool weights, AttnPagedPlan* p,
                           bool four_bits = false) {
  if (heads == 0 || heads % kv.kv_heads != 0)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "%u query heads over %u kv heads", heads, kv.kv_heads);
  p->group = heads / kv.kv_heads;
  p->head_tiles = (uint32_t)ceil_div(p->group, 16);
  const uint64_t slots = paged_slots(kv), pairs = (uint64_t)kv.rows * kv.kv_heads, units = pairs * p->head_tiles;
  const uint64_t tiles = units * ceil_div(slots, 32);
  // (a grid's second side is 65535 at most: 4 pieces a head of a kv head, and with
  // weights a strip for every 1024 slots)
  if (units > 0x7FFFFFFull || tiles > 0x7FFFFFFFull || 4ull * p->group + (weights ? slots / 1024 + 1 : 0) > 65535)
    return fail(CATENA_ERR_UNSUPPORTED, "too many rows, heads and slots");
  // Whole units while a row's slots take no longer than cutting them costs: a row
  // at one CU's 38 GB/s against a join and, the more units there are, their short
  // parts.  Units x slots of 128 (ragged from 256 on), a workgroup a unit / cut, us:
  // 16 x 384 6.7 / 8.0, x 512 7.9 / 8.0, x 2048 28.5 / 9.4; 64 x 512 10.1 / 9.0; 128 x
  // 640 12.8 / 13.0; 256 x 1024 18.0 / 25.5, x 1536 25.9 / 32.9 (a unit for every CU;
  // the bound that this gives 129 to 256 units is too high for the fewer of them, and
  // for few full rows among short ones: 136 units x 1952 32.7 / 28.1, of which one row's
  // 8 are full and the others 64 slots 27.5 / 11.3; 192 35.1 / 36.3, 28.0 / 11.4);
  // 512 x 1024 32.6 / 37, x 1536 47.7 / 44.7, x 4096 119 / 89; 1024 x 2048 97 / 101, x
  // 4096 209 / 178; 2048 x 2048 191 / 214, x 4096 364 / 356.
  // Where a full table is that short, a workgroup per unit and no second kernel
  // (which weights of several units of one kv head need all the same); else two
  // workgroups a CU at most (one where a long table's few units fill no more), no
  // fewer than four tiles each, and both kernels apply the rule to the longest row
  // that they find: 64 rows x 8 heads in tables of 4096 slots, 1 .. 100 of them in
  // use 8.6 us (cut 16), 1 .. 300 14.3 (27), 1 .. 600 22 (32).
  const uint64_t short_row = units > 128 && units <= 256 ? 1000000 : 230000 + 850 * units;
  p->short_slots = (uint32_t)std::min<uint64_t>(short_row / (kv.head_dim * 4), slots);
  if (p->short_slots == slots && !(weights && p->head_tiles > 1))
    p->blocks = 0;
  else
    p->blocks = (uint32_t)std::min<uint64_t>(tiles >= 16384 && units <= 256 ? 256 : 512, ceil_div(tiles, 4));
  if (four_bits) {
    // a table that never holds a row to cut: one row alone is the first
    const uint64_t longest = ceil_div(slots, kAttnQ4Slots), all = units * longest;
    const uint64_t alone = (uint64_t)kv.kv_heads * p->head_tiles * longest;
    const bool whole = longest <= kAttnQ4WholeMost && longest * kAttnQ4WholeShare <= alone + 2 * kAttnQ4WholeShare;
    p->blocks = whole ? 0 : (uint32_t)std::min<uint64_t>(kv.head_dim == 64 && all >= kAttnQ4TwoACu ? 768 : 512, all);
  }
  // the join by a unit's number of parts: a thread takes all of them, or some, or
  // some of a quarter of the columns (1 part a unit 5.0 / 6.6 us, 5 parts 4.5 / 3.7 /
  // 4.6, 64 parts - / 26 / 5)
  p->pieces = p->blocks <= 2 * units ? 0 : p->blocks <= 16 * units ? 1 : 4;
  const uint64_t parts = 2ull * p->blocks * std::min(p->group, 16u);
  p->part_ml = parts * kv.head_dim * 4;
  p->whole_ml = p->part_ml + parts * 8;
  p->scores = round_up(p->whole_ml + (weights && p->blocks ? pairs * p->group * 8 : 0), 16);
  p->bytes = p->scores + (weights ? pairs * p->group * slots * 4 : 0);
  return CATENA_OK;
}

}  // namespace catena
