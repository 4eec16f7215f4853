// Kernel ABI of the key-value cache in pages (attn_paged.hip,
// kv_paged.hip).
//
// Arguments are checked before the device is looked for, so a refused call is
// refused without one.
#include <algorithm>
#include <cstdint>

#include "../kernels/paged.h"
#include "internal.h"

using namespace catena;

namespace {
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
uint64_t round_up(uint64_t a, uint64_t to) { return ceil_div(a, to) * to; }
// a grid's first side, whose threads may not pass 32 bits
constexpr uint64_t grid_most(uint32_t threads) { return 0xFFFFFFFFull / threads; }

// The cache's sizes (and with `pools` its pointers) checked, as the kernels
// take them.
int paged_check(const catena_paged_kv_t* kv, bool pools, PagedKv* out) {
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

int attn_paged_plan(const PagedKv& kv, uint32_t heads, bool weights, AttnPagedPlan* p) {
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

constexpr uint32_t kEvictAtOnce = 128;  // moves that its lists in LDS hold
constexpr uint32_t kEvictMoves = 64;  // a workgroup of catena_kv_evict_move
// Most moves of a (row, kv head): slots below the budget, and slots from it on
uint32_t evict_most(const PagedKv& kv, uint32_t budget) {
  const uint32_t slots = paged_slots(kv);
  return budget >= slots ? 0 : std::min(budget, slots - budget);
}
// a workgroup for a (row, kv head): small while that holds the table (tables of 528
// slots, one too many, 8 rows x 16 heads 4.3 us against 4.6, 64 rows 5.0 / 15.7)
uint32_t evict_threads(const PagedKv& kv) { return paged_slots(kv) <= 1024 ? 256 : 1024; }
// count[pairs], holes[pairs][most], sources[pairs][most]
int evict_plan(const PagedKv& kv, uint32_t budget, uint64_t* bytes) {
  if (budget == 0) return fail(CATENA_ERR_INVALID_ARGUMENT, "a budget of no slots");
  const uint64_t pairs = (uint64_t)kv.rows * kv.kv_heads;
  if (pairs > grid_most(evict_threads(kv))) return fail(CATENA_ERR_UNSUPPORTED, "too many rows and heads");
  if (evict_most(kv, budget) > 65535 * kEvictMoves) return fail(CATENA_ERR_UNSUPPORTED, "eviction of too many slots");
  *bytes = pairs * 4 * (1 + 2ull * evict_most(kv, budget));
  return CATENA_OK;
}

constexpr uint32_t kReorderFew = 8, kReorderMost = 128;
}  // namespace

extern "C" {

int catena_mi355x_attn_paged_plan(const catena_paged_kv_t* kv, uint32_t heads, int weights, uint32_t* parts,
                                  uint64_t* workspace_bytes) {
  if (!parts || !workspace_bytes) return fail(CATENA_ERR_INVALID_ARGUMENT, "null output");
  PagedKv c;
  AttnPagedPlan p;
  int st = paged_check(kv, false, &c);
  if (!st) st = attn_paged_plan(c, heads, weights != 0, &p);
  if (st) return st;
  *parts = p.blocks;
  *workspace_bytes = p.bytes;
  return CATENA_OK;
}

int catena_mi355x_attn_paged_bf16(const catena_paged_kv_t* kv, const uint16_t* q, const uint32_t* lens, void* o,
                                  uint32_t heads, float scale, int out_f32, const float* acc_in, float* acc_out,
                                  void* workspace, uint64_t workspace_bytes) {
  AttnPagedArgs a{};
  AttnPagedPlan p;
  int st = paged_check(kv, true, &a.kv);
  if (!st) st = attn_paged_plan(a.kv, heads, acc_out != nullptr, &p);
  if (st) return st;
  if ((acc_in != nullptr) != (acc_out != nullptr))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "accumulated weights need an input and an output");
  if (a.kv.rows == 0) return CATENA_OK;
  if (!q || !lens || !o) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (!aligned(q, 16) || !aligned(o, 16) || !aligned(lens, 4) || !aligned(acc_in, 4) || !aligned(acc_out, 4))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "paged attention needs 16-byte aligned q and o");
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || !aligned(workspace, 16)))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "paged attention needs %llu bytes of 16-byte aligned workspace",
                (unsigned long long)p.bytes);
  st = ensure_init();
  if (st) return st;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  a.q = q;
  a.lens = lens;
  a.o = o;
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + p.part_ml);
  a.whole_ml = reinterpret_cast<float*>(ws + p.whole_ml);
  a.scores = reinterpret_cast<float*>(ws + p.scores);
  a.acc_in = acc_in;
  a.acc_out = acc_out;
  a.group = p.group;
  a.head_tiles = p.head_tiles;
  a.blocks = p.blocks;
  a.short_slots = p.short_slots;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  // kernels in the order of their ids: D128 f32, D128 bf16, D64 f32, D64 bf16
  const int form = (a.kv.head_dim == 64 ? 2 : 0) + (out_f32 ? 0 : 1);
  const uint64_t pairs = (uint64_t)a.kv.rows * a.kv.kv_heads;
  const KernelId first = acc_out ? KernelId::AttnPagedWeightsD128F32 : KernelId::AttnPagedD128F32;
  void* args[] = {&a};
  st = launch(static_cast<KernelId>(static_cast<int>(first) + form),
              dim3(p.blocks ? p.blocks : (unsigned)std::min(pairs * p.head_tiles, grid_most(256))), dim3(256), 0, args);
  if (st || p.blocks == 0) return st;
  uint32_t pieces = p.pieces;
  const uint64_t joins = pieces ? (uint64_t)p.group * pieces : ceil_div((uint64_t)p.group * a.kv.head_dim, 1024);
  const uint64_t items = joins + (acc_out ? ceil_div(paged_slots(a.kv), 1024) : 0);
  const uint64_t rows = std::min<uint64_t>(a.kv.rows, std::max<uint64_t>(1, kJoinBlocks / (items * a.kv.kv_heads)));
  void* jargs[] = {&a, &pieces};
  return launch(static_cast<KernelId>(static_cast<int>(KernelId::AttnPagedJoinD128F32) + form),
                dim3(a.kv.kv_heads, (unsigned)items, (unsigned)rows), dim3(256), 0, jargs);
}

int catena_mi355x_rope_qkv_paged_bf16(const catena_paged_kv_t* kv, const float* qkv, const float* rope_tab,
                                      uint32_t table_positions, const uint32_t* lens, const uint32_t* seen,
                                      uint16_t* q, uint32_t tq, uint32_t heads, float* acc, uint32_t* slot_pos) {
  PagedKv c;
  int st = paged_check(kv, true, &c);
  if (st) return st;
  if (heads == 0 || heads % c.kv_heads != 0)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "%u query heads over %u kv heads", heads, c.kv_heads);
  if ((acc != nullptr) != (slot_pos != nullptr))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "a tracked cache has weights and positions");
  const uint64_t tokens = (uint64_t)c.rows * tq;
  if (tokens == 0) return CATENA_OK;
  if (!qkv || !rope_tab || !lens || !q) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (table_positions == 0) return fail(CATENA_ERR_INVALID_ARGUMENT, "empty rotation table");
  if (!aligned(qkv, 16) || !aligned(rope_tab, 16) || !aligned(q, 16) || !aligned(lens, 4) || !aligned(seen, 4) ||
      !aligned(acc, 4) || !aligned(slot_pos, 4))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "paged append needs 16-byte aligned qkv, rope_tab and q");
  const uint64_t blocks = ceil_div(((uint64_t)heads + 2ull * c.kv_heads) * (c.head_dim / 8), 256);
  if (tokens > grid_most(256) || blocks > 65535) return fail(CATENA_ERR_UNSUPPORTED, "paged append too large");
  st = ensure_init();
  if (st) return st;
  void* args[] = {&c, &qkv, &rope_tab, &table_positions, &lens, &seen, &q, &tq, &heads, &acc, &slot_pos};
  return launch(KernelId::RopeQkvPaged, dim3((unsigned)tokens, (unsigned)blocks), dim3(256), 0, args);
}

int catena_mi355x_kv_evict_paged_plan(const catena_paged_kv_t* kv, uint32_t budget, uint64_t* workspace_bytes) {
  if (!workspace_bytes) return fail(CATENA_ERR_INVALID_ARGUMENT, "null output");
  PagedKv c;
  int st = paged_check(kv, false, &c);
  if (!st) st = evict_plan(c, budget, workspace_bytes);
  return st;
}

int catena_mi355x_kv_evict_paged_bf16(const catena_paged_kv_t* kv, const uint32_t* lens, const uint32_t* seen,
                                      const float* acc_in, const uint32_t* slot_pos_in, uint32_t* lens_out,
                                      float* acc_out, uint32_t* slot_pos_out, uint32_t budget, uint32_t recent,
                                      void* workspace, uint64_t workspace_bytes) {
  EvictArgs a{};
  PagedKv& c = a.kv;
  uint64_t need = 0;
  int st = paged_check(kv, true, &c);
  if (!st) st = evict_plan(c, budget, &need);
  if (st) return st;
  if (c.rows == 0) return CATENA_OK;
  if (!lens || !seen || !acc_in || !slot_pos_in || !lens_out || !acc_out || !slot_pos_out)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  const void* words[] = {lens, seen, acc_in, slot_pos_in, lens_out, acc_out, slot_pos_out};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(CATENA_ERR_INVALID_ARGUMENT, "misaligned operand");
  if (!aligned(acc_in, 16) || !aligned(slot_pos_in, 16) || !aligned(acc_out, 16) || !aligned(slot_pos_out, 16))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "eviction needs 16-byte aligned weights and positions");
  if (lens_out == lens || lens_out == seen)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "eviction's new lengths may not replace the old or the positions' count");
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "eviction needs %llu bytes of 16-byte aligned workspace",
                (unsigned long long)need);
  st = ensure_init();
  if (st) return st;
  const uint32_t pairs = c.rows * c.kv_heads, threads = evict_threads(c);
  a.lens = lens;
  a.seen = seen;
  a.acc_in = acc_in;
  a.pos_in = slot_pos_in;
  a.lens_out = lens_out;
  a.acc_out = acc_out;
  a.pos_out = slot_pos_out;
  a.most = evict_most(c, budget);
  a.count = static_cast<uint32_t*>(workspace);
  a.holes = a.count + pairs;
  a.sources = a.holes + (uint64_t)pairs * a.most;
  a.budget = budget;
  a.recent = recent;
  // Few moves are made by the workgroup that chose them, which saves a launch;
  // more by workgroups of 64 each (8 rows x 16 heads of 128, at most 128 moves, of 32
  // slots too many 6.9 us against 9.1, of 64 8.3 / 10.7, of 96 11.0 / 11.2; at most
  // 144, of 128 slots 12.8 / 11.5).
  a.at_once = a.most <= kEvictAtOnce;
  void* args[] = {&a};
  // (kernels of their own where more slots than the budget may be recent: the test
  // for it in the others took 5.7 us instead of 5.4 for one of 5121 slots)
  const KernelId choose = threads == 256
                              ? (recent > budget ? KernelId::KvEvictChoose1kManyRecent : KernelId::KvEvictChoose1k)
                              : (recent > budget ? KernelId::KvEvictChoose8kManyRecent : KernelId::KvEvictChoose8k);
  st = launch(choose, dim3(pairs), dim3(threads), 0, args);
  if (st || a.at_once) return st;
  return launch(KernelId::KvEvictMove, dim3(pairs, (unsigned)ceil_div(a.most, kEvictMoves)), dim3(256), 0, args);
}

int catena_mi355x_beam_reorder_paged_bf16(const catena_paged_kv_t* kv, uint16_t* const* pools, uint32_t n_pools,
                                          const uint32_t* lens, const uint32_t* parents, const uint32_t* spare,
                                          uint32_t* table_out, uint32_t* lens_out, uint32_t* spare_out) {
  PagedKv c;
  int st = paged_check(kv, false, &c);
  if (st) return st;
  if (c.rows == 0) return CATENA_OK;
  if (!c.table || (n_pools > 0 && !pools) || !lens || !parents || !spare || !table_out || !lens_out || !spare_out)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  const void* words[] = {c.table, lens, parents, spare, table_out, lens_out, spare_out};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(CATENA_ERR_INVALID_ARGUMENT, "misaligned operand");
  for (uint32_t i = 0; i < n_pools; ++i)
    if (!pools[i] || !aligned(pools[i], 16))
      return fail(CATENA_ERR_INVALID_ARGUMENT, "page pools must be 16-byte aligned");
  if (table_out == c.table || lens_out == lens || spare_out == spare)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "reorder's outputs may not replace its inputs");
  if (c.rows > grid_most(256)) return fail(CATENA_ERR_UNSUPPORTED, "too many rows");
  st = ensure_init();
  if (st) return st;
  // the pools in as many launches as their pointers need; the table once
  for (uint32_t first = 0; first == 0 || first < n_pools; first += kReorderMost) {
    ReorderArgs a{c, lens, parents, spare, table_out, lens_out, spare_out, std::min(n_pools - first, kReorderMost),
                  first == 0};
    ReorderPools<kReorderMost> p;
    const bool few = a.n_pools <= kReorderFew;
    for (uint32_t i = 0; i < (few ? kReorderFew : kReorderMost); ++i)
      p.p[i] = i < a.n_pools ? pools[first + i] : nullptr;
    void* args[] = {&a, &p};
    st = launch(few ? KernelId::KvReorder8 : KernelId::KvReorder128,
                dim3(c.rows, a.n_pools ? c.kv_heads : 1, a.n_pools ? a.n_pools : 1), dim3(256), 0, args);
    if (st) return st;
  }
  return CATENA_OK;
}

}  // extern "C"
