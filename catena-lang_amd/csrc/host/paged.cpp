// Kernel ABI of the key-value cache in pages (attn_paged.hip,
// kv_paged.hip).
//
// Arguments are checked before the device is looked for, so a refused call is
// refused without one.
#include "paged_host.h"

using namespace catena;

namespace {
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
