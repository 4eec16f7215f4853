// Kernel ABI of a step over requests of different lengths: pages and slot maps
// (kv_admit.hip), packed rotation into a cache in pages (rope_packed.hip), causal
// attention of packed sequences (attn_prompt.hip), a cache held in 4 bits
// (attn_paged_q4.hip).
//
// Arguments are checked before the device is looked for, so a refused call is
// refused without one.
#include <cmath>

#include "paged_host.h"

using namespace catena;

namespace {
int paged4_check(const catena_paged_kv4_t* kv, bool pools, PagedKv4* out) {
  if (!kv) return fail(CATENA_ERR_INVALID_ARGUMENT, "null cache");
  const catena_paged_kv_t sizes{nullptr, nullptr, nullptr, kv->num_pages, kv->page_size, kv->rows, kv->max_pages,
                                kv->kv_heads, kv->head_dim};
  PagedKv c;
  const int st = paged_check(&sizes, false, &c);
  if (st) return st;
  if (pools && kv->rows > 0) {
    if (!kv->k || !kv->v || !kv->k_scale || !kv->v_scale || !kv->table)
      return fail(CATENA_ERR_INVALID_ARGUMENT, "null page pool or table");
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16) || !aligned(kv->k_scale, 16) || !aligned(kv->v_scale, 16) ||
        !aligned(kv->table, 4))
      return fail(CATENA_ERR_INVALID_ARGUMENT, "page pools must be 16-byte aligned");
  }
  *out = PagedKv4{kv->k, kv->v, kv->k_scale, kv->v_scale, kv->table, c.num_pages, c.page_shift, c.rows, c.max_pages,
                  c.kv_heads, c.head_dim};
  return CATENA_OK;
}

int rope_packed_check(uint32_t kv_heads, uint32_t dim, const void* qkv, const float* rope_tab, uint32_t positions,
                      uint32_t rot, const uint32_t* token_pos, const uint64_t* slot_map, const uint16_t* q,
                      const uint16_t* k_out, const uint16_t* v_out, uint64_t tokens, uint32_t heads) {
  if (heads == 0 || heads % kv_heads != 0)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "%u query heads over %u kv heads", heads, kv_heads);
  if (rot == 0 || rot % 16 != 0 || rot > dim)
    return fail(CATENA_ERR_UNSUPPORTED, "rotary_dim %u is not a multiple of 16 up to head_dim %u", rot, dim);
  if ((k_out != nullptr) != (v_out != nullptr))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "copies of keys and values come together");
  // (a workgroup's threads take runs of 16 values of a token in turn, up to 8 a head: their number, with a turn
  // past it, stay below 2^32)
  if (tokens > grid_most(256) || (uint64_t)heads + 2ull * kv_heads > (0xFFFFFFFFull - 256) / 8)
    return fail(CATENA_ERR_UNSUPPORTED, "packed rotation too large");
  if (tokens == 0) return CATENA_OK;
  if (!qkv || !rope_tab || !token_pos || !q) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (positions == 0) return fail(CATENA_ERR_INVALID_ARGUMENT, "empty rotation table");
  if (!aligned(qkv, 16) || !aligned(rope_tab, 16) || !aligned(q, 16) || !aligned(k_out, 16) || !aligned(v_out, 16) ||
      !aligned(token_pos, 4) || !aligned(slot_map, 8))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "packed rotation needs 16-byte aligned qkv, rope_tab and outputs");
  return CATENA_OK;
}

struct PromptPlan {
  uint32_t units;   // of 256 query rows of a row and kv head, at most
  bool list;        // dealt out from a list, long ones first and cut
  uint32_t items, splits, part_rows;
  uint64_t splits_at, ml_at, o_at, bytes;  // in the workspace: counts, items, splits, part_ml, part_o
};
// slots: of a row, at most
int prompt_plan(uint32_t rows, uint64_t tokens, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint64_t slots,
                PromptPlan* p) {
  if (heads == 0 || kv_heads == 0 || heads % kv_heads != 0)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "%u query heads over %u kv heads", heads, kv_heads);
  const uint32_t group = heads / kv_heads;
  if (tokens > 0x7FFFFFFFull || rows > 0x7FFFFFFFu || kv_heads > 65535)
    return fail(CATENA_ERR_UNSUPPORTED, "too many tokens, rows or heads");
  if (tokens * group > 0x7FFFFFFFull) return fail(CATENA_ERR_UNSUPPORTED, "too many tokens and heads");
  const uint64_t units = tokens * group / 256 + std::min<uint64_t>(rows, tokens);
  if (units * kv_heads > grid_most(512)) return fail(CATENA_ERR_UNSUPPORTED, "too many tokens, rows and heads");
  p->units = (uint32_t)units;
  // A list costs two more launches, and spares every workgroup of many the search for its unit: rows that may have no
  // more than 1024 slots, direct / listed, us: 8 prompts of up to 500 tokens 48 / 61, 32 of them 147 / 150, 6 beside 250
  // single tokens 116 / 90; single tokens, 256 of them 109 / 68, 1024 454 / 204, 4096 2427 / 503 (all with p in one term, 1 to 2 % less
  // than single tokens take in two).
  p->list = slots > 1024 || units > 256;
  p->bytes = 0;
  if (!p->list) return CATENA_OK;
  p->items = p->units + kPromptParts;
  p->splits = (uint32_t)std::min<uint64_t>(units, std::max(1u, kPromptParts / 2 / kv_heads));
  p->part_rows = (uint32_t)std::min<uint64_t>(kPromptNarrow, tokens * group);
  p->splits_at = kPromptCountBytes + (uint64_t)p->items * sizeof(PromptItem);
  p->ml_at = p->splits_at + (uint64_t)p->splits * sizeof(PromptItem);
  p->o_at = p->ml_at + (uint64_t)kPromptParts * p->part_rows * 8;
  p->bytes = p->o_at + (uint64_t)kPromptParts * p->part_rows * head_dim * 4;
  return CATENA_OK;
}
int prompt_launch(AttnPromptArgs a, bool paged, const PromptPlan& p, void* workspace) {
  const bool d64 = a.kv.head_dim == 64;
  const KernelId id = paged ? (d64 ? KernelId::AttnPromptD64 : KernelId::AttnPromptD128)
                            : (d64 ? KernelId::AttnPackedD64 : KernelId::AttnPackedD128);
  const size_t lds = 8 * 32 * (a.kv.head_dim * 4 + 8);  // the waves' results; the tiles take less
  void* args[] = {&a};
  if (!p.list) return launch(id, dim3(p.units * a.kv.kv_heads), dim3(512), lds, args);
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  static_assert(sizeof(PromptCounts) <= kPromptCountBytes, "the list's place");
  a.counts = reinterpret_cast<PromptCounts*>(ws);
  a.items = reinterpret_cast<PromptItem*>(ws + kPromptCountBytes);
  a.splits = reinterpret_cast<PromptItem*>(ws + p.splits_at);
  a.part_ml = reinterpret_cast<float*>(ws + p.ml_at);
  a.part_o = reinterpret_cast<float*>(ws + p.o_at);
  a.part_rows = p.part_rows;
  a.max_items = p.items;
  a.max_splits = p.splits;
  int st = launch(paged ? KernelId::AttnPromptList : KernelId::AttnPackedList, dim3(1), dim3(1024), 0, args);
  if (!st) st = launch(id, dim3(kPromptCus), dim3(512), lds, args);
  if (st) return st;
  return launch(d64 ? KernelId::AttnPromptJoinD64 : KernelId::AttnPromptJoinD128, dim3(std::min(p.splits, std::max(1u, 256 / a.kv.kv_heads)), a.kv.kv_heads, 16),
                dim3(256), 0, args);
}
// The scale as the kernels take it: above 0, a negative one's sign to q
struct Scale {
  float log2;
  uint32_t flip;
};
Scale scale_of(float scale) {
  // (0 would meet the -inf of what is not seen: the least normal number instead, which
  // leaves the scores of any values below 2^100 apart by nothing that f32 keeps)
  return Scale{scale == 0 ? 0x1p-126f : (float)(std::fabs((double)scale) * 1.4426950408889634),
               scale < 0 ? 0x80008000u : 0u};
}
void prompt_scale(float scale, AttnPromptArgs* a) {
  const Scale s = scale_of(scale);
  a->scale_log2 = s.log2;
  a->flip = s.flip;
}
}  // namespace

extern "C" {

int catena_mi355x_kv_admit_paged(const catena_paged_kv_t* kv, uint32_t* table, const uint32_t* lens,
                                 const uint32_t* held, const uint32_t* want, const uint32_t* free_pages,
                                 const uint32_t* free_count, uint32_t* lens_out, uint32_t* held_out, uint32_t* starts,
                                 uint32_t* free_count_out, uint32_t* token_pos, uint64_t* slot_map,
                                 uint32_t max_tokens, const uint32_t* seen, uint32_t* seen_out) {
  PagedKv c;
  const int st = paged_check(kv, false, &c);
  if (st) return st;
  if ((seen != nullptr) != (seen_out != nullptr))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "counted positions need an input and an output");
  if (c.rows > 0x7FFFFFFFu || max_tokens > 0x7FFFFFFFu) return fail(CATENA_ERR_UNSUPPORTED, "too many rows or tokens");
  if (!free_count || !starts || !free_count_out) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (c.rows > 0 && (!table || !lens || !held || !want || !free_pages || !lens_out || !held_out))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (max_tokens > 0 && (!token_pos || !slot_map)) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  const void* words[] = {table,    lens,   held,           want,      free_pages, free_count, lens_out,
                         held_out, starts, free_count_out, token_pos, seen,       seen_out};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(CATENA_ERR_INVALID_ARGUMENT, "misaligned operand");
  if (!aligned(slot_map, 8)) return fail(CATENA_ERR_INVALID_ARGUMENT, "misaligned operand");
  // every workgroup reads the inputs
  const void* in[] = {lens, held, want, free_pages, free_count, seen};
  const void* out[] = {table, lens_out, held_out, starts, free_count_out, token_pos, slot_map, seen_out};
  for (const void* x : in)
    for (const void* y : out)
      if (x && x == y) return fail(CATENA_ERR_INVALID_ARGUMENT, "the outputs of admission may not replace its inputs");
  const int init = ensure_init();
  if (init) return init;
  AdmitArgs a{c.rows, c.max_pages, c.page_shift,   c.num_pages, table,    lens,     held,   want,
              seen,   free_pages,  free_count,     lens_out,    held_out, seen_out, starts, free_count_out,
              token_pos, slot_map, max_tokens};
  void* args[] = {&a};
  const unsigned blocks = (unsigned)std::min<uint64_t>(256, std::max<uint64_t>(1, ceil_div(max_tokens, 1024)));
  return launch(KernelId::KvAdmit, dim3(blocks), dim3(256), 0, args);
}

int catena_mi355x_kv_release_paged(const catena_paged_kv_t* kv, uint32_t* table, const uint32_t* lens,
                                   const uint32_t* held, const uint32_t* finished, uint32_t* free_pages,
                                   const uint32_t* free_count, uint32_t* lens_out, uint32_t* held_out,
                                   uint32_t* free_count_out) {
  PagedKv c;
  const int st = paged_check(kv, false, &c);
  if (st) return st;
  // (the pages given back are counted in 32 bits)
  if (c.rows > 0x7FFFFFFFu || (uint64_t)c.rows * c.max_pages > 0xFFFFFFFFull)
    return fail(CATENA_ERR_UNSUPPORTED, "too many rows and pages");
  if (!free_count || !free_count_out) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (c.rows > 0 && (!table || !lens || !held || !finished || !free_pages || !lens_out || !held_out))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  const void* words[] = {table, lens, held, finished, free_pages, free_count, lens_out, held_out, free_count_out};
  for (const void* p : words)
    if (!aligned(p, 4)) return fail(CATENA_ERR_INVALID_ARGUMENT, "misaligned operand");
  const void* in[] = {lens, held, finished, free_count};
  const void* out[] = {table, lens_out, held_out, free_pages, free_count_out};
  for (const void* x : in)
    for (const void* y : out)
      if (x && x == y) return fail(CATENA_ERR_INVALID_ARGUMENT, "the outputs of release may not replace its inputs");
  const int init = ensure_init();
  if (init) return init;
  ReleaseArgs a{c.rows, c.max_pages, c.num_pages, table, lens, held, finished, free_pages, free_count, lens_out,
                held_out, free_count_out};
  void* args[] = {&a};
  const uint64_t most = std::min<uint64_t>((uint64_t)c.rows * c.max_pages, c.num_pages);
  const unsigned blocks = (unsigned)std::min<uint64_t>(64, std::max<uint64_t>(1, ceil_div(most, 1024)));
  return launch(KernelId::KvRelease, dim3(blocks), dim3(256), 0, args);
}

int catena_mi355x_rope_inv_freq_scaled(double* out_host, uint32_t rotary_dim, double base, uint32_t kind,
                                       double factor, double trained, double low, double high) {
  if (!out_host) return fail(CATENA_ERR_INVALID_ARGUMENT, "null output");
  if (rotary_dim == 0 || rotary_dim % 2 != 0)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "rotary_dim %u is not even", rotary_dim);
  if (!(base > 0) || !std::isfinite(base)) return fail(CATENA_ERR_INVALID_ARGUMENT, "base must be above 0");
  if (kind > CATENA_ROPE_PARTS) return fail(CATENA_ERR_UNSUPPORTED, "unknown kind of scaling %u", kind);
  if (kind != CATENA_ROPE_PLAIN && (!(factor > 0) || !std::isfinite(factor)))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "factor must be above 0");
  if (kind == CATENA_ROPE_BASE && rotary_dim < 4)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "a raised base needs two frequencies");
  if (kind == CATENA_ROPE_PARTS && (!(trained > 0) || !(low >= 0) || !(high > low) || !std::isfinite(high)))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "scaling by parts needs a trained length and 0 <= low < high");
  const double d = rotary_dim;
  if (kind == CATENA_ROPE_BASE) base *= std::pow(factor, d / (d - 2));
  for (uint32_t i = 0; i < rotary_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * i / d);
    if (kind == CATENA_ROPE_LINEAR) f /= factor;
    if (kind == CATENA_ROPE_PARTS) {
      const double turns = trained * f / (2 * M_PI);
      const double keep = std::min(1.0, std::max(0.0, (turns - low) / (high - low)));
      f = keep * f + (1 - keep) * f / factor;
    }
    out_host[i] = f;
  }
  return CATENA_OK;
}

int catena_mi355x_rope_table_scaled_f32(const double* inv_freq, float* tab, uint32_t first, uint32_t positions,
                                        uint32_t rotary_dim, double mscale) {
  if (rotary_dim == 0 || rotary_dim % 2 != 0)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "rotary_dim %u is not even", rotary_dim);
  if (positions == 0) return CATENA_OK;
  if (!inv_freq || !tab) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (!aligned(inv_freq, 8) || !aligned(tab, 8)) return fail(CATENA_ERR_INVALID_ARGUMENT, "misaligned operand");
  if ((uint64_t)first + positions > 0xFFFFFFFFull) return fail(CATENA_ERR_UNSUPPORTED, "positions past 32 bits");
  uint32_t half = rotary_dim / 2;
  const uint64_t blocks = ceil_div((uint64_t)positions * half, 256);
  if (blocks > grid_most(256)) return fail(CATENA_ERR_UNSUPPORTED, "rotation table too large");
  const int st = ensure_init();
  if (st) return st;
  void* args[] = {&inv_freq, &tab, &first, &positions, &half, &mscale};
  return launch(KernelId::RopeTableF64, dim3((unsigned)blocks), dim3(256), 0, args);
}

int catena_mi355x_rope_packed_bf16(const catena_paged_kv_t* kv, const void* qkv, int qkv_f32, const float* rope_tab,
                                   uint32_t table_positions, uint32_t rotary_dim, int interleaved,
                                   const uint32_t* token_pos, const uint64_t* slot_map, uint16_t* q, uint64_t tokens,
                                   uint32_t heads, uint16_t* k_out, uint16_t* v_out) {
  PagedKv c;
  int st = paged_check(kv, false, &c);
  if (!st)
    st = rope_packed_check(c.kv_heads, c.head_dim, qkv, rope_tab, table_positions, rotary_dim, token_pos, slot_map, q,
                           k_out, v_out, tokens, heads);
  if (st || tokens == 0) return st;
  if (slot_map && (!c.k || !c.v || !aligned(c.k, 16) || !aligned(c.v, 16)))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "page pools must be there, 16-byte aligned");
  st = ensure_init();
  if (st) return st;
  RopePackedArgs a{qkv, rope_tab, token_pos, slot_map, q, k_out, v_out, table_positions, rotary_dim,
                   interleaved ? 1u : 0u, heads};
  void* args[] = {&c, &a};
  return launch(qkv_f32 ? KernelId::RopePackedF32 : KernelId::RopePackedBf16, dim3((unsigned)tokens), dim3(256), 0,
                args);
}

int catena_mi355x_rope_packed_q4(const catena_paged_kv4_t* kv, const void* qkv, int qkv_f32, const float* rope_tab,
                                 uint32_t table_positions, uint32_t rotary_dim, int interleaved,
                                 const uint32_t* token_pos, const uint64_t* slot_map, uint16_t* q, uint64_t tokens,
                                 uint32_t heads, uint16_t* k_out, uint16_t* v_out) {
  PagedKv4 c;
  int st = paged4_check(kv, false, &c);
  if (!st)
    st = rope_packed_check(c.kv_heads, c.head_dim, qkv, rope_tab, table_positions, rotary_dim, token_pos, slot_map, q,
                           k_out, v_out, tokens, heads);
  if (st) return st;
  if (c.kv_heads > 128) return fail(CATENA_ERR_UNSUPPORTED, "more than 128 kv heads in 4 bits");
  if (tokens == 0) return CATENA_OK;
  if (slot_map && (!c.k || !c.v || !c.k_scale || !c.v_scale || !aligned(c.k, 16) || !aligned(c.v, 16) ||
                   !aligned(c.k_scale, 16) || !aligned(c.v_scale, 16)))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "page pools must be there, 16-byte aligned");
  st = ensure_init();
  if (st) return st;
  RopePackedArgs a{qkv, rope_tab, token_pos, slot_map, q, k_out, v_out, table_positions, rotary_dim,
                   interleaved ? 1u : 0u, heads};
  void* args[] = {&c, &a};
  return launch(qkv_f32 ? KernelId::RopePackedQ4F32 : KernelId::RopePackedQ4Bf16, dim3((unsigned)tokens), dim3(256),
                4ull * c.kv_heads * c.head_dim, args);
}

int catena_mi355x_attn_prompt_plan(const catena_paged_kv_t* kv, uint64_t tokens, uint32_t heads,
                                   uint64_t* workspace_bytes) {
  if (!workspace_bytes) return fail(CATENA_ERR_INVALID_ARGUMENT, "null output");
  PagedKv c;
  PromptPlan p;
  int st = paged_check(kv, false, &c);
  if (!st) st = prompt_plan(c.rows, tokens, heads, c.kv_heads, c.head_dim, paged_slots(c), &p);
  if (!st) *workspace_bytes = p.bytes;
  return st;
}

int catena_mi355x_attn_prompt_bf16(const catena_paged_kv_t* kv, const uint16_t* q, const uint32_t* starts,
                                   const uint32_t* lens, uint16_t* o, uint64_t tokens, uint32_t heads, float scale,
                                   void* workspace, uint64_t workspace_bytes) {
  AttnPromptArgs a{};
  PromptPlan p;
  int st = paged_check(kv, true, &a.kv);
  if (!st) st = prompt_plan(a.kv.rows, tokens, heads, a.kv.kv_heads, a.kv.head_dim, paged_slots(a.kv), &p);
  if (st || a.kv.rows == 0 || tokens == 0) return st;
  if (!q || !starts || !lens || !o) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (!aligned(q, 16) || !aligned(o, 16) || !aligned(starts, 4) || !aligned(lens, 4))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "prompt attention needs 16-byte aligned q and o");
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || !aligned(workspace, 16)))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "prompt attention needs %llu bytes of 16-byte aligned workspace",
                (unsigned long long)p.bytes);
  st = ensure_init();
  if (st) return st;
  a.q = q;
  a.starts = starts;
  a.lens = lens;
  a.o = o;
  a.tokens = (uint32_t)tokens;
  a.group = heads / a.kv.kv_heads;
  prompt_scale(scale, &a);
  return prompt_launch(a, true, p, workspace);
}

int catena_mi355x_attn_packed_plan(uint32_t rows, uint64_t tokens, uint32_t heads, uint32_t kv_heads,
                                   uint32_t head_dim, uint64_t* workspace_bytes) {
  if (!workspace_bytes) return fail(CATENA_ERR_INVALID_ARGUMENT, "null output");
  PromptPlan p;
  if (head_dim != 64 && head_dim != 128)
    return fail(CATENA_ERR_UNSUPPORTED, "packed attention head_dim %u unsupported (64 or 128)", head_dim);
  const int st = prompt_plan(rows, tokens, heads, kv_heads, head_dim, tokens, &p);
  if (!st) *workspace_bytes = p.bytes;
  return st;
}

int catena_mi355x_attn_packed_bf16(const uint16_t* q, const uint16_t* k, const uint16_t* v, const uint32_t* starts,
                                   uint16_t* o, uint32_t rows, uint64_t tokens, uint32_t heads, uint32_t kv_heads,
                                   uint32_t head_dim, uint64_t kv_stride, float scale, void* workspace,
                                   uint64_t workspace_bytes) {
  AttnPromptArgs a{};
  PromptPlan p;
  if (head_dim != 64 && head_dim != 128)
    return fail(CATENA_ERR_UNSUPPORTED, "packed attention head_dim %u unsupported (64 or 128)", head_dim);
  int st = prompt_plan(rows, tokens, heads, kv_heads, head_dim, tokens, &p);
  if (st) return st;
  if (kv_stride == 0) kv_stride = (uint64_t)kv_heads * head_dim;
  if (kv_stride < (uint64_t)kv_heads * head_dim || kv_stride % 8 != 0)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "a stride of %llu elements between tokens' keys",
                (unsigned long long)kv_stride);
  if (kv_stride > (1ull << 25)) return fail(CATENA_ERR_UNSUPPORTED, "tokens' keys too far apart");
  if (rows == 0 || tokens == 0) return CATENA_OK;
  if (!q || !k || !v || !starts || !o) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(o, 16) || !aligned(starts, 4))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "packed attention needs 16-byte aligned q, k, v and o");
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || !aligned(workspace, 16)))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "packed attention needs %llu bytes of 16-byte aligned workspace",
                (unsigned long long)p.bytes);
  st = ensure_init();
  if (st) return st;
  a.kv = PagedKv{const_cast<uint16_t*>(k), const_cast<uint16_t*>(v), nullptr, 0, 0, rows, 0, kv_heads, head_dim};
  a.q = q;
  a.starts = starts;
  a.o = o;
  a.stride = kv_stride;
  a.tokens = (uint32_t)tokens;
  a.group = heads / kv_heads;
  prompt_scale(scale, &a);
  return prompt_launch(a, false, p, workspace);
}

int catena_mi355x_attn_paged_q4_plan(const catena_paged_kv4_t* kv, uint32_t heads, uint32_t* parts,
                                     uint64_t* workspace_bytes) {
  if (!parts || !workspace_bytes) return fail(CATENA_ERR_INVALID_ARGUMENT, "null output");
  PagedKv4 c;
  AttnPagedPlan p;
  int st = paged4_check(kv, false, &c);
  if (st) return st;
  const PagedKv sizes{nullptr, nullptr, c.table, c.num_pages, c.page_shift, c.rows, c.max_pages, c.kv_heads, c.head_dim};
  st = attn_paged_plan(sizes, heads, false, &p, true);
  if (st) return st;
  *parts = p.blocks;
  *workspace_bytes = p.bytes;
  return CATENA_OK;
}

int catena_mi355x_attn_paged_q4(const catena_paged_kv4_t* kv, const uint16_t* q, const uint32_t* lens, uint16_t* o,
                                uint32_t heads, float scale, void* workspace, uint64_t workspace_bytes) {
  PagedKv4 c;
  AttnPagedArgs a{};
  AttnPagedPlan p;
  int st = paged4_check(kv, true, &c);
  if (st) return st;
  a.kv = PagedKv{nullptr, nullptr, c.table, c.num_pages, c.page_shift, c.rows, c.max_pages, c.kv_heads, c.head_dim};
  st = attn_paged_plan(a.kv, heads, false, &p, true);
  if (st || c.rows == 0) return st;
  if (!q || !lens || !o) return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  if (!aligned(q, 16) || !aligned(o, 16) || !aligned(lens, 4))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "attention over 4 bits needs 16-byte aligned q and o");
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes || !aligned(workspace, 16)))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "attention over 4 bits needs %llu bytes of 16-byte aligned workspace",
                (unsigned long long)p.bytes);
  st = ensure_init();
  if (st) return st;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  a.q = q;
  a.lens = lens;
  a.o = o;
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + p.part_ml);
  a.group = p.group;
  a.head_tiles = p.head_tiles;
  a.blocks = p.blocks;
  a.short_slots = p.short_slots;
  const Scale s = scale_of(scale);
  a.scale_log2 = s.log2;
  AttnQ4Pools pools{c.k, c.v, c.k_scale, c.v_scale, s.flip};
  const uint64_t pairs = (uint64_t)c.rows * c.kv_heads;
  void* args[] = {&a, &pools};
  const KernelId id = c.head_dim == 64 ? (p.group <= 8 ? KernelId::AttnPagedQ4D64 : KernelId::AttnPagedQ4D64Wide)
                                       : (p.group <= 8 ? KernelId::AttnPagedQ4D128 : KernelId::AttnPagedQ4D128Wide);
  // (a workgroup a unit also where units may be cut: what there is not to do for one it leaves)
  const uint64_t grid = std::min(std::max<uint64_t>(pairs * p.head_tiles, p.blocks), grid_most(256));
  st = launch(id, dim3((unsigned)grid), dim3(256), 0, args);
  if (st || p.blocks == 0) return st;
  uint32_t pieces = p.pieces;
  const uint64_t joins = pieces ? (uint64_t)p.group * pieces : ceil_div((uint64_t)p.group * c.head_dim, 1024);
  const uint64_t rows = std::min<uint64_t>(c.rows, std::max<uint64_t>(1, kJoinBlocks / (joins * c.kv_heads)));
  void* jargs[] = {&a, &pieces};
  return launch(c.head_dim == 64 ? KernelId::AttnPagedQ4JoinD64 : KernelId::AttnPagedQ4JoinD128,
                dim3(c.kv_heads, (unsigned)joins, (unsigned)rows), dim3(256), 0, jargs);
}

}  // extern "C"
