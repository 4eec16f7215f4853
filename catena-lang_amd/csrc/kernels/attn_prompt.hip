// Causal attention of packed sequences of different lengths, grouped heads, over a
// key-value cache in pages or over packed keys and values.
//
//   token t of row r's n new ones sees the row's first lens[r] - n + t + 1 slots:
//   s_j = scale * q . k_j,  o = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)
//
// Bound: the matrix cores: 4 D flop for each (query head, slot seen), against 4 D
// bytes a slot and kv head that 256 query rows share.  They run at the chip's power limit
// (1.6 GHz of 2.4, matrix instructions in 55 % of the cycles): 11250 to 12000 tokens x 32 heads
// of 128 980 to 1077 us (1.07 PFLOP/s; a large matrix product of random values 1.2 to 1.36 on
// the same cards), 8 ragged prompts of 1024 to 4096 tokens 440 to 700 by their lengths (1.38 to
// 1.49 times the operations' time at 1.31 PFLOP/s); 4 chunks of 469 to 500 tokens and 28
// single ones over up to 8000 slots 203 to 314, half of them above 259 (2.0 to 2.5 times the
// larger of operations and bytes); 5 prompts of up to 130 tokens 7.8 to 9.8.
//
// A workgroup takes 256 query rows of one row and kv head (a unit): query row m is token
// m / group, head m % group of the kv head's, so that short sequences with grouped heads
// fill the rows too, and all rows share K and V.  Each of its eight waves has 32 rows.
// K and V come 64 slots at a time straight to LDS, into rings of three tiles.
//   S^T = K Q^T (32 x 32 x 16 products): lane (c, h) = (lane & 31, lane >> 5) holds
//     query row c's scores of slots 32 b + 8 (i / 4) + 4 h + i % 4 (register i of
//     block b), so the softmax's maximum and sum of a query row need one exchange, and
//     P stays where it is as the second product's operand: the order of slots in the
//     sum is free, and V's operand takes the same.
//   O^T = V^T P^T: V's columns by transposed reads of 4 slots x 16 columns.
// Blocks of 32 slots go through a pipeline of three phases (scores, exponentials, o), so
// that the exponentials of one block run under the products of its neighbours.
//
// Units of up to 64 query rows (single tokens, short chunks) leave most waves without
// rows and wait for memory instead: there each wave takes blocks of 32 slots of its own,
// with its own loads and no barrier, for 32 rows, and the waves' results are joined at
// the end.  Eight waves share a unit; of many such units (2048) two do, and a workgroup
// takes four kv heads' at a time, since what a unit costs besides its loads is latency
// (8 kv heads, 256 single tokens behind up to 400 slots 106 us with eight waves, 68 with
// two, behind up to 4000 407 / 400; of fewer units the larger items end unevenly: 130
// tokens behind up to 4000 251 us with eight waves, 281 with four; p in one term, which was 1
// to 2 % less than in two).
//
// Units are dealt out in one of two ways.  Few short ones: a workgroup each, which finds
// it from the rows' lengths.  Else a kernel before lists them by length, long ones first,
// units above a CU's even share cut into equal parts, and a workgroup a CU takes them
// from the list; a third kernel joins the parts.
//
// The maximum is raised only where a score passes it by more than 8 in base 2, by whole
// numbers, so that what is there is scaled exactly.
// Range: p enters the products times a power of two (and so does the sum, so that it leaves
// again in the division) that keeps those of a row's n slots below half the largest |v|:
// sums of finite values never overflow.  2^-9 / n and not less of it: at the other end
// products below 2^-126 may be lost, 6 n of them (two terms of p, sums between them), which
// the division by 2^-10 / n or more makes n^2 2^-113 of o at most; and an infinity's p must not become 0.
// Rounding: scores, sums and o in f32.  p is rounded to bf16, as the products take it, and
// the sum is that of the rounded ones.  Narrow units, whose products hide under their loads, take p
// in two terms, the upper half of its bits and the rest (2^-16 of p), as attention of one
// token does (256 single tokens 68.8 -> 70.2 us, a mixed step 238 -> 239).  Wide ones would
// take 1.45 times as long (12000 tokens 1102 -> 1611 us, with heads of 64 695 -> 1039), for o off by 1.6e-3
// of itself instead of 2.2e-3, of which its own rounding is 1.6e-3.
// What a query row does not see has p = 0; an infinity or NaN in V there would still
// reach it through the product, so tiles that are not seen whole are searched for
// them, and where there are any they are taken out of the product and entered by
// products of their own that say which sums they reach.
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kWaves = 8;
constexpr uint32_t kRows = kPromptRows, kNarrow = kPromptNarrow;
static_assert(kRows == 32 * kWaves, "a wave's query rows");
constexpr int kKeys = 64;                // slots of a tile
constexpr int kStages = 3;               // tiles of K, and of V, in LDS
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4;
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4;

CATENA_DEV uint32_t lane_of(uint32_t x, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)lane); }
CATENA_DEV float anchor(float m) { return m == kNegInf ? 0.0f : m; }
// Of sums with the reference point m beside others with m2 >= m: never 0, so that an infinity stays one
CATENA_DEV float weight(float m, float m2) {
  return __builtin_fmaxf(__builtin_amdgcn_exp2f(m - anchor(m2)), 0x1p-126f);
}
CATENA_DEV float larger(float x, float y) { return __builtin_elementwise_maximum(x, y); }  // NaN where one is

// Uniform words that this kernel does not write, by scalar loads
CATENA_DEV uint32_t scalar_word(const uint32_t* p, uint64_t i) {
  typedef const uint32_t __attribute__((address_space(4))) * word;
  return ((word)(uintptr_t)p)[i];
}
CATENA_DEV u32x4_t scalar_four(const void* p, uint64_t i) {
  typedef const u32x4_t __attribute__((address_space(4))) * four;
  return ((four)(uintptr_t)p)[i];
}

// l + the two bf16 values of a word
CATENA_DEV float add_pair(uint32_t w, float l) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0x3F803F80u), l, false);
}

// A row's new tokens: first and number, cut to the batch
struct Tokens {
  uint32_t first, n;
};
CATENA_DEV Tokens tokens_of(const AttnPromptArgs& a, uint32_t row) {
  const uint32_t beg = a.starts[row], upto = a.starts[row + 1], end = upto < a.tokens ? upto : a.tokens;
  return Tokens{beg, beg < end ? end - beg : 0u};
}
CATENA_DEV uint32_t units_of(const AttnPromptArgs& a, uint32_t n) {
  return (n * a.group + (kRows - 1)) / kRows;  // (the host sees to it that n * group < 2^31)
}
// Slots of a row in front of its n new tokens; below 0: the first of them see nothing
template <bool PAGED>
CATENA_DEV int32_t old_of(const AttnPromptArgs& a, uint32_t row, uint32_t n) {
  if constexpr (PAGED) return (int32_t)paged_len(a.kv, a.lens[row]) - (int32_t)n;
  return 0;
}
// Slots that the last token of a row's unit sees
CATENA_DEV int32_t most_of(const AttnPromptArgs& a, uint32_t unit, uint32_t n, int32_t old) {
  const uint32_t last = (unit * kRows + (kRows - 1)) / a.group;  // (rows stay below 2^31)
  return old + (int32_t)(last < n ? last + 1 : n);
}
CATENA_DEV uint32_t tiles_of(int32_t slots) { return slots > 0 ? ((uint32_t)slots + kKeys - 1) / kKeys : 0u; }

// Unit `index` of all rows' units in one line, the last (longest) of a row first, as one
// piece; row 0xFFFFFFFF: there is none
template <bool PAGED>
CATENA_DEV PromptItem item_at(const AttnPromptArgs& a, uint32_t index) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t before = 0;
  for (uint32_t r0 = 0; r0 < a.kv.rows; r0 += 64) {
    Tokens t{0, 0};
    int32_t old = 0;
    if (r0 + lane < a.kv.rows) {
      t = tokens_of(a, r0 + lane);
      old = old_of<PAGED>(a, r0 + lane, t.n);
    }
    const uint32_t upto = before + wave_prefix(units_of(a, t.n));
    const uint64_t past = __ballot(upto > index);
    if (past) {
      const uint32_t j = (uint32_t)__ffsll((unsigned long long)past) - 1;
      PromptItem x{r0 + j, lane_of(upto, j) - 1 - index, lane_of(t.first, j), lane_of(t.n, j),
                   (int32_t)lane_of((uint32_t)old, j), 0, 0, kPromptWhole};
      x.end = tiles_of(most_of(a, x.unit, x.n, x.old));
      return x;
    }
    before = lane_of(upto, 63);
  }
  return PromptItem{0xFFFFFFFFu, 0, 0, 0, 0, 0, 0, 0};
}

// (the pools as arguments that nothing else points into: the compiler then does not make reads of LDS wait for
// the loads into it, whose order the barriers below give)
// kvh0: the kv head, or the first of 8 / unit_waves of a narrow unit's.  put, get: called by all threads with a barrier
// between, get in front of the last stores, to look ahead
template <int D, bool PAGED, class Put, class Get>
CATENA_DEV void attn_prompt_item(const AttnPromptArgs& a, const PromptItem& it, uint32_t kvh0, uint32_t unit_waves,
                                 const uint16_t* __restrict__ pool_k, const uint16_t* __restrict__ pool_v,
                                 const Put& put, const Get& get) {
  constexpr int KS = D / 16;        // steps of a score's sum
  constexpr int DB = D / 32;        // blocks of o's columns
  constexpr int kTile = kKeys * D;  // elements of K or V of a tile
  // A tile in LDS: blocks of 16 slots x 32 columns (1 KiB, what one load brings), a run of slots' blocks behind
  // each other.  In a block, K column by column of 16 bytes, V slot by slot: so the reads of a product's operand,
  // 16 slots' 16 bytes of K or 4 slots' 64 bytes of V, lie in all banks, and the operands of all steps a constant apart.
  constexpr int kAcross = D / 32;               // blocks of a run
  constexpr int kLoads = 4 * kAcross / kWaves;  // a wave's blocks, of one run
  constexpr int kWavesARun = kWaves / 4;
  extern __shared__ __attribute__((aligned(1024))) uint16_t smem[];  // K x kStages, V x kStages
  const uint32_t lane = threadIdx.x & 63u, c = lane & 31u, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t heads = a.group * a.kv.kv_heads;
  const uint32_t len = (uint32_t)(it.old + (int32_t)it.n);  // slots in use
  const float ease = (float)(41 - __builtin_clz(len | 1u));   // p's power of two: len of p <= 2^8 stay below 1/2

  // The lane's query row.  Up to 64 rows: one or two blocks of 32 (in turn over the waves, which share out the slots).
  const uint32_t rows_left = it.n * a.group - it.unit * kRows, rows = rows_left < kRows ? rows_left : kRows;
  const bool narrow = rows <= kNarrow;
  const uint32_t blocks = rows <= 32 ? 1 : 2;
  const uint32_t kvh_w = kvh0 + (narrow ? wave / unit_waves : 0u), kvh = min(kvh_w, a.kv.kv_heads - 1);
  const uint32_t w_row = it.unit * kRows + 32 * (narrow ? wave % blocks : wave), m_row = w_row + c, t_row = m_row / a.group;
  const bool live = t_row < it.n;
  const uint64_t q_at =
      ((uint64_t)(it.first + (live ? t_row : 0u)) * heads + kvh * a.group + (live ? m_row % a.group : 0u)) * D;
  const int32_t sees = live ? it.old + (int32_t)t_row + 1 : 0;  // slots
  const uint32_t count = it.end - it.beg;
  // whether any of the wave's rows is live, and the slots that any of them sees
  const bool awake = w_row / a.group < it.n;
  const uint32_t w_last = (w_row + 31) / a.group;
  const int32_t w_most = awake ? it.old + (int32_t)(w_last < it.n ? w_last + 1 : it.n) : 0;

  // Loads: run wave / kWavesARun of a tile, which lies inside one page
  const uint32_t row_bytes = PAGED ? D * 2 : (uint32_t)(a.stride * 2);
  const uint32_t run = wave / kWavesARun, first_block = wave % kWavesARun * kLoads;
  // (a block's 64 bytes of a row by the scalar offset, which the range check leaves out: rows are inside or not)
  const uint32_t k_off = (lane & 15u) * row_bytes + 16 * (lane >> 4), v_off = (lane >> 2) * row_bytes + 16 * (lane & 3u);
  auto page_of = [&](uint32_t slot) -> uint32_t {
    if constexpr (PAGED)
      return slot < len ? scalar_word(a.kv.table, (uint64_t)it.row * a.kv.max_pages + (slot >> a.kv.page_shift)) : 0xFFFFFFFFu;
    return 0;
  };
  // A run of 16 slots: where they are and how many.  Its page is looked up a tile before they are asked for, so that
  // nothing waits for it.
  struct Slots {
    uint64_t at;
    uint32_t n;
  };
  auto slots_at = [&](uint32_t slot, uint32_t page) {
    Slots r{0, slot < len ? (len - slot < 16 ? len - slot : 16u) : 0u};
    if constexpr (PAGED) {
      if (page < a.kv.num_pages)
        r.at = paged_offset(a.kv, page, kvh, slot & ((1u << a.kv.page_shift) - 1u));
      else
        r.n = 0;
    } else {
      r.at = ((uint64_t)it.first + (r.n ? slot : 0u)) * a.stride + kvh * D;
    }
    return r;
  };
  // Blocks first .. first + N - 1 of their K (what 0) or V (1) to LDS
  auto load = [&](const Slots& r, int what, uint32_t first, auto n_, uint16_t* dst) {
    const int bytes = r.n ? (int)((r.n - 1) * row_bytes + D * 2) : 0;
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)((what ? pool_v : pool_k) + r.at), (short)0, bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < n_.value; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(dst + 512 * i), 16, (int)(what ? v_off : k_off),
                                               (int)(64 * (first + i)), 0, 0);
  };
  // The wave's run of the item's tile i
  auto run_slot = [&](uint32_t i) { return (it.beg + i) * kKeys + 16 * run; };
  auto look_up = [&](uint32_t i) { return page_of(run_slot(i)); };
  auto slots_of = [&](uint32_t i, uint32_t page) { return slots_at(run_slot(i), page); };
  auto issue = [&](uint32_t stage, const Slots& r, int what) {
    load(r, what, first_block, std::integral_constant<int, kLoads>{},
         smem + ((what ? kStages : 0) + stage) * kTile + (run * kAcross + first_block) * 512);
  };
  // All that this wave has asked for is in LDS, what it has read of LDS has arrived, and so for the others
  auto arrive = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // The last item's reads of LDS are done with, for all waves
  auto begin = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // The first loads, before anything waits: a wide unit's first tiles, q
  uint32_t after = 0;
  Slots next{0, 0};  // of the tile behind the one worked on
  if (!narrow) {
    const uint32_t p0 = look_up(0), p1 = look_up(1);
    after = look_up(2);
    next = slots_of(0, p0);
    begin();
    if (count > 0) {
      issue(0, next, 0);
      issue(0, next, 1);
    }
    next = slots_of(1, p1);
    if (count > 1) issue(1, next, 0);
  } else {
    begin();
  }
  bf16x8_t qf[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    u32x4_t w = *reinterpret_cast<const u32x4_t*>(a.q + q_at + 16 * i + 8 * h);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] ^= a.flip;
    qf[i] = __builtin_bit_cast(bf16x8_t, w);
  }
  // Of the item's tiles, the first `whole` are seen by all its rows (rows that are not live see none, and need
  // not) and have their pages
  const int32_t least = it.old + (int32_t)(it.unit * kRows / a.group) + 1;
  uint32_t upto = least > 0 ? (uint32_t)least / kKeys : 0u;
  if constexpr (PAGED) {
    const uint32_t last = upto < it.end ? upto : it.end;
    const uint32_t entries = (uint32_t)(((uint64_t)last * kKeys + (1u << a.kv.page_shift) - 1) >> a.kv.page_shift);
    const uint32_t* row = a.kv.table + (uint64_t)it.row * a.kv.max_pages;
    uint32_t gone = 0xFFFFFFFFu;  // the first one without a page, of the lane's
    for (uint32_t e = ((it.beg * kKeys) >> a.kv.page_shift) + lane; e < entries; e += 4 * 64) {
      uint32_t page[4];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) page[i] = row[e + 64 * i < entries ? e + 64 * i : e];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        if (page[i] >= a.kv.num_pages) gone = min(gone, e + 64 * i < entries ? e + 64 * i : e);
    }
    if (__any(gone != 0xFFFFFFFFu)) {
#pragma unroll
      for (int d = 1; d < 64; d *= 2) gone = min(gone, (uint32_t)__shfl_xor((int)gone, d));
      gone = (uint32_t)__builtin_amdgcn_readfirstlane((int)gone);
      upto = (uint32_t)(((uint64_t)gone << a.kv.page_shift) / kKeys);
    }
  }
  const uint32_t whole = upto <= it.beg ? 0u : upto < it.end ? upto - it.beg : count;

  // The query row's exponents' reference point (base 2; a whole number, with ease in it), and from where on a score (in
  // units of the products) raises it; l of the lane's half of the slots
  float m = kNegInf, limit = kNegInf, l = 0.0f;
  f32x16_t acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;

  // Operands from LDS.  K: 32 slots (half a tile) x 16 of d.  V: block d of the columns, 16 slots: two transposed
  // reads of 4 slots x 16 columns by 16 lanes each.
  const uint32_t k_lane = (c >> 4) * (kAcross * 1024) + h * 256 + (c & 15u) * 16;
  const uint32_t v_lane = (4 * h + ((lane & 15u) >> 2)) * 64 + 32 * (lane >> 4 & 1u) + 8 * (lane & 3u);
  // (a lane's place in a tile, kept from being taken apart: the steps' constants then fit the instructions)
  auto place = [&](const uint16_t* tile, uint32_t at) {
    lds_char* p = (lds_char*)tile + at;
    asm("" : "+v"(p));
    return p;
  };
  auto k_frag = [&](lds_char* k, int half, int i) {
    return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<lds_u32x4*>(k + half * (2 * kAcross * 1024) + 512 * i));
  };
  auto v_frag = [&](lds_char* v, int d, int s) {
    lds_char* p = v + (s * kAcross + d) * 1024;
    const u32x2_t x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p));
    const u32x2_t y = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 512)));
    return u32x4_t{x[0], x[1], y[0], y[1]};
  };
  auto k_tile = [&](uint32_t i) { return place(smem + i % kStages * kTile, k_lane); };
  auto v_tile = [&](uint32_t i) { return place(smem + (kStages + i % kStages) * kTile, v_lane); };

  // The reference point raised to `top` (a lane's own maximum) where any passes it by more than 8; with what is in
  // o, p of the block that is not in it yet is scaled
  bf16x8_t pr[2][2];
  float top;
  auto raise = [&](bf16x8_t* pending) {
    const float t = __builtin_ceilf(__builtin_fmaxf(top, __shfl_xor(top, 32)) * a.scale_log2) + ease;
    const float m2 = __builtin_fmaxf(m, t);
    const int down = (int)__builtin_fmaxf(m - m2, -126.0f);  // (nothing is there yet where m is -inf)
    const float f = __uint_as_float((uint32_t)(127 + down) << 23);
    m = m2;
    limit = (m2 + (8.0f - ease)) / a.scale_log2;
    l = l * f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[d][i] = acc[d][i] * f;
    if (pending) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4_t w = __builtin_bit_cast(u32x4_t, pending[x]);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(bf16lo(w[i]) * f, bf16hi(w[i]) * f);
        pending[x] = __builtin_bit_cast(bf16x8_t, w);
      }
    }
  };
  auto passes = [&]() { return __any(top > limit) != 0; };

  // A block of 32 slots from `slot` on by itself, in two halves: its scores, and the rest.  fine: p in two terms.
  // check: some rows may not see all of it.
  auto block_scores = [&](lds_char* k, int half) {
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(k, half, i), qf[i], s, 0, 0, 0);
    return s;
  };
  auto block_rest = [&](auto fine_, f32x16_t s, lds_char* v, const uint16_t* v_rows, int half, uint32_t slot, bool check) {
    constexpr bool fine = fine_.value;
    bool odd = false;
    if (check) {
      uint32_t found = 0;
#pragma unroll
      for (int i = 0; i < kTile / 16 / 64; ++i) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(v_rows + half * (kTile / 2) + 8 * (64 * i + lane));
#pragma unroll
        for (int j = 0; j < 4; ++j) found |= ((w[j] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
      }
      odd = __any(found != 0) != 0;
      uint32_t runs = 3u;  // runs of 16 slots whose page exists
      if constexpr (PAGED)
        runs = (page_of(slot) < a.kv.num_pages ? 1u : 0u) | (page_of(slot + 16) < a.kv.num_pages ? 2u : 0u);
      const int32_t left = sees - (int32_t)slot - 4 * (int32_t)h;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool seen = (8 * (i / 4) + i % 4 < left) & ((runs >> (i / 8) & 1u) != 0);
        s[i] = seen ? s[i] : kNegInf;
      }
    }
    top = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = larger(top, s[i]);
    if (passes()) raise(nullptr);
    const float base = anchor(m);
    bf16x8_t p[2], low[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      u32x4_t w, r;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * y + 2 * i], a.scale_log2, -base));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * y + 2 * i + 1], a.scale_log2, -base));
        if constexpr (fine) {
          // the upper half, and what it leaves over, which is above 0 where p is (an infinity of V meets both)
          const uint32_t b0 = __float_as_uint(e0), b1 = __float_as_uint(e1);
          w[i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
          r[i] = pack_bf16x2(__builtin_fmaxf(e0 - __uint_as_float(b0 & 0xFFFF0000u), e0 * 0x1p-20f),
                             __builtin_fmaxf(e1 - __uint_as_float(b1 & 0xFFFF0000u), e1 * 0x1p-20f));
          l = l + e0;
          l = l + e1;
        } else {
          w[i] = pack_bf16x2(e0, e1);
          l = add_pair(w[i], l);
        }
      }
      p[y] = __builtin_bit_cast(bf16x8_t, w);
      if constexpr (fine) low[y] = __builtin_bit_cast(bf16x8_t, r);
    }
    // V's values of one kind: the finite ones as they are (0), ones for inf (1), -inf (2), NaN (3)
    auto only = [&](int kind, int d, int x) {
      u32x4_t w = v_frag(v, d, 2 * half + x);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t two[2] = {w[j] & 0xFFFFu, w[j] >> 16};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t y = two[e];
          const int is = (y & 0x7F80u) != 0x7F80u ? 0 : y == 0x7F80u ? 1 : y == 0xFF80u ? 2 : 3;
          two[e] = is != kind ? 0u : kind == 0 ? y : 0x3F80u;
        }
        w[j] = two[0] | two[1] << 16;
      }
      return __builtin_bit_cast(bf16x8_t, w);
    };
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      if (!odd) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const bf16x8_t y = __builtin_bit_cast(bf16x8_t, v_frag(v, d, 2 * half + x));
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y, p[x], acc[d], 0, 0, 0);
          if constexpr (fine) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y, low[x], acc[d], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const bf16x8_t y = only(0, d, x);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y, p[x], acc[d], 0, 0, 0);
          if constexpr (fine) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y, low[x], acc[d], 0, 0, 0);
        }
#pragma unroll 1
        for (int kind = 1; kind < 4; ++kind) {
          f32x16_t r;
#pragma unroll
          for (int i = 0; i < 16; ++i) r[i] = 0.0f;
#pragma unroll
          for (int x = 0; x < 2; ++x) r = __builtin_amdgcn_mfma_f32_32x32x16_bf16(only(kind, d, x), p[x], r, 0, 0, 0);
          const float what = kind == 1 ? -kNegInf : kind == 2 ? kNegInf : __builtin_nanf("");
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] = acc[d][i] + (r[i] > 0.0f ? what : 0.0f);
        }
      }
    }
  };

  if (narrow) {
    // Wave w of a unit: blocks of 32 slots w / blocks, + unit_waves / blocks, ...; K and V of one at a time in its own
    // part of LDS, each asked for as soon as its place has been read
    constexpr int kBlock = 2 * kAcross;  // loads of a block's K, or V
    const uint32_t step = unit_waves / blocks, all = kvh == kvh_w ? 2 * count : 0u;
    uint16_t* mine = smem + wave * kTile;
    lds_char *k = place(mine, k_lane), *v = place(mine + kTile / 2, v_lane);
    auto slot_of = [&](uint32_t b) { return it.beg * kKeys + 32 * b; };
    struct Pair {
      Slots s[2];
    };
    auto pair_of = [&](uint32_t b, uint32_t p0, uint32_t p1) {
      return Pair{{slots_at(slot_of(b), p0), slots_at(slot_of(b) + 16, p1)}};
    };
    auto bring = [&](const Pair& p, int what) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        load(p.s[r], what, 0, std::integral_constant<int, kAcross>{}, mine + what * (kTile / 2) + r * kAcross * 512);
    };
    auto fence = [] { asm volatile("" ::: "memory"); };
    uint32_t b = wave % unit_waves / blocks;
    Pair pair = pair_of(b, page_of(slot_of(b)), page_of(slot_of(b) + 16));
    uint32_t p0 = page_of(slot_of(b + step)), p1 = page_of(slot_of(b + step) + 16);
    if (b < all) {
      bring(pair, 0);
      bring(pair, 1);
    }
#pragma clang loop unroll(disable)
    for (; b < all; b += step) {
      const bool more = b + step < all;
      pair = pair_of(b + step, p0, p1);
      p0 = page_of(slot_of(b + 2 * step));
      p1 = page_of(slot_of(b + 2 * step) + 16);
      fence();
      __builtin_amdgcn_s_waitcnt(0x0F70 | kBlock);  // vmcnt: all but V's loads
      fence();
      const f32x16_t s = block_scores(k, 0);
      fence();
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): K has been read
      if (more) bring(pair, 0);
      fence();
      if (more)
        __builtin_amdgcn_s_waitcnt(0x0F70 | kBlock);  // all but the next K's
      else
        __builtin_amdgcn_s_waitcnt(0x0F70);
      fence();
      // (a block inside `upto` tiles is seen by all rows)
      block_rest(std::true_type{}, s, v, mine + kTile / 2, 0, slot_of(b), slot_of(b) + 32 > upto * kKeys);
      fence();
      __builtin_amdgcn_s_waitcnt(0xC07F);
      if (more) bring(pair, 1);
    }
    l = l + __shfl_xor(l, 32);
    put();
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);
    float* sml = so + kWaves * 32 * D;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<f32x4_t*>(so + (wave * 32 + c) * D + 32 * d + 2 * i + 4 * h) =
            f32x4_t{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
    if (h == 0) {
      sml[2 * (wave * 32 + c)] = m;
      sml[2 * (wave * 32 + c) + 1] = l;
    }
    get();
    __syncthreads();
    const uint32_t units = min(kWaves / unit_waves, a.kv.kv_heads - kvh0);
    for (uint32_t id = threadIdx.x; id < units * rows * (D / 4); id += 64 * kWaves) {
      const uint32_t u = id / (D / 4) / rows, row = id / (D / 4) % rows, d = id % (D / 4) * 4;
      const uint32_t mine = u * unit_waves + row / 32, end = (u + 1) * unit_waves;
      float mm = kNegInf, ll = 0.0f;
      f32x4_t oo = {0, 0, 0, 0};
      for (uint32_t w = mine; w < end; w += blocks) mm = __builtin_fmaxf(mm, sml[2 * (w * 32 + row % 32)]);
      for (uint32_t w = mine; w < end; w += blocks) {
        const uint32_t at = w * 32 + row % 32;
        const float f = weight(sml[2 * at], mm);
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(so + at * D + d);
        ll = ll + sml[2 * at + 1] * f;
#pragma unroll
        for (int i = 0; i < 4; ++i) oo[i] = oo[i] + y[i] * f;
      }
      if (it.part != kPromptWhole) {
        const uint64_t at = ((uint64_t)it.part * a.kv.kv_heads + kvh0 + u) * a.part_rows + row;
        if (d == 0) {
          a.part_ml[2 * at] = mm;
          a.part_ml[2 * at + 1] = ll;
        }
        *reinterpret_cast<f32x4_t*>(a.part_o + at * D + d) = oo;
        continue;
      }
      const uint32_t r = it.unit * kRows + row, t = r / a.group;
      const float by = 1.0f / (it.old + (int32_t)t + 1 > 0 ? ll : 1.0f);
      uint2 w;
      w.x = pack_bf16x2(oo[0] * by, oo[1] * by);
      w.y = pack_bf16x2(oo[2] * by, oo[3] * by);
      *reinterpret_cast<uint2*>(a.o + ((uint64_t)(it.first + t) * heads + (kvh0 + u) * a.group + r % a.group) * D + d) = w;
    }
    return;
  }

  // Whole tiles: blocks of 32 slots, whose softmax runs under the products of their neighbours.  Phase j, between
  // the products of the scores of block j + 1 and of o of block j - 1: the exponentials of block j, the maximum of
  // block j + 1, and the operands from LDS, kAhead of them ahead of their products (so the first ones of the next
  // phase: K of block j + 2, V of block j).  The scores' products are one chain, so o's stand between them.
  constexpr int kAhead = 4, kV = 2 * DB;
  struct Block {
    lds_char* at;  // the lane's place in the tile
    int half;      // 32 slots of it
  };
  bf16x8_t kf[kAhead], vf[kAhead];
  f32x16_t sc[2];
  auto phase = [&](auto cur_, Block k, Block k_next, Block v, Block v_next) {
    constexpr int cur = cur_.value, nxt = 1 - cur;
    constexpr int kSteps = KS + kV, kEach = (16 + kSteps - 1) / kSteps;  // exponentials a step
    const float base = anchor(m);
    u32x4_t w[2];
    float even = 0.0f;
#pragma unroll
    for (int n = 0; n < kSteps; ++n) {
      const bool score = n * KS / kSteps != (n + 1) * KS / kSteps;
      const int f = score ? n * KS / kSteps : n - n * KS / kSteps, g = f + kAhead;
      if (score) {
        if (f == 0)
#pragma unroll
          for (int x = 0; x < 16; ++x) sc[nxt][x] = 0.0f;
        sc[nxt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[f % kAhead], qf[f], sc[nxt], 0, 0, 0);
        kf[f % kAhead] = g < KS ? k_frag(k.at, k.half, g) : k_frag(k_next.at, k_next.half, g - KS);
      } else {
        acc[f % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[f % kAhead], pr[nxt][f / DB], acc[f % DB], 0, 0, 0);
        vf[f % kAhead] = __builtin_bit_cast(bf16x8_t, g < kV ? v_frag(v.at, g % DB, 2 * v.half + g / DB)
                                                            : v_frag(v_next.at, (g - kV) % DB, 2 * v_next.half + (g - kV) / DB));
      }
#pragma unroll
      for (int i = n * kEach; i < (n + 1) * kEach && i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[cur][i], a.scale_log2, -base));
        if (i % 2 == 0) {
          even = p;
        } else {
          w[i / 8][i % 8 / 2] = pack_bf16x2(even, p);
          l = add_pair(w[i / 8][i % 8 / 2], l);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    top = sc[nxt][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = larger(top, sc[nxt][i]);
#pragma unroll
    for (int x = 0; x < 2; ++x) pr[cur][x] = __builtin_bit_cast(bf16x8_t, w[x]);
  };

  arrive();
  put();
  if (count == 0) __syncthreads();
  if (whole > 0) {
    // (there is no block -1: its p is 0, and V at its place too)
    const u32x4_t none = {0, 0, 0, 0};
    for (uint32_t i = threadIdx.x; i < kTile / 16; i += 64 * kWaves)
      *reinterpret_cast<u32x4_t*>(smem + (2 * kStages - 1) * kTile + kTile / 2 + 8 * i) = none;
    __syncthreads();
    lds_char* k0 = k_tile(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vf[i] = __builtin_bit_cast(bf16x8_t, none);
    pr[1][0] = pr[1][1] = __builtin_bit_cast(bf16x8_t, none);
#pragma unroll
    for (int x = 0; x < 16; ++x) sc[0][x] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(k0, 0, i), qf[i], sc[0], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = k_frag(k0, 1, i);
    top = sc[0][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = larger(top, sc[0][i]);
    // (K of i + 1 and V of i are there; K of i - 1 and V of i - 2 are done with)
#pragma clang loop unroll(disable)
    for (uint32_t i = 0; i < whole; ++i) {
      if (i + 1 < count) issue((i + 1) % kStages, next, 1);
      next = slots_of(i + 2, after);
      if (i + 2 < count) issue((i + 2) % kStages, next, 0);
      after = look_up(i + 3);
      if (awake) {
        const Block k1{k_tile(i), 1}, k2{k_tile(i + 1), 0}, k3{k2.at, 1};
        const Block v0{v_tile(i + kStages - 1), 1}, v1{v_tile(i), 0}, v2{v1.at, 1};
        if (passes()) raise(pr[1]);
        phase(std::integral_constant<int, 0>{}, k1, k2, v0, v1);
        if (passes()) raise(pr[0]);
        phase(std::integral_constant<int, 1>{}, k2, k3, v1, v2);
      }
      arrive();
    }
    lds_char* v = v_tile(whole - 1);
#pragma unroll
    for (int f = 0; f < kV; ++f) {
      const bf16x8_t x = f < kAhead ? vf[f % kAhead] : __builtin_bit_cast(bf16x8_t, v_frag(v, f % DB, 2 + f / DB));
      acc[f % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, pr[1][f / DB], acc[f % DB], 0, 0, 0);
    }
  }
  // (K and V of i are there, the first time K of i + 1 too; those of i - 2 are done with)
  for (uint32_t i = whole; i < count; ++i) {
    if (i + 1 < count) {
      if (i > whole) issue((i + 1) % kStages, next, 0);
      issue((i + 1) % kStages, next, 1);
    }
    next = slots_of(i + 2, after);
    after = look_up(i + 3);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t slot = (it.beg + i) * kKeys + 32 * half;
      if ((int32_t)slot < w_most)
        block_rest(std::false_type{}, block_scores(k_tile(i), half), v_tile(i), smem + (kStages + i % kStages) * kTile, half, slot, true);
    }
    arrive();
  }

  get();
  l = l + __shfl_xor(l, 32);
  if (!live) return;
  if (it.part != kPromptWhole) {
    const uint64_t at = ((uint64_t)it.part * a.kv.kv_heads + kvh * prompt_places(false)) * a.part_rows + wave * 32 + c;
    if (h == 0) {
      a.part_ml[2 * at] = m;
      a.part_ml[2 * at + 1] = l;
    }
    float* o = a.part_o + at * D + 4 * h;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<f32x4_t*>(o + 32 * d + 2 * i) = f32x4_t{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
    return;
  }
  const float by = 1.0f / (sees > 0 ? l : 1.0f);  // (l: p's sum times 2^-ease, from 2^-42 on)
  uint16_t* o = a.o + q_at + 4 * h;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      uint2 w;
      w.x = pack_bf16x2(acc[d][i] * by, acc[d][i + 1] * by);
      w.y = pack_bf16x2(acc[d][i + 2] * by, acc[d][i + 3] * by);
      *reinterpret_cast<uint2*>(o + 32 * d + 2 * i) = w;
    }
}

template <int D, bool PAGED>
CATENA_DEV void attn_prompt_run(const AttnPromptArgs& a) {
  if (!a.items) {
    const PromptItem it = item_at<PAGED>(a, blockIdx.x / a.kv.kv_heads);
    auto nothing = [] {};
    if (it.row != 0xFFFFFFFFu) attn_prompt_item<D, PAGED>(a, it, blockIdx.x % a.kv.kv_heads, kWaves, a.kv.k, a.kv.v, nothing, nothing);
    return;
  }
  // The list is two, of the rows with wide units and of the narrow ones, which some of the workgroups begin with; who
  // finds no more of one kind goes on with the other.  Work n of a kind is kv head (or heads) n % groups of its item n /
  // groups, by tickets of eight queues: workgroups of one queue run on one XCD, whose L2 then holds the K and V of
  // few heads.  (Each queue has every eighth work, so they end alike.)
  __shared__ uint32_t s_ticket;
  constexpr uint32_t kNone = 0xFFFFFFFFu;
  const uint32_t queue = blockIdx.x % kPromptQueues, place = blockIdx.x / kPromptQueues;
  const uint32_t items = scalar_word(&a.counts->items, 0), wide = scalar_word(&a.counts->wide, 0);
  const uint32_t first = kPromptCus / kPromptQueues - scalar_word(&a.counts->narrow_first, 0);  // narrow from this place on
  const uint32_t narrow_waves = scalar_word(&a.counts->narrow_waves, 0), narrow_heads = kWaves / narrow_waves;
  const uint32_t narrow_groups = (a.kv.kv_heads + narrow_heads - 1) / narrow_heads;
  uint32_t kind = place >= first, ticket = kind ? place - first : place;
  auto next = [&](uint32_t t) {  // a ticket's work; kNone: no more of the kind
    const uint32_t n = t * kPromptQueues + queue;
    return n < (kind ? (items - wide) * narrow_groups : wide * a.kv.kv_heads) ? n : kNone;
  };
  auto draw = [&] { return threadIdx.x == 0 ? atomicAdd(&a.counts->tickets[kind][queue], 1u) : 0u; };
  auto shared = [&] { return (uint32_t)__builtin_amdgcn_readfirstlane((int)s_ticket); };
  u32x4_t x, y;
  auto read = [&](uint32_t n) {
    const uint64_t at = 2 * (kind ? (uint64_t)wide + n / narrow_groups : n / a.kv.kv_heads);
    x = scalar_four(a.items, at);
    y = scalar_four(a.items, at + 1);
  };
  uint32_t n = next(ticket);
  if (n != kNone) read(n);
  for (bool other = false;;) {
    if (n == kNone) {
      if (other) return;
      other = true;
      kind ^= 1u;
      ticket = draw();
      __syncthreads();  // the last one has been read
      if (threadIdx.x == 0) s_ticket = ticket;
      __syncthreads();
      n = next(shared());
      if (n != kNone) read(n);
      continue;
    }
    // The next ticket is drawn before the item is worked on, and its item read before its last stores.
    ticket = draw();
    const PromptItem it{x[0], x[1], x[2], x[3], (int32_t)y[0], y[1], y[2], y[3]};
    const uint32_t kvh = kind ? n % narrow_groups * narrow_heads : n % a.kv.kv_heads;
    attn_prompt_item<D, PAGED>(
        a, it, kvh, kind ? narrow_waves : kWaves, a.kv.k, a.kv.v,
        [&] {
          if (threadIdx.x == 0) s_ticket = ticket;
        },
        [&] {
          n = next(shared());
          if (n != kNone) read(n);
        });
  }
}

// Number of the first n (a power of two) ascending words that are <= x, less one; s[0] <= x
CATENA_DEV uint32_t last_at_most(const uint32_t* s, uint32_t n, uint32_t x) {
  uint32_t at = 0;
  for (uint32_t step = n / 2; step > 0; step /= 2)
    if (s[at + step] <= x) at += step;
  return at;
}

// The list: one workgroup of 1024 threads.  A unit costs its tiles, a narrow one, which waits for memory beside
// the others' products, half of them; one of more than three quarters of a CU's share of all the work
// is cut into equal parts.
// Rows stand in the order of their dearest unit's cost, in 32 classes, and a row's units behind each other, the
// last (longest) first: so the short ones end the work, and the workgroups of an XCD read the same K and V at a time
// (8 ragged prompts of up to 4096 tokens: units by length alone 645 us, by rows 486).  Rows of one narrow unit stand
// behind the others, in classes of their own: they wait for memory, the others for the matrix cores, so that both are
// worked on at a time.
// Which of two rows of a class comes first, and which place a part gets, is left to the order of the threads: no
// result depends on it.
template <bool PAGED>
CATENA_DEV void attn_prompt_list(const AttnPromptArgs& a) {
  constexpr uint32_t kThreads = 1024, kClasses = 64;
  __shared__ uint32_t s_start[kThreads], s_first[kThreads], s_n[kThreads], s_old[kThreads], s_at[kThreads], s_wave[16];
  __shared__ uint32_t s_class[kClasses], s_parts, s_splits;
  __shared__ unsigned long long s_work, s_narrow;
  __shared__ uint32_t s_alone;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  if (tid < kClasses) s_class[tid] = 0;
  if (tid == 0) {
    s_work = s_narrow = 0;
    s_parts = s_splits = s_alone = 0;
  }
  struct Row {
    uint32_t units;
    Tokens t;
    int32_t old;
  };
  struct Cost {
    uint32_t tiles, cost;
    bool narrow;
  };
  auto cost_of = [&](uint32_t unit, uint32_t n, int32_t old) {
    const uint32_t tiles = tiles_of(most_of(a, unit, n, old));
    const bool narrow = n * a.group - unit * kRows <= kNarrow;
    return Cost{tiles, narrow ? tiles : 2 * tiles, narrow};
  };
  auto alone = [&](uint32_t n) { return n * a.group <= kNarrow; };  // a row of one narrow unit
  PromptCut cut = {};
  auto most_for = [&](const Cost& x) { return x.narrow ? cut.most_narrow : cut.most; };
  auto parts_of = [&](const Cost& x) { return prompt_parts(cut, x.cost, x.narrow); };
  // items of a row's units from `unit` on: of the wide units only the last ones are cut
  auto items_from = [&](uint32_t unit, uint32_t units, uint32_t n, int32_t old) {
    uint32_t items = units - unit;
    for (uint32_t u = units; u > unit; --u) {
      const uint32_t parts = parts_of(cost_of(u - 1, n, old));
      if (parts == 1 && u < units) break;
      items += parts - 1;
    }
    return items;
  };
  auto place_of = [&](const Row& r) {
    const Cost last = cost_of(r.units - 1, r.t.n, r.old);
    uint32_t cost = min(last.cost, most_for(last));
    if (r.units > 1) cost = max(cost, min(cost_of(r.units - 2, r.t.n, r.old).cost, cut.most));
    const uint32_t from = (uint32_t)((float)(cut.most - cost) * cut.share * (kClasses / 2 - 1));
    return atomicAdd(&s_class[from + (alone(r.t.n) ? kClasses / 2 : 0u)], items_from(0, r.units, r.t.n, r.old));
  };
  auto put = [&](uint32_t row, uint32_t place, uint32_t unit, const Cost& cost) {
    const uint32_t n = s_n[place];
    const int32_t old = (int32_t)s_old[place];
    const uint32_t tiles = cost.tiles, parts = parts_of(cost), each = parts > 1 ? (tiles + parts - 1) / parts : tiles;
    const uint32_t at = s_at[place] + items_from(unit + 1, units_of(a, n), n, old);
    PromptItem y{row, unit, s_first[place], n, old, 0, tiles, kPromptWhole};
    if (parts > 1) {
      y.part = atomicAdd(&s_parts, parts * prompt_places(cost.narrow));
      PromptItem z = y;
      z.beg = parts;
      const uint32_t split = atomicAdd(&s_splits, 1u);
      if (split < a.max_splits) a.splits[split] = z;
    }
    for (uint32_t p = 0; p < parts; ++p) {
      y.beg = p * each < tiles ? p * each : tiles;
      y.end = y.beg + each < tiles ? y.beg + each : tiles;
      if (at + p < a.max_items) a.items[at + p] = y;  // (always, but for rows that overlap; so above)
      if (parts > 1) y.part += prompt_places(cost.narrow);
    }
  };
  // Three times (pass: the costs' sum, the classes' sizes, the list) every row to a thread, 1024 at a time, and every
  // unit of theirs to one.  Where there are no more rows than that they are looked at once.  (A loop, since code that
  // runs once waits for its instructions.)
  Row x;
  uint32_t all = 0;
  uint64_t mine = 0, narrow = 0;
#pragma clang loop unroll(disable)
  for (uint32_t pass = 0; pass < 3; ++pass) {
    for (uint32_t r0 = 0; r0 < a.kv.rows; r0 += kThreads) {
      if (pass == 0 || a.kv.rows > kThreads) {
        const uint32_t row = r0 + tid < a.kv.rows ? r0 + tid : a.kv.rows - 1;
        x.t = tokens_of(a, row);
        x.t.n = r0 + tid < a.kv.rows ? x.t.n : 0u;
        x.old = old_of<PAGED>(a, row, x.t.n);
        x.units = units_of(a, x.t.n);
        const uint32_t in = wave_prefix(x.units);
        if (lane == 63) s_wave[wave] = in;
        __syncthreads();
        const uint32_t sums = wave_prefix(lane < 16 ? s_wave[lane] : 0u);
        const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane((int)wave);
        all = lane_of(sums, 15);
        s_start[tid] = (w ? lane_of(sums, w - 1) : 0u) + in - x.units;  // (rows without units are never the last one at most)
        s_first[tid] = x.t.first;
        s_n[tid] = x.t.n;
        s_old[tid] = (uint32_t)x.old;
      }
      if (pass > 0 && x.units > 0) s_at[tid] = place_of(x);
      if (pass == 1) {
        const uint64_t some = __ballot(x.units > 0 && alone(x.t.n));
        if (lane == 0 && some) atomicAdd(&s_alone, (uint32_t)__popcll((unsigned long long)some));
      }
      __syncthreads();
      for (uint32_t k = pass == 1 ? all : tid; k < all; k += kThreads) {
        const uint32_t at = last_at_most(s_start, kThreads, k), unit = k - s_start[at];
        const Cost cost = cost_of(unit, s_n[at], (int32_t)s_old[at]);
        if (pass == 0) {
          mine += cost.cost;
          narrow += alone(s_n[at]) ? cost.cost : 0u;
        } else {
          put(r0 + at, at, unit, cost);
        }
      }
      __syncthreads();
    }
    if (pass == 0) {
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        mine += (uint64_t)__shfl_xor((unsigned long long)mine, d);
        narrow += (uint64_t)__shfl_xor((unsigned long long)narrow, d);
      }
      if (lane == 0 && mine) atomicAdd(&s_work, (unsigned long long)mine);
      if (lane == 0 && narrow) atomicAdd(&s_narrow, (unsigned long long)narrow);
      __syncthreads();
      cut = prompt_cut(s_work * a.kv.kv_heads);
    } else if (pass == 1) {
      if (tid < 64) {
        const uint32_t n = s_class[tid], upto = wave_prefix(n);
        s_class[tid] = upto - n;
        if (tid == kClasses / 2 - 1) a.counts->wide = upto < a.max_items ? upto : a.max_items;
        if (tid == kClasses - 1) a.counts->items = upto < a.max_items ? upto : a.max_items;
      }
      __syncthreads();
    }
  }
  // Of a queue's workgroups three quarters of the narrow rows' share begin with them, so that wide units, of which
  // the parts are larger, do not end the work
  constexpr uint32_t kPlaces = kPromptCus / kPromptQueues;
  const uint32_t some = s_work ? (uint32_t)(0.75f * kPlaces * (float)s_narrow / (float)s_work) : 0u;
  const uint32_t first = s_narrow == 0 ? 0u : s_narrow == s_work ? kPlaces : some < 1 ? 1u : some;
  if (tid == 0) {
    a.counts->splits = s_splits < a.max_splits ? s_splits : a.max_splits;
    a.counts->narrow_first = first;
    const uint64_t narrow_units = (uint64_t)s_alone * a.kv.kv_heads;
    a.counts->narrow_waves = narrow_units >= 8 * kPromptCus ? 2u : (uint32_t)kWaves;
  }
  if (tid < 2 * kPromptQueues) a.counts->tickets[tid / kPromptQueues][tid % kPromptQueues] = tid / kPromptQueues ? first : kPlaces - first;
}

// The parts of cut units to o: blockIdx.x, in turn, the units, blockIdx.y the kv head, blockIdx.z in turns of 256 / (D /
// 4) query rows; a thread four columns
template <int D>
CATENA_DEV void attn_prompt_join(const AttnPromptArgs& a) {
  const uint32_t splits = a.counts->splits;
  for (uint32_t split = blockIdx.x; split < splits; split += gridDim.x) {
    const PromptItem x = a.splits[split];
    constexpr uint32_t kLanes = D / 4, kAtOnce = 256 / kLanes;
    const uint32_t kvh = blockIdx.y, heads = a.group * a.kv.kv_heads, d = threadIdx.x % kLanes * 4;
    const uint32_t places = prompt_places(x.n * a.group - x.unit * kRows <= kNarrow);
    for (uint32_t row = blockIdx.z * kAtOnce + threadIdx.x / kLanes; row < kRows; row += gridDim.z * kAtOnce) {
      const uint32_t m_row = x.unit * kRows + row, t = m_row / a.group;
      if (t >= x.n) break;
      float m = kNegInf, l = 0.0f;
      f32x4_t o = {0, 0, 0, 0};
#pragma unroll 4
      for (uint32_t p = 0; p < x.beg; ++p) {
        const uint64_t at = ((uint64_t)(x.part + p * places) * a.kv.kv_heads + kvh * places) * a.part_rows + row;
        const float pm = a.part_ml[2 * at], pl = a.part_ml[2 * at + 1];
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(a.part_o + at * D + d);
        const float m2 = __builtin_fmaxf(m, pm);
        const float f = weight(m, m2), e = weight(pm, m2);
        m = m2;
        l = l * f + pl * e;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * f + y[i] * e;
      }
      const float by = 1.0f / (x.old + (int32_t)t + 1 > 0 ? l : 1.0f);
      uint2 w;
      w.x = pack_bf16x2(o[0] * by, o[1] * by);
      w.y = pack_bf16x2(o[2] * by, o[3] * by);
      *reinterpret_cast<uint2*>(a.o + ((uint64_t)(x.first + t) * heads + kvh * a.group + m_row % a.group) * D + d) = w;
    }
  }
}

}  // namespace

// grid: without a list kv_heads * units that there may be, heads fastest; with one a workgroup a CU
#define CATENA_ATTN_PROMPT(D, NAME, PAGED)                                                                   \
  extern "C" __global__ __launch_bounds__(512, 2) void catena_attn_##NAME##_d##D(AttnPromptArgs a) {          \
    attn_prompt_run<D, PAGED>(a);                                                                            \
  }
CATENA_ATTN_PROMPT(128, prompt, true)
CATENA_ATTN_PROMPT(64, prompt, true)
CATENA_ATTN_PROMPT(128, packed, false)
CATENA_ATTN_PROMPT(64, packed, false)

extern "C" __global__ __launch_bounds__(1024) void catena_attn_prompt_list(AttnPromptArgs a) { attn_prompt_list<true>(a); }
extern "C" __global__ __launch_bounds__(1024) void catena_attn_packed_list(AttnPromptArgs a) { attn_prompt_list<false>(a); }
extern "C" __global__ __launch_bounds__(256) void catena_attn_prompt_join_d128(AttnPromptArgs a) { attn_prompt_join<128>(a); }
extern "C" __global__ __launch_bounds__(256) void catena_attn_prompt_join_d64(AttnPromptArgs a) { attn_prompt_join<64>(a); }
