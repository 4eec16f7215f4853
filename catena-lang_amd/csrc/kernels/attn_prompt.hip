// Causal attention of packed sequences of different lengths, grouped heads, over a
// key-value cache in pages or over packed keys and values.
//
//   token t of row r's n new ones sees the row's first lens[r] - n + t + 1 slots:
//   s_j = scale * q . k_j,  o = sum_j exp(s_j - max) v_j / sum_j exp(s_j - max)
//
// Bound: the matrix cores: 4 D flop for each (query head, slot seen), against 4 D
// bytes a slot and kv head that 128 query rows share.
//
// A workgroup takes 128 query rows of one row and kv head: query row m is token m /
// group, head m % group of the kv head's, so that short sequences with grouped heads
// fill the rows too, and all rows share K and V.  A wave has 32 of them.
// K and V come 64 slots at a time straight to LDS (two buffers: the next tile arrives
// while one is worked on), in rows of D whose 16-byte chunks are swizzled, K so that
// 16 rows' equal chunks and V so that 4 rows' neighbouring chunks lie in all banks.
//   S^T = K Q^T (32 x 32 x 16 products): lane (c, h) = (lane & 31, lane >> 5) holds
//     query row c's scores of slots 32 b + 8 (i / 4) + 4 h + i % 4 (register i of
//     block b), so the softmax's maximum and sum of a query row need one exchange, and
//     P stays where it is as the second product's operand: the order of slots in the
//     sum is free, and V's operand takes the same.
//   O^T = V^T P^T: V's columns by transposed reads of 4 slots x 16 columns.
//
// The maximum is raised only where a score passes it by more than 8 in base 2.
// Range: p enters the products times 2^-40 (and so does the sum, so that it leaves
// again in the division): sums of finite values never overflow.
// p is rounded to bf16, as the products take it; scores, sums and o are f32.
// What a query row does not see has p = 0; an infinity or NaN in V there would still
// reach it through the product, so tiles that are not seen whole are searched for
// them, and where there are any they are taken out of the product and entered by
// products of their own that say which sums they reach.
#include <type_traits>

#include "common.h"
#include "paged.h"

namespace {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kEase = 40.0f;
constexpr int kKeys = 64;  // slots of a tile
constexpr int kStages = 3;  // tiles of K, and of V, in LDS
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) u32x4_t lds_u32x4;
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4;

CATENA_DEV uint32_t lane_of(uint32_t x, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)lane); }
CATENA_DEV float anchor(float m) { return m == kNegInf ? 0.0f : m; }

// A uniform word that this kernel does not write, by a scalar load
CATENA_DEV uint32_t scalar_word(const uint32_t* p, uint64_t i) {
  typedef const uint32_t __attribute__((address_space(4))) * word;
  return ((word)(uintptr_t)p)[i];
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
  if (row >= a.kv.rows) return Tokens{0, 0};
  const uint32_t beg = a.starts[row], upto = a.starts[row + 1], end = upto < a.tokens ? upto : a.tokens;
  return Tokens{beg, beg < end ? end - beg : 0u};
}

// The workgroup's query rows: `rows` a tile, tiles of all rows in one line, the last
// (longest) tile of a row first
struct Unit {
  uint32_t row, tile, first, n;
  bool any;
};
CATENA_DEV Unit unit_of(const AttnPromptArgs& a, uint32_t index, uint32_t rows) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t before = 0;
  for (uint32_t r0 = 0; r0 < a.kv.rows; r0 += 64) {
    const Tokens t = tokens_of(a, r0 + lane);
    const uint32_t tiles = (uint32_t)(((uint64_t)t.n * a.group + rows - 1) / rows);
    const uint32_t upto = before + wave_prefix(tiles);
    const uint64_t past = __ballot(upto > index);
    if (past) {
      const uint32_t j = (uint32_t)__ffsll((unsigned long long)past) - 1;
      return Unit{r0 + j, lane_of(upto, j) - 1 - index, lane_of(t.first, j), lane_of(t.n, j), true};
    }
    before = lane_of(upto, 63);
  }
  return Unit{0, 0, 0, 0, false};
}

template <int D, int QB, int WAVES, bool PAGED>
CATENA_DEV void attn_prompt_run(const AttnPromptArgs& a, const uint16_t* __restrict__ pool_k, const uint16_t* __restrict__ pool_v) {
  constexpr int KS = D / 16;   // steps of a score's sum
  constexpr int DB = D / 32;   // blocks of o's columns
  constexpr int kRows = 32 * QB * WAVES;  // query rows of a workgroup
  constexpr int kTile = kKeys * D;  // elements of K or V of a tile
  // A tile in LDS: blocks of 16 slots x 32 columns (1 KiB, what one load brings), a run of slots' blocks behind
  // each other.  In a block, K column by column of 16 bytes, V slot by slot: so the reads of a product's operand,
  // 16 slots' 16 bytes of K or 4 slots' 64 bytes of V, lie in all banks, and the operands of all steps a constant apart.
  constexpr int kAcross = D / 32;  // blocks of a run
  constexpr int kLoads = 4 * kAcross / WAVES;  // a wave's blocks, of one run
  constexpr int kWavesARun = WAVES / 4;
  extern __shared__ __attribute__((aligned(1024))) uint16_t smem[];  // K x kStages, V x kStages
  const uint32_t lane = threadIdx.x & 63u, c = lane & 31u, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t kvh = blockIdx.x % a.kv.kv_heads, heads = a.group * a.kv.kv_heads;
  const Unit unit = unit_of(a, blockIdx.x / a.kv.kv_heads, kRows);
  if (!unit.any) return;
  // slots in use, and how many of them lie before the new tokens
  uint32_t len = unit.n;
  if (a.lens) len = scalar_word(a.lens, unit.row);
  if (PAGED) len = paged_len(a.kv, len);
  const int32_t old = (int32_t)len - (int32_t)unit.n;  // below 0: the first tokens see nothing

  // the lane's query rows: one in each of the wave's blocks of 32
  const uint32_t w_row = unit.tile * kRows + wave * 32 * QB;
  bool live[QB];
  uint64_t q_at[QB];
  int32_t sees[QB];  // slots
  bf16x8_t qf[QB][KS];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    const uint32_t m_row = w_row + 32 * b + c, t = m_row / a.group, head = kvh * a.group + m_row % a.group;
    live[b] = t < unit.n;
    q_at[b] = ((uint64_t)(unit.first + (live[b] ? t : 0u)) * heads + (live[b] ? head : kvh * a.group)) * D;
    sees[b] = live[b] ? old + (int32_t)t + 1 : 0;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      u32x4_t w = *reinterpret_cast<const u32x4_t*>(a.q + q_at[b] + 16 * i + 8 * h);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] ^= a.flip;
      qf[b][i] = __builtin_bit_cast(bf16x8_t, w);
    }
  }
  // tiles: as far as the workgroup's last token sees; `whole` of them are seen by all its rows (rows that are
  // not live see none, and need not) and have their pages
  const uint32_t last_t = (unit.tile * kRows + kRows - 1) / a.group, t_end = last_t < unit.n ? last_t + 1 : unit.n;
  const int32_t most = old + (int32_t)t_end, least = old + (int32_t)(unit.tile * kRows / a.group) + 1;
  const uint32_t tiles = most > 0 ? ((uint32_t)most + kKeys - 1) / kKeys : 0u;
  uint32_t whole = least > 0 ? (uint32_t)least / kKeys : 0u;
  if constexpr (PAGED) {
    const uint32_t entries = (uint32_t)(((uint64_t)whole * kKeys + (1u << a.kv.page_shift) - 1) >> a.kv.page_shift);
    const uint32_t* row = a.kv.table + (uint64_t)unit.row * a.kv.max_pages;
    for (uint32_t e = 0; e < entries; e += 64) {
      const uint64_t gone = __ballot(e + lane < entries && row[e + lane] >= a.kv.num_pages);
      if (gone) {
        const uint32_t first = e + (uint32_t)__ffsll((unsigned long long)gone) - 1;
        whole = (first << a.kv.page_shift) / kKeys;
        break;
      }
    }
  }
  // slots that any of the wave's rows sees
  const uint32_t w_last = (w_row + 32 * QB - 1) / a.group, w_end = w_last < unit.n ? w_last + 1 : unit.n;
  const int32_t w_most = w_row / a.group < unit.n ? old + (int32_t)w_end : 0;

  // Loads: run wave / kWavesARun of a tile, which lies inside one page
  const uint32_t row_bytes = PAGED ? D * 2 : (uint32_t)(a.stride * 2);
  const uint32_t run = wave / kWavesARun, first_block = wave % kWavesARun * kLoads;
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    k_off[i] = (lane & 15u) * row_bytes + 64 * (first_block + i) + 16 * (lane >> 4);
    v_off[i] = (lane >> 2) * row_bytes + 64 * (first_block + i) + 16 * (lane & 3u);
  }
  auto page_of = [&](uint32_t slot) -> uint32_t {
    if constexpr (PAGED) return slot < len ? scalar_word(a.kv.table, (uint64_t)unit.row * a.kv.max_pages + (slot >> a.kv.page_shift)) : 0xFFFFFFFFu;
    return 0;
  };
  // The wave's rows of a tile: where they are and how many.  Their page is looked up a tile before they are asked
  // for, so that nothing waits for it.
  struct Rows {
    uint64_t at;
    uint32_t n;
  };
  auto rows_of = [&](uint32_t tile, uint32_t page) {
    const uint32_t slot = tile * kKeys + 16 * run;
    Rows r{0, slot < len ? (len - slot < 16 ? len - slot : 16u) : 0u};
    if constexpr (PAGED) {
      if (page < a.kv.num_pages)
        r.at = paged_offset(a.kv, page, kvh, slot & ((1u << a.kv.page_shift) - 1u));
      else
        r.n = 0;
    } else {
      r.at = ((uint64_t)unit.first + (r.n ? slot : 0u)) * a.stride + kvh * D;
    }
    return r;
  };
  auto look_up = [&](uint32_t tile) { return page_of(tile * kKeys + 16 * run); };
  // K (what 0) or V (1) of them to their place in the ring
  auto issue = [&](uint32_t stage, const Rows& r, int what) {
    const int bytes = r.n ? (int)((r.n - 1) * row_bytes + D * 2) : 0;
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)((what ? pool_v : pool_k) + r.at), (short)0, bytes, 0x00020000);
    uint16_t* dst = smem + ((what ? kStages : 0) + stage) * kTile + (run * kAcross + first_block) * 512;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(dst + 512 * i), 16,
                                               (int)(what ? v_off[i] : k_off[i]), 0, 0, 0);
  };
  // All that this wave has asked for is in LDS, what it has read of LDS has arrived, and so for the others
  auto arrive = [&]() {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  // of a query row: the exponents' reference point, a whole number (base 2), and from where on a score (in units
  // of the products) raises it; l of the lane's half of the slots
  float m[QB], limit[QB], l[QB];
  f32x16_t acc[QB][DB];
#pragma unroll
  for (int b = 0; b < QB; ++b) {
    m[b] = limit[b] = kNegInf;
    l[b] = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[b][d][i] = 0.0f;
  }

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
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p));
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 512)));
    return u32x4_t{x[0], x[1], y[0], y[1]};
  };
  // The reference points raised to `top` (a lane's own maximum) where any passes them by more than 8: by whole
  // numbers, so that what is there already is scaled exactly, p of the block that is not in o yet among it
  bf16x8_t pr[2][QB][2];
  float top[QB];
  auto raise = [&](bf16x8_t (*pending)[2]) {
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      const float t = __builtin_ceilf(__builtin_fmaxf(top[b], __shfl_xor(top[b], 32)) * a.scale_log2);
      const float m2 = __builtin_fmaxf(m[b], t);
      const int down = (int)__builtin_fmaxf(m[b] - m2, -126.0f);  // (nothing is there yet where m is -inf)
      const float f = __uint_as_float((uint32_t)(127 + down) << 23);
      m[b] = m2;
      limit[b] = (m2 + 8.0f) / a.scale_log2;
      l[b] = l[b] * f;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][d][i] = acc[b][d][i] * f;
      if (pending) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          u32x4_t w = __builtin_bit_cast(u32x4_t, pending[b][x]);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(bf16lo(w[i]) * f, bf16hi(w[i]) * f);
          pending[b][x] = __builtin_bit_cast(bf16x8_t, w);
        }
      }
    }
  };
  auto passes = [&]() {
    bool any = false;
#pragma unroll
    for (int b = 0; b < QB; ++b) any = any | (top[b] > limit[b]);
    return __any(any) != 0;
  };
  auto larger = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };

  // A tile that not all rows see, block by block of query rows
  auto take_masked = [&](uint32_t tile) {
    const uint16_t* v_rows = smem + (kStages + tile % kStages) * kTile;
    lds_char* k = place(smem + tile % kStages * kTile, k_lane);
    lds_char* v = place(v_rows, v_lane);
    uint32_t found = 0;
#pragma unroll 4
    for (uint32_t i = lane; i < kTile / 8; i += 64) {
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(v_rows + 8 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) found |= ((w[j] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
    }
    const bool odd = __any(found != 0) != 0;
    uint32_t runs = 0xFu;  // runs of 16 slots whose page exists
    if constexpr (PAGED) {
      runs = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) runs |= (page_of(tile * kKeys + 16 * r) < a.kv.num_pages ? 1u : 0u) << r;
    }
    f32x16_t s[QB][2];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      top[b] = kNegInf;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[b][y][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < KS; ++i)
          s[b][y] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(k, y, i), qf[b][i], s[b][y], 0, 0, 0);
        const int32_t left = sees[b] - (int32_t)(tile * kKeys) - 4 * (int32_t)h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool seen = (32 * y + 8 * (i / 4) + i % 4 < left) & ((runs >> (2 * y + i / 8) & 1u) != 0);
          s[b][y][i] = seen ? s[b][y][i] : kNegInf;
          top[b] = larger(top[b], s[b][y][i]);
        }
      }
    }
    if (passes()) raise(nullptr);
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      const float base = anchor(m[b]) + kEase;
      bf16x8_t p[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[b][y / 2][8 * (y % 2) + 2 * i], a.scale_log2, -base)),
                             __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][y / 2][8 * (y % 2) + 2 * i + 1], a.scale_log2, -base)));
          l[b] = add_pair(w[i], l[b]);
        }
        p[y] = __builtin_bit_cast(bf16x8_t, w);
      }
      // V's values of one kind: the finite ones as they are (0), ones for inf (1), -inf (2), NaN (3)
      auto only = [&](int kind, int d, int x) {
        u32x4_t w = v_frag(v, d, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t half[2] = {w[j] & 0xFFFFu, w[j] >> 16};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t y = half[e];
            const int is = (y & 0x7F80u) != 0x7F80u ? 0 : y == 0x7F80u ? 1 : y == 0xFF80u ? 2 : 3;
            half[e] = is != kind ? 0u : kind == 0 ? y : 0x3F80u;
          }
          w[j] = half[0] | half[1] << 16;
        }
        return __builtin_bit_cast(bf16x8_t, w);
      };
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        if (!odd) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            acc[b][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v_frag(v, d, x)), p[x], acc[b][d], 0, 0, 0);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            acc[b][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(only(0, d, x), p[x], acc[b][d], 0, 0, 0);
#pragma unroll 1
          for (int kind = 1; kind < 4; ++kind) {
            f32x16_t r;
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = 0.0f;
#pragma unroll
            for (int x = 0; x < 4; ++x) r = __builtin_amdgcn_mfma_f32_32x32x16_bf16(only(kind, d, x), p[x], r, 0, 0, 0);
            const float what = kind == 1 ? -kNegInf : kind == 2 ? kNegInf : __builtin_nanf("");
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[b][d][i] = acc[b][d][i] + (r[i] > 0.0f ? what : 0.0f);
          }
        }
      }
    }
  };

  // Whole tiles: blocks of 32 slots, whose softmax runs under the products of their neighbours.  Phase j, between
  // the products of the scores of block j + 1 and of o of block j - 1: the exponentials of block j, the maximum of
  // block j + 1, and the operands from LDS, kAhead of them ahead of their products (so the first ones of the next
  // phase: K of block j + 2, V of block j).
  constexpr int kAhead = 4, kV = 2 * DB;
  struct Block {
    lds_char* at;  // the lane's place in the tile
    int half;      // 32 slots of it
  };
  bf16x8_t kf[kAhead], vf[kAhead];
  f32x16_t sc[2][QB];
  auto phase = [&](auto cur_, Block k, Block k_next, Block v, Block v_next) {
    constexpr int cur = cur_.value, nxt = 1 - cur;
    constexpr int kScores = KS * QB, kO = kV * QB, kSteps = kScores + kO;
    constexpr int kEach = (16 * QB + kSteps - 1) / kSteps;  // exponentials a step
    float base[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) base[b] = anchor(m[b]) + kEase;
    u32x4_t w[QB][2];
    float even = 0.0f;
    // two chains of scores take as long as their products; a single one alternates with o's products
    constexpr bool kFirst = QB > 1;
#pragma unroll
    for (int n = 0; n < kSteps; ++n) {
      const bool score = kFirst ? n < kScores : (n * kScores / kSteps != (n + 1) * kScores / kSteps);
      const int y = kFirst ? (score ? n : n - kScores) : (score ? n * kScores / kSteps : n - n * kScores / kSteps);
      const int f = y / QB, b = y % QB;
      if (score) {
        if (f == 0)
#pragma unroll
          for (int x = 0; x < 16; ++x) sc[nxt][b][x] = 0.0f;
        sc[nxt][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[f % kAhead], qf[b][f], sc[nxt][b], 0, 0, 0);
        if (b == QB - 1) {
          const int g = f + kAhead;
          kf[f % kAhead] = g < KS ? k_frag(k.at, k.half, g) : k_frag(k_next.at, k_next.half, g - KS);
        }
      } else {
        acc[b][f % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[f % kAhead], pr[nxt][b][f / DB], acc[b][f % DB], 0, 0, 0);
        if (b == QB - 1) {
          const int g = f + kAhead;
          vf[f % kAhead] = __builtin_bit_cast(bf16x8_t, g < kV ? v_frag(v.at, g % DB, 2 * v.half + g / DB)
                                                              : v_frag(v_next.at, (g - kV) % DB, 2 * v_next.half + (g - kV) / DB));
        }
      }
#pragma unroll
      for (int x = n * kEach; x < (n + 1) * kEach && x < 16 * QB; ++x) {
        const int e = x / 16, i = x % 16;
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[cur][e][i], a.scale_log2, -base[e]));
        if (i % 2 == 0) {
          even = p;
        } else {
          w[e][i / 8][i % 8 / 2] = pack_bf16x2(even, p);
          l[e] = add_pair(w[e][i / 8][i % 8 / 2], l[e]);
        }
      }
      if (kFirst && n >= kScores + 2) {
        constexpr int kLeft = kO - 2;
#pragma unroll
        for (int x = (n - kScores - 2) * 8 * QB / kLeft; x < (n - kScores - 1) * 8 * QB / kLeft; ++x) {
          const int e = x / 8, i = x % 8;
          const float z = larger(sc[nxt][e][2 * i], sc[nxt][e][2 * i + 1]);
          top[e] = i == 0 ? z : larger(top[e], z);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      if (!kFirst) {
        top[b] = sc[nxt][b][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top[b] = larger(top[b], sc[nxt][b][i]);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) pr[cur][b][x] = __builtin_bit_cast(bf16x8_t, w[b][x]);
    }
  };

  auto k_tile = [&](uint32_t t) { return place(smem + t % kStages * kTile, k_lane); };
  auto v_tile = [&](uint32_t t) { return place(smem + (kStages + t % kStages) * kTile, v_lane); };
  const Rows now = rows_of(0, look_up(0));
  Rows next = rows_of(1, look_up(1));  // of the tile behind the one worked on
  uint32_t after = look_up(2);
  issue(0, now, 0);
  issue(0, now, 1);
  issue(1, next, 0);
  arrive();
  if (whole > 0) {
    // (there is no block -1: its p is 0, and V at its place too)
    const u32x4_t none = {0, 0, 0, 0};
    for (uint32_t i = threadIdx.x; i < kTile / 16; i += 64 * WAVES)
      *reinterpret_cast<u32x4_t*>(smem + (2 * kStages - 1) * kTile + kTile / 2 + 8 * i) = none;
    __syncthreads();
    lds_char* k0 = k_tile(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) vf[i] = __builtin_bit_cast(bf16x8_t, none);
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      pr[1][b][0] = pr[1][b][1] = __builtin_bit_cast(bf16x8_t, none);
#pragma unroll
      for (int x = 0; x < 16; ++x) sc[0][b][x] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const bf16x8_t f = k_frag(k0, 0, i);
#pragma unroll
      for (int b = 0; b < QB; ++b) sc[0][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, qf[b][i], sc[0][b], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = k_frag(k0, 1, i);
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      top[b] = sc[0][b][0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top[b] = larger(top[b], sc[0][b][i]);
    }
    // (K of t + 1 and V of t are there; K of t - 1 and V of t - 2 are done with)
#pragma clang loop unroll(disable)
    for (uint32_t t = 0; t < whole; ++t) {
      issue((t + 1) % kStages, next, 1);
      next = rows_of(t + 2, after);
      issue((t + 2) % kStages, next, 0);
      after = look_up(t + 3);
      const Block k1{k_tile(t), 1}, k2{k_tile(t + 1), 0}, k3{k2.at, 1};
      const Block v0{v_tile(t + kStages - 1), 1}, v1{v_tile(t), 0}, v2{v1.at, 1};
      if (passes()) raise(pr[1]);
      phase(std::integral_constant<int, 0>{}, k1, k2, v0, v1);
      if (passes()) raise(pr[0]);
      phase(std::integral_constant<int, 1>{}, k2, k3, v1, v2);
      arrive();
    }
    lds_char* v = v_tile(whole - 1);
#pragma unroll
    for (int f = 0; f < kV; ++f)
#pragma unroll
      for (int b = 0; b < QB; ++b) {
        const bf16x8_t x = f < kAhead ? vf[f % kAhead] : __builtin_bit_cast(bf16x8_t, v_frag(v, f % DB, 2 + f / DB));
        acc[b][f % DB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, pr[1][b][f / DB], acc[b][f % DB], 0, 0, 0);
      }
  }
  // (K and V of t are there, the first time K of t + 1 too; those of t - 2 are done with)
  for (uint32_t t = whole; t < tiles; ++t) {
    if (t > whole) issue((t + 1) % kStages, next, 0);
    issue((t + 1) % kStages, next, 1);
    next = rows_of(t + 2, after);
    after = look_up(t + 3);
    if ((int32_t)(t * kKeys) < w_most) take_masked(t);
    arrive();
  }

#pragma unroll
  for (int b = 0; b < QB; ++b) {
    l[b] = l[b] + __shfl_xor(l[b], 32);
    if (!live[b]) continue;
    const float by = sees[b] > 0 ? l[b] : 1.0f;
    uint16_t* o = a.o + q_at[b];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        uint2 w;
        w.x = pack_bf16x2(acc[b][d][i] / by, acc[b][d][i + 1] / by);
        w.y = pack_bf16x2(acc[b][d][i + 2] / by, acc[b][d][i + 3] / by);
        *reinterpret_cast<uint2*>(o + 32 * d + 8 * (i / 4) + 4 * h) = w;
      }
  }
}

}  // namespace

// grid = kv_heads * tiles of 128 or 256 query rows that there may be, heads fastest
#define CATENA_ATTN_PROMPT(D, NAME, PAGED)                                                                   \
  extern "C" __global__ __launch_bounds__(256, 2) void catena_attn_##NAME##_d##D##_w4(AttnPromptArgs a) {    \
    attn_prompt_run<D, 1, 4, PAGED>(a, a.kv.k, a.kv.v);                                                      \
  }                                                                                                          \
  extern "C" __global__ __launch_bounds__(512, 2) void catena_attn_##NAME##_d##D##_w8(AttnPromptArgs a) {    \
    attn_prompt_run<D, 1, 8, PAGED>(a, a.kv.k, a.kv.v);                                                      \
  }
CATENA_ATTN_PROMPT(128, prompt, true)
CATENA_ATTN_PROMPT(64, prompt, true)
CATENA_ATTN_PROMPT(128, packed, false)
CATENA_ATTN_PROMPT(64, packed, false)
