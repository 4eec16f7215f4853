// How the kernels that read a cache in pages for one token a row (attn_paged.hip,
// attn_paged_q4.hip) deal out their work, and what they share of the softmax's
// arithmetic.
#pragma once

#include "common.h"
#include "paged.h"

namespace {

constexpr float kNegInf = -__builtin_huge_valf();

CATENA_DEV uint32_t lane_of(uint32_t x, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)lane); }

// A uniform word that no workgroup of this kernel writes: by a scalar load, which
// the compiler does not choose by itself behind the kernel's own stores, and
// which leaves the order of the cache's vector loads alone
CATENA_DEV uint32_t scalar_word(const uint32_t* p, uint32_t i) {
  typedef const uint32_t __attribute__((address_space(4))) * word;
  return ((word)(uintptr_t)p)[i];
}

// The work in one line: rows one after the other, a row's units (kv head and 16
// query heads) one after the other, a unit's tiles of 32 slots in order.
struct Line {
  uint32_t tiles;  // in all
  uint32_t per;    // a workgroup's
  bool whole;      // not cut: a workgroup takes whole units in turn
};
// A row on it
struct RowOnLine {
  uint32_t row, len, tiles, first;  // tiles of one unit; place of the row's first
};

CATENA_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// the reference point of exponents: 0 while no score is above -inf
CATENA_DEV float anchor(float m) { return m == kNegInf ? 0.0f : m; }
// p's power of two in the products of a row of n > 0 slots: n of p < 2^8 stay below 1/2
CATENA_DEV float ease_of(uint32_t n) { return __uint_as_float((uint32_t)(127 - 41 + __builtin_clz(n)) << 23); }

// Four columns of o / l of a row of n slots, whose o is the eased sum; 0 where there are
// none
template <bool F32>
CATENA_DEV void store_o(const AttnPagedArgs& a, uint64_t at, f32x4_t o, float l, uint32_t n) {
  l = n ? l * ease_of(n) : 1.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = o[i] / l;
  if constexpr (F32) {
    *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.o) + at) = o;
  } else {
    uint2 w;
    w.x = pack_bf16x2(o[0], o[1]);
    w.y = pack_bf16x2(o[2], o[3]);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = w;
  }
}

// Lane r's row among the first 64, kept for the look-ups that follow
struct FirstRows {
  uint32_t len, upto;  // its slots, and the tiles of the rows up to it
};
CATENA_DEV uint32_t len_of(const AttnPagedArgs& a, uint32_t row) {
  return row < a.kv.rows ? paged_len(a.kv, a.lens[row]) : 0u;
}
CATENA_DEV FirstRows first_rows(const AttnPagedArgs& a) {
  const uint32_t len = len_of(a, threadIdx.x & 63u);
  return FirstRows{len, wave_prefix((len + 31) / 32)};
}
CATENA_DEV Line line_of(const AttnPagedArgs& a, const FirstRows& f) {
  uint32_t all = lane_of(f.upto, 63);
  bool whole = f.len <= a.short_slots;
  if (a.kv.rows > 64) {
    uint32_t n = 0;
#pragma unroll 4
    for (uint32_t r = 64 + (threadIdx.x & 63u); r < a.kv.rows; r += 64) {
      const uint32_t len = len_of(a, r);
      n += (len + 31) / 32;
      whole = whole && len <= a.short_slots;
    }
    all += lane_of(wave_prefix(n), 63);
  }
  all *= a.kv.kv_heads * a.head_tiles;
  // long parts: one workgroup a CU (D = 128, 32768 tiles: 83.1 us against 85.3 with
  // two; D = 64, whose tiles are half as long, ragged rows: 59.6 against 57.3)
  const uint32_t blocks = all >= 16384 && a.blocks > 256 && a.kv.head_dim == 128 ? 256 : a.blocks;
  return Line{all, (all + blocks - 1) / blocks, __all(whole) != 0};
}
// The row that place `at` of the line (below its end) belongs to
CATENA_DEV RowOnLine row_at_place(const AttnPagedArgs& a, const FirstRows& f, uint32_t at) {
  const uint32_t lane = threadIdx.x & 63u, units = a.kv.kv_heads * a.head_tiles;
  uint32_t len = f.len, upto = f.upto, r0 = 0;
  uint64_t past = __ballot(upto * units > at);
  while (!past && r0 + 64 < a.kv.rows) {
    r0 += 64;
    len = len_of(a, r0 + lane);
    upto = lane_of(upto, 63) + wave_prefix((len + 31) / 32);
    past = __ballot(upto * units > at);
  }
  const uint32_t j = (uint32_t)__ffsll((unsigned long long)past) - 1, n = lane_of(len, j), tiles = (n + 31) / 32;
  return RowOnLine{r0 + j, n, tiles, (lane_of(upto, j) - tiles) * units};
}
CATENA_DEV RowOnLine row_on_line(const AttnPagedArgs& a, const FirstRows& f, uint32_t row) {
  const uint32_t len = row < 64 ? lane_of(f.len, row) : paged_len(a.kv, scalar_word(a.lens, row));
  const uint32_t tiles = (len + 31) / 32;
  uint32_t before = lane_of(f.upto, row < 64 ? row : 63);
  if (row >= 64) {
    uint32_t n = 0;
    for (uint32_t r = 64 + (threadIdx.x & 63u); r <= row; r += 64) n += (len_of(a, r) + 31) / 32;
    before += lane_of(wave_prefix(n), 63);
  }
  return RowOnLine{row, len, tiles, (before - tiles) * a.kv.kv_heads * a.head_tiles};
}

// A workgroup's part of a unit: tiles [beg, end) of query heads 16 ht .. + gn - 1 of
// a (row, kv head)
struct Part {
  uint32_t row, len, tiles, kvh, ht, gn, beg, end;
};
CATENA_DEV Part part_from(const AttnPagedArgs& a, uint32_t row, uint32_t len, uint32_t unit, uint32_t beg,
                          uint32_t most) {
  Part p;
  p.row = row;
  p.len = len;
  p.tiles = (len + 31) / 32;
  p.kvh = a.head_tiles == 1 ? unit : unit / a.head_tiles;
  p.ht = unit - p.kvh * a.head_tiles;
  p.gn = a.group - 16 * p.ht < 16 ? a.group - 16 * p.ht : 16;
  p.beg = beg;
  p.end = p.tiles - beg < most ? p.tiles : beg + most;
  return p;
}
// The part behind p, of at most `most` tiles; there is one
CATENA_DEV Part part_behind(const AttnPagedArgs& a, const Part& p, uint32_t most) {
  const uint32_t unit = p.kvh * a.head_tiles + p.ht + 1;
  if (unit < a.kv.kv_heads * a.head_tiles) return part_from(a, p.row, p.len, unit, 0, most);
  uint32_t row = p.row, len = 0;
  while (len == 0 && ++row < a.kv.rows) len = paged_len(a.kv, scalar_word(a.lens, row));
  return part_from(a, row, len, 0, 0, most);
}

}  // namespace
