// How the kernels that read a cache in pages for one token a row (attn_paged.hip,
// attn_paged_q4.hip) deal out their work, join what they cut, and what they share of the
// softmax's arithmetic.
//
// The file that includes this says before that how many slots a tile has, kTileSlots, and
// how many tiles in all go to one workgroup a CU, kOneACu, below how many to two at most,
// kTwoACu, and what units are not cut:
// while no row has more than args.short_slots slots (kWholeShare 0), or while no row has
// more than kWholeMost tiles and kWholeShare times the longest row's are no more than all
// and twice kWholeShare.
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

CATENA_DEV uint32_t tiles_of(uint32_t len) { return (len + (kTileSlots - 1)) / kTileSlots; }

// The work in one line: rows one after the other, a row's units (kv head and 16
// query heads) one after the other, a unit's tiles in order.
struct Line {
  uint32_t tiles;   // in all
  uint32_t per;     // a workgroup's
  uint32_t blocks;  // workgroups that share them out
  bool whole;       // not cut: a workgroup takes whole units in turn
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
  return FirstRows{len, wave_prefix(tiles_of(len))};
}
CATENA_DEV Line line_of(const AttnPagedArgs& a, const FirstRows& f) {
  uint32_t all = lane_of(f.upto, 63), most = f.len;
  bool whole = f.len <= a.short_slots;
  if (a.kv.rows > 64) {
    uint32_t n = 0;
#pragma unroll 4
    for (uint32_t r = 64 + (threadIdx.x & 63u); r < a.kv.rows; r += 64) {
      const uint32_t len = len_of(a, r);
      n += tiles_of(len);
      whole = whole && len <= a.short_slots;
      most = len > most ? len : most;
    }
    all += lane_of(wave_prefix(n), 63);
  }
  all *= a.kv.kv_heads * a.head_tiles;
  if constexpr (kWholeShare > 0) {
    most = tiles_of(most);
    whole = most <= kWholeMost && kWholeShare * most <= all + 2 * kWholeShare;  // (for the lane's rows; below for all)
  }
  uint32_t blocks = all >= kOneACu && a.blocks > 256 && a.kv.head_dim == 128 ? 256 : a.blocks;
  if constexpr (kTwoACu > 0) blocks = all < kTwoACu && blocks > 512 ? 512 : blocks;
  return Line{all, (all + blocks - 1) / blocks, blocks, __all(whole) != 0};
}
// The row that place `at` of the line (below its end) belongs to
CATENA_DEV RowOnLine row_at_place(const AttnPagedArgs& a, const FirstRows& f, uint32_t at) {
  const uint32_t lane = threadIdx.x & 63u, units = a.kv.kv_heads * a.head_tiles;
  uint32_t len = f.len, upto = f.upto, r0 = 0;
  uint64_t past = __ballot(upto * units > at);
  while (!past && r0 + 64 < a.kv.rows) {
    r0 += 64;
    len = len_of(a, r0 + lane);
    upto = lane_of(upto, 63) + wave_prefix(tiles_of(len));
    past = __ballot(upto * units > at);
  }
  const uint32_t j = (uint32_t)__ffsll((unsigned long long)past) - 1, n = lane_of(len, j), tiles = tiles_of(n);
  return RowOnLine{r0 + j, n, tiles, (lane_of(upto, j) - tiles) * units};
}
CATENA_DEV RowOnLine row_on_line(const AttnPagedArgs& a, const FirstRows& f, uint32_t row) {
  const uint32_t len = row < 64 ? lane_of(f.len, row) : paged_len(a.kv, scalar_word(a.lens, row));
  const uint32_t tiles = tiles_of(len);
  uint32_t before = lane_of(f.upto, row < 64 ? row : 63);
  if (row >= 64) {
    uint32_t n = 0;
    for (uint32_t r = 64 + (threadIdx.x & 63u); r <= row; r += 64) n += tiles_of(len_of(a, r));
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
  p.tiles = tiles_of(len);
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

// Where the parts of a unit are: the workgroups that have one are numbered on
struct Parts {
  uint32_t first, n;  // n < 2: one workgroup had the unit
};
CATENA_DEV Parts parts_of(const Line& line, const RowOnLine& r, uint32_t unit) {
  if (r.tiles == 0) return Parts{0, 0};
  const uint32_t beg = r.first + unit * r.tiles, first = beg / line.per;
  return Parts{first, (beg + r.tiles - 1) / line.per - first + 1};
}

// Place of a unit's part i for head h of its 16: the unit's first part lies in the
// second of its workgroup's places
CATENA_DEV uint64_t part_place(const AttnPagedArgs& a, const Parts& p, uint32_t i, uint32_t h) {
  return ((uint64_t)(p.first + i) * 2 + (i == 0)) * (a.group < 16 ? a.group : 16) + h;
}

// One thread's parts i = first, first + step, ... of a unit's head, with a running
// maximum: four columns of o from `col` on
struct Joined {
  f32x4_t o;
  float m, l;
};
template <int D>
CATENA_DEV Joined join_parts(const AttnPagedArgs& a, const Parts& p, uint32_t h, uint32_t col, uint32_t first,
                             uint32_t step) {
  Joined j{f32x4_t{0, 0, 0, 0}, kNegInf, 0.0f};
#pragma unroll 4
  for (uint32_t i = first; i < p.n; i += step) {
    const uint64_t at = part_place(a, p, i, h);
    const float pm = a.part_ml[2 * at], pl = a.part_ml[2 * at + 1];
    const f32x4_t y = *reinterpret_cast<const f32x4_t*>(a.part_o + at * D + col);
    const float m = __builtin_fmaxf(j.m, pm), f = exp2_fast(j.m - anchor(m)), e = exp2_fast(pm - anchor(m));
    j.m = m;
    j.l = j.l * f + pl * e;
#pragma unroll
    for (int c = 0; c < 4; ++c) j.o[c] = j.o[c] * f + y[c] * e;
  }
  return j;
}

// Workgroups (blockIdx.y) that join a row's and kv head's o: 1024 / D query heads, a thread four columns (pieces 0, for
// units of few parts), or D / pieces columns of one head, a thread some of the parts
template <int D>
CATENA_DEV uint32_t joins_of(const AttnPagedArgs& a, uint32_t pieces) {
  return pieces ? a.group * pieces : (a.group * (D / 4) + 255) / 256;
}
// The o of the units that were cut (and 0 of rows without slots).  blockIdx.x: the kv head, blockIdx.z: rows in turn.
template <int D, bool F32>
CATENA_DEV void join_o(const AttnPagedArgs& a, const FirstRows& rows, const Line& line, uint32_t pieces) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  __shared__ f32x2 s_ml[64];
  __shared__ __attribute__((aligned(16))) float s_o[256 * 4];
  constexpr uint32_t LANES = D / 4;
  const uint32_t tid = threadIdx.x, heads = a.group * a.kv.kv_heads, kvh = blockIdx.x;
  const uint32_t quarters = pieces == 4 ? 2 : 0;  // pieces: 0, 1 or 4
  if (line.whole) return;
  const uint32_t lanes = LANES >> quarters;  // of a head's columns, 16 bytes each
  const uint32_t head = pieces ? blockIdx.y >> quarters : blockIdx.y * (256 / LANES) + tid / LANES;
  const uint32_t col = (pieces == 4 ? blockIdx.y % 4 * lanes * 4 : 0u) + tid % lanes * 4;
  const uint32_t mine = tid / lanes, step = 256 / lanes;
  for (uint32_t row = blockIdx.z; row < a.kv.rows; row += gridDim.z) {
    const RowOnLine r = row_on_line(a, rows, row);
    const uint64_t at = ((uint64_t)row * heads + kvh * a.group + head) * D + col;
    const Parts p = parts_of(line, r, kvh * a.head_tiles + head / 16);
    if (!pieces) {
      if (head >= a.group || p.n == 1) continue;
      const Joined j = join_parts<D>(a, p, head % 16, col, 0, 1);
      store_o<F32>(a, at, j.o, j.l, r.len);
      continue;
    }
    if (p.n == 1) continue;
    const Joined j = join_parts<D>(a, p, head % 16, col, mine, step);
    __syncthreads();  // the last one's values have been read
    *reinterpret_cast<f32x4_t*>(&s_o[4 * tid]) = j.o;
    if (tid % lanes == 0) s_ml[mine] = f32x2{j.m, j.l};
    __syncthreads();
    if (tid < lanes) {
      float m = kNegInf, l = 0.0f;
      f32x4_t o = f32x4_t{0, 0, 0, 0};
      for (uint32_t i = 0; i < step; ++i) m = __builtin_fmaxf(m, s_ml[i][0]);
      for (uint32_t i = 0; i < step; ++i) {
        const float f = exp2_fast(s_ml[i][0] - anchor(m));
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(&s_o[4 * (i * lanes + tid)]);
        l = l + s_ml[i][1] * f;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = o[c] + y[c] * f;
      }
      store_o<F32>(a, at, o, l, r.len);
    }
  }
}

}  // namespace
