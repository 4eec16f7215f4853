// Attention of one new token per row over a key-value cache held in 4 bits.
//
//   k_j = 2^(e - 127) c (a power of two for 32 values), v_j = s_j c (one scale a
//   slot and head), c in e2m1; s_j = scale * q . k_j, o = softmax(s) . v
//
// as attn_paged.hip has it for bf16: the same line of tiles, parts and join.
//
// Bound: the cache is read once, D + D / 32 + 2 bytes per (slot, kv head), so HBM, beside
// about 1000 vector instructions of a wave for 128 slots of 128 columns (15800 a SIMD
// in 121000 cycles of a ragged batch, half of its time by the counter of active ones).  64 rows x
// 4096 slots x 8 kv heads of 128 take 57 us (281 MB, 4.9 TB/s), 64 of 1 .. 8192 62 to 75 by the lengths (as
// bf16 pages 88 for half the slots), one row of 131072 of 64 columns 25 (6 the join), one of
// 640 and 16 heads 9 to 10.
//
// A wave takes 128 slots at a time, its lane group g (lanes 16 g ..) slots 32 g ..
// 32 g + 31 of them.
//   S^T = K Q^T (16 x 16 x 32 products): instruction set u of eight takes slots 32 (c
//     / 4) + 4 u + c % 4 as its 16 rows, so that the results leave lane (c, g) with
//     head c's scores of its own group's slots 32 g + 4 u + j (j: the register).  The
//     order of d in the sum is free: the lane loads a quarter of a slot's codes, D / 8
//     bytes, which lie in one block of 32, and converts them with that block's scale
//     (two values an instruction).
//   O^T = V^T P^T: v lies by pairs of columns, so a lane's 32 slots of one pair are 32
//     bytes in two runs of 16.  Halves of two dwords mixed give eight codes of one
//     column, slots (0, 4, 1, 5, 2, 6, 3, 7), and P's terms are packed in that order.
//     The slots' scales go into P.
// P enters as two bf16 terms, together exact to 2^-16.  Up to 8 heads stand in a product's
// 16 columns twice, and the second ones take the second term; more heads need a second
// product.
// K of the next 128 slots is asked for as soon as the scores are there, V once it has been
// read, or of the workgroup's next unit or part of one, so that a wave's loads are under way
// all the time (64 rows of 1 .. 8192 slots: 74.7 us without the next part's, 70.4 with).
//
// Codes are finite whatever their bits, so what lies behind a row's end is masked in
// the scores and the scales alone.
#include "common.h"
#include "paged.h"

namespace {
constexpr int kWaves = 4;
constexpr uint32_t kTileSlots = kAttnQ4Slots, kOneACu = 0xFFFFFFFFu, kTwoACu = kAttnQ4TwoACu;
constexpr uint32_t kWholeShare = kAttnQ4WholeShare, kWholeMost = kAttnQ4WholeMost;
static_assert(kTileSlots == 128 * kWaves, "a turn of a workgroup");
}  // namespace

#include "attn_line.h"

namespace {

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

template <int D>
struct Shared {
  float m[kWaves][16], l[kWaves][16];
  __attribute__((aligned(16))) float o[kWaves][16][D + 4];
};

// Eight codes times a power of two, in bf16 (exact)
CATENA_DEV bf16x8_t widen8(uint32_t codes, float unit) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, unit, 0);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, unit, 1);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, unit, 2);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, unit, 3);
  return __builtin_bit_cast(bf16x8_t, u32x4_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                                              __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)});
}

template <int D>
struct Tile {
  u32x4_t k[8];          // D = 64: the first two dwords
  u32x4_t ks[2];         // block scales of the 32 slots of group c / 4
  u32x4_t v[D / 32][2];  // pair of columns 16 i + c, slots 16 h .. + 15 of the lane's group
  u32x4_t vs[2][2];      // their scales
};

// TWICE: groups of up to 8 heads, which stand in columns c and c + 8
template <int D, bool TWICE>
CATENA_DEV void attn_paged_q4_run(const AttnPagedArgs& a, const AttnQ4Pools& pools) {
  constexpr int KC = D / 32;  // products of S
  constexpr int VG = D / 32;  // groups of 16 column pairs
  __shared__ Shared<D> sh;
  const uint32_t lane = threadIdx.x & 63u, c = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t heads = a.group * a.kv.kv_heads;
  const uint32_t part_heads = a.group < 16 ? a.group : 16;
  const uint32_t head = TWICE ? c & 7u : c;
  const uint32_t page_size = 1u << a.kv.page_shift, mask = page_size - 1u;

  // (the lane's number by a register of its own, so that no address parts are kept through the loop: there is no
  // room)
  auto own_lane = [&] {
    uint32_t x = lane;
    asm("" : "+v"(x));
    return x;
  };
  // Pages of the tile's eight runs of 16 slots.  Looked up by lanes, run lane % 8, a turn before the loads that they
  // say where to find: so nothing waits for them that does not wait for older loads too.
  struct Pages {
    uint32_t n[8];
    CATENA_DEV uint32_t of(uint32_t group, int run) const {
      const uint32_t low = group & 1u ? n[2 + run] : n[run], high = group & 1u ? n[6 + run] : n[4 + run];
      return group & 2u ? high : low;
    }
  };
  auto look_up = [&](const Part& p, uint32_t slot, uint32_t end) {
    const uint32_t s = slot + 16 * (own_lane() & 7u);
    const uint32_t page = (a.kv.table + (uint64_t)p.row * a.kv.max_pages)[(s < end ? s : 0u) >> a.kv.page_shift];
    return s < end ? page : 0xFFFFFFFFu;
  };
  auto spread = [&](uint32_t pages) {
    Pages x;
#pragma unroll
    for (uint32_t r = 0; r < 8; ++r) x.n[r] = lane_of(pages, r);
    return x;
  };
  // (what is not there is read from the pool's first page and masked)
  auto request_k = [&](Tile<D>& x, uint32_t kvh, uint32_t slot, const Pages& at) {
    const uint32_t me = own_lane(), c = me & 15u, g = me >> 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t s = (slot + 32 * (c >> 2) + 16 * r) & mask;
      const uint32_t page = at.of(c >> 2, r);
      const uint64_t kc = paged_cells(a.kv.kv_heads, a.kv.page_shift, page < a.kv.num_pages ? page : 0u, kvh);
      const uint8_t* k = pools.k + (kc + s + (c & 3u)) * (D / 2) + g * (D / 8);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if constexpr (D == 128) {
          x.k[4 * r + u] = *reinterpret_cast<const u32x4_t*>(k + 4 * u * (D / 2));
        } else {
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(k + 4 * u * (D / 2));
          x.k[4 * r + u][0] = w[0];
          x.k[4 * r + u][1] = w[1];
        }
      }
      x.ks[r] = *reinterpret_cast<const u32x4_t*>(pools.k_scale + kc * (D / 32) + (uint64_t)(g * (D / 32) / 4) * page_size + s);
    }
  };
  auto request_v = [&](Tile<D>& x, uint32_t kvh, uint32_t slot, const Pages& at) {
    const uint32_t me = own_lane(), c = me & 15u, g = me >> 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t s = (slot + 32 * g + 16 * r) & mask;
      const uint32_t page = at.of(g, r);
      const uint64_t vc = paged_cells(a.kv.kv_heads, a.kv.page_shift, page < a.kv.num_pages ? page : 0u, kvh);
      const uint8_t* v = pools.v + vc * (D / 2) + (uint64_t)c * page_size + s;
#pragma unroll
      for (int i = 0; i < VG; ++i) x.v[i][r] = *reinterpret_cast<const u32x4_t*>(v + (uint64_t)(16 * i) * page_size);
      const u32x4_t* vs = reinterpret_cast<const u32x4_t*>(pools.v_scale + vc + s);
      x.vs[r][0] = vs[0];
      x.vs[r][1] = vs[1];
    }
  };

  // m: the head's reference point (base 2); p and l are kept times ease
  bf16x8_t qf[KC];
  float m, limit, l, ease_log2;
  f32x4_t acc[VG][2];
  auto begin = [&](const Part& p) {
    const uint16_t* q = a.q + ((uint64_t)p.row * heads + p.kvh * a.group + 16 * p.ht + (head < p.gn ? head : 0)) * D;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      u32x4_t w = *reinterpret_cast<const u32x4_t*>(q + (D / 4) * g + 8 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = head < p.gn ? w[j] ^ pools.flip : 0u;
      qf[i] = __builtin_bit_cast(bf16x8_t, w);
    }
    m = limit = kNegInf;
    l = 0.0f;
    ease_log2 = (float)(__builtin_clz(p.len | 1u) - 41);  // of ease_of
#pragma unroll
    for (int i = 0; i < VG; ++i) acc[i][0] = acc[i][1] = f32x4_t{0, 0, 0, 0};
  };

  // s[4 u + j]: slot 32 g + 4 u + j of the head, in units of the products
  auto scores = [&](const Tile<D>& x, float (&s)[32]) {
    const uint32_t c = own_lane() & 15u;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t byte = x.ks[u / 4][u % 4] >> (8 * (c & 3u)) & 255u;
      const float unit = __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
      f32x4_t y = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KC; ++i)
        y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(x.k[u][i], unit), qf[i], y, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[4 * u + j] = y[j];
      if (u % 2) __builtin_amdgcn_sched_barrier(0);  // (few registers over those of the loads)
    }
  };
  auto take = [&](const Tile<D>& x, float (&s)[32], const Part& p, uint32_t slot, const Pages& at) {
    bool full = slot + 128 <= p.len;
#pragma unroll
    for (int r = 0; r < 8; ++r) full = full & (at.n[r] < a.kv.num_pages);
    if (!full) {
      const uint32_t g = own_lane() >> 4;
      const uint32_t first = slot + 32 * g;
      const bool here0 = at.of(g, 0) < a.kv.num_pages, here1 = at.of(g, 1) < a.kv.num_pages;
#pragma unroll
      for (int i = 0; i < 32; ++i) s[i] = first + i < p.len && (i < 16 ? here0 : here1) ? s[i] : kNegInf;
    }
    float top = s[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) top = __builtin_elementwise_maximum(top, s[i]);
    if (__any(top > limit)) {
      top = __builtin_fmaxf(top, __shfl_xor(top, 16));
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      const float m2 = __builtin_fmaxf(m, top * a.scale_log2);
      const float f = exp2_fast(m - anchor(m2));
      m = m2;
      limit = (m2 + 8.0f) / a.scale_log2;
      l = l * f;
#pragma unroll
      for (int i = 0; i < VG; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][0][j] = acc[i][0][j] * f;
          acc[i][1][j] = acc[i][1][j] * f;
        }
    }
    const float base = ease_log2 - anchor(m);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // eight slots: p to l, times the slots' scales to two bf16 terms
      float p8[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float e = exp2_fast(__builtin_fmaf(s[8 * j + u], a.scale_log2, base));
        l = l + e;
        const uint32_t w = x.vs[j / 2][j % 2][u / 2];
        p8[u] = e * (u % 2 ? bf16hi(w) : bf16lo(w));
        if (!full) p8[u] = s[8 * j + u] == kNegInf ? 0.0f : p8[u];  // a scale that is not the row's may be anything
      }
      u32x4_t hi, lo;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        hi[b] = pack_bf16x2(p8[b], p8[b + 4]);
        lo[b] = pack_bf16x2(p8[b] - bf16lo(hi[b]), p8[b + 4] - bf16hi(hi[b]));
        if (TWICE) hi[b] = c >= 8 ? lo[b] : hi[b];
      }
      const bf16x8_t p0 = __builtin_bit_cast(bf16x8_t, hi), p1 = __builtin_bit_cast(bf16x8_t, lo);
#pragma unroll
      for (int i = 0; i < VG; ++i) {
        const uint32_t w0 = x.v[i][j / 2][2 * (j % 2)], w1 = x.v[i][j / 2][2 * (j % 2) + 1];
        const uint32_t even = (w0 & 0x0F0F0F0Fu) | (w1 << 4 & 0xF0F0F0F0u);
        const uint32_t odd = (w0 >> 4 & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u);
        const bf16x8_t v0 = widen8(even, 1.0f), v1 = widen8(odd, 1.0f);
        acc[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, p0, acc[i][0], 0, 0, 0);
        acc[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, p0, acc[i][1], 0, 0, 0);
        if (!TWICE) {
          acc[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, p1, acc[i][0], 0, 0, 0);
          acc[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, p1, acc[i][1], 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  bool whole = a.blocks == 0;  // units are not cut
  auto finish = [&](const Part& p) {
    l = l + __shfl_xor(l, 16);
    l = l + __shfl_xor(l, 32);
    l = l * __uint_as_float((uint32_t)(127 - (int)ease_log2) << 23);
    if constexpr (TWICE) {
#pragma unroll
      for (int i = 0; i < VG; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][0][j] = acc[i][0][j] + __shfl_xor(acc[i][0][j], 8);
          acc[i][1][j] = acc[i][1][j] + __shfl_xor(acc[i][1][j], 8);
        }
    }
    __syncthreads();  // the last unit's values have been read
    if (g == 0) {
      sh.m[wave][c] = m;
      sh.l[wave][c] = l;
    }
    if (c < p.gn) {
      // lane (c, g), register j of acc[i][e]: column 2 (16 i + 4 g + j) + e of head c
#pragma unroll
      for (int i = 0; i < VG; ++i)
#pragma unroll
        for (int j = 0; j < 4; j += 2)
          *reinterpret_cast<f32x4_t*>(&sh.o[wave][c][2 * (16 * i + 4 * g + j)]) =
              f32x4_t{acc[i][0][j], acc[i][1][j], acc[i][0][j + 1], acc[i][1][j + 1]};
    }
    __syncthreads();
    for (uint32_t id = threadIdx.x; id < p.gn * (D / 4); id += 64 * kWaves) {
      const uint32_t h = id / (D / 4), d = id % (D / 4) * 4;
      float mm = kNegInf;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) mm = __builtin_fmaxf(mm, sh.m[w][h]);
      float ll = 0.0f;
      f32x4_t o = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = exp2_fast(sh.m[w][h] - anchor(mm));
        ll = ll + sh.l[w][h] * f;
        const f32x4_t y = *reinterpret_cast<const f32x4_t*>(&sh.o[w][h][d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] + y[i] * f;
      }
      if (p.beg != 0 || p.end != p.tiles) {
        // the first part of a unit in the workgroup's second place, else the first
        const uint64_t at = ((uint64_t)blockIdx.x * 2 + (p.beg == 0)) * part_heads + h;
        if (d == 0) {
          a.part_ml[2 * at] = mm;
          a.part_ml[2 * at + 1] = ll;
        }
        *reinterpret_cast<f32x4_t*>(a.part_o + at * D + d) = o;
        continue;
      }
      store_o<false>(a, ((uint64_t)p.row * heads + p.kvh * a.group + 16 * p.ht + h) * D + d, o, ll, p.len);
    }
  };

  // what is left behind `now`: places of the line, or whole units
  const uint32_t units = a.kv.kv_heads * a.head_tiles;
  uint32_t at, last;
  Part now;
  auto unit_from = [&](uint32_t u) {
    const uint32_t row = u / units;
    return part_from(a, row, paged_len(a.kv, scalar_word(a.lens, row)), u % units, 0, 0xFFFFFFFFu);
  };
  if (!whole) {
    const FirstRows rows = first_rows(a);
    const Line line = line_of(a, rows);
    whole = line.whole;
    if (!whole) {
      const Stretch mine = stretch_of(line.tiles, line.per, line.blocks, blockIdx.x);
      if (mine.beg == mine.end) return;
      at = mine.beg;
      last = mine.end;
      const RowOnLine r = row_at_place(a, rows, at);
      now = part_from(a, r.row, r.len, (at - r.first) / r.tiles, (at - r.first) % r.tiles, last - at);
      at += now.end - now.beg;
    }
  }
  if (whole) {
    at = blockIdx.x;
    last = a.kv.rows * units;
    if (at >= last) return;
    now = unit_from(at);
    at += gridDim.x;
  }
  // A tile a turn, 128 slots a wave; a row's last tile may leave a wave without any.  A turn's loads, of the next turn or
  // of the next part's first one, are under way while the one before is worked on.
  auto first_of = [&](const Part& p) { return p.beg * kTileSlots + 128 * wave; };
  auto end_of = [&](const Part& p) { return p.end * kTileSlots < p.len ? p.end * kTileSlots : p.len; };
  Tile<D> x;
  uint32_t slot = first_of(now), end = end_of(now);
  begin(now);
  Pages pages = spread(look_up(now, slot, end));
  if (slot < end) {
    request_k(x, now.kvh, slot, pages);
    request_v(x, now.kvh, slot, pages);
  }
  uint32_t ahead = look_up(now, slot + kTileSlots, end);
  for (;;) {
    const bool more = at < last;
    Part then = now;
    uint32_t then_slot = 0, then_end = 0, behind = 0xFFFFFFFFu;
    if (more) {
      then = whole ? unit_from(at) : part_behind(a, now, last - at);
      at += whole ? gridDim.x : then.end - then.beg;
      then_slot = first_of(then);
      then_end = end_of(then);
      behind = look_up(then, then_slot, then_end);
    }
    if (slot >= end && then_slot < then_end) {
      pages = spread(behind);
      request_k(x, then.kvh, then_slot, pages);
      request_v(x, then.kvh, then_slot, pages);
    }
#pragma clang loop unroll(disable)
    for (; slot < end; slot += kTileSlots) {
      const bool here = !more || slot + kTileSlots < end;
      const uint32_t kvh = here ? now.kvh : then.kvh, s2 = here ? slot + kTileSlots : then_slot;
      float s[32];
      scores(x, s);
      const Pages next = spread(here ? ahead : behind);
      ahead = look_up(now, slot + 2 * kTileSlots, end);
      request_k(x, kvh, s2, next);
      __builtin_amdgcn_sched_barrier(0);
      take(x, s, now, slot, pages);
      request_v(x, kvh, s2, next);
      pages = next;
    }
    finish(now);
    if (!more) return;
    now = then;
    slot = then_slot;
    end = then_end;
    begin(now);
    ahead = look_up(now, slot + kTileSlots, end);
  }
}

}  // namespace

#define CATENA_ATTN_Q4(D, NAME, TWICE)                                                                          \
  extern "C" __global__ __launch_bounds__(256, 2) void catena_attn_paged_q4_##NAME(AttnPagedArgs a, AttnQ4Pools pools) { \
    attn_paged_q4_run<D, TWICE>(a, pools);                                                                      \
  }
CATENA_ATTN_Q4(128, d128, true)
CATENA_ATTN_Q4(64, d64, true)
CATENA_ATTN_Q4(128, d128_wide, false)
CATENA_ATTN_Q4(64, d64_wide, false)

// (grid as the other join's)
extern "C" __global__ __launch_bounds__(256) void catena_attn_paged_q4_join_d128(AttnPagedArgs a, uint32_t pieces) {
  const FirstRows rows = first_rows(a);
  join_o<128, false>(a, rows, line_of(a, rows), pieces);
}
extern "C" __global__ __launch_bounds__(256) void catena_attn_paged_q4_join_d64(AttnPagedArgs a, uint32_t pieces) {
  const FirstRows rows = first_rows(a);
  join_o<64, false>(a, rows, line_of(a, rows), pieces);
}
