// Attention of one new token per row over a key-value cache in pages.
//
//   s_j = scale * q . k_j,  p_j = exp(s_j - max) / sum,  o = sum_j p_j v_j
//
// over the row's first lens[row] slots, grouped heads (query head h reads kv
// head h / (heads / kv_heads)); a row without slots gives 0.  With weights,
// acc_out[j] = acc_in[j] + the sum of p_j over the query heads of a kv head.
//
// Bound: the cache is read once, 4 D bytes per (slot, kv head), against 4 D
// flops per query head, so HBM.  One pass: the running maximum and sum of the
// softmax beside the running o.
//
// Work is dealt out in one of two ways.  A workgroup takes whole units ((row, kv
// head) and up to 16 query heads) while rows are short; they need no join.  One CU
// brings in about 38 GB/s, so long rows are cut: all units' tiles form one line in
// the order of rows, every workgroup takes an equal stretch of it (ends of units
// in it and all), and a second kernel joins the units that were cut.  The stretches
// follow from the rows' own lengths, so ragged batches are even: 64 rows of 1 ..
// 4096 slots x 8 kv heads of 128 take 85 us (6.3 TB/s) and 5 to join, against 112
// with the rows cut alike; 131072 slots x 8 heads in one row 80 us (6.7 TB/s).
// Where even a full table is short, the host launches a workgroup per unit and no
// join; else both kernels see by the rows' lengths which it is.
//
// A wave takes 32 slots at a time (two runs of 16, each inside one page).
// Products on the matrix cores with the cache as the A operand, straight from
// memory with no transpose through LDS:
//   S^T = K Q^T: lane (c, g) = (lane & 15, lane >> 4) holds slot c, d = 32 i +
//     8 g .. + 7 of K and of query head c; the result holds head c and slots 4 g
//     .. + 3 of either run.
//   O^T = V^T P^T over the 32 slots, whose order in the sum is free: element
//     (g, j) of the sum is the slot that S left in lane group g, register j, so P
//     needs no move.  The lane loads V rows of its own eight slots, columns
//     VC c .. + VC - 1 of each (VC = D / 16), and transposes 8 x VC in
//     registers; product e then gives columns VC m + e, m = 0 .. 15, so that
//     lane (c, g) ends with o of head c, columns 4 VC g .. + 4 VC - 1.
// Heads past the group's last fill the 16 columns with zeros; the matrix cores
// have time for that (64 D flop of one slot against its 4 D bytes).
//
// Rounding: scores and sums in f32.  p goes into the product as bf16 terms,
// each the upper half of what the one before left over: three (all 24 bits) for
// an f32 output, two (2^-16 relative) for a bf16 one; the further products hide
// under the cache's stream (1 to 3 % of a bf16 output's time).  A term that would be 0
// behind another is 2^-30 p instead, so that an infinity in V gives infinity and not 0 *
// infinity.
//
// The maximum is raised only where a score passes it by more than 8 in base 2,
// for all lanes of a head at once: until then p stays below 2^8, which costs no
// accuracy, and most tiles need no exchange between lanes.
//
// Range: the sums of p v are divided by that of p at the end alone.  p enters the
// products times a power of two below 2^-8 / n, so that no sum passes half the
// largest |v| and any finite values give a finite mean; the division takes the
// power back.  (It costs the other end: products of values below some 2^-80 are f32's
// smallest numbers and lose their last bits.)
#include "common.h"
#include "paged.h"

namespace {
// long parts go to one workgroup a CU (D = 128, 32768 tiles: 83.1 us against 85.3 with
// two; D = 64, whose tiles are half as long, ragged rows: 59.6 against 57.3)
constexpr uint32_t kTileSlots = 32, kOneACu = 16384, kTwoACu = 0, kWholeShare = 0, kWholeMost = 0;
}  // namespace

#include "attn_line.h"

namespace {

// p of heads h0 .. + hn - 1 (of 2^(score - base[h]) share[h]) summed over them, four
// slots at a time from `slot` on, and added to the slots' weights
CATENA_DEV void add_weights(const AttnPagedArgs& a, uint32_t row, uint32_t kvh, uint32_t h0, uint32_t hn, uint32_t len,
                            uint32_t slot, uint32_t step, const float* base, const float* share) {
  const uint32_t slots = paged_slots(a.kv);
  const uint64_t pair = (uint64_t)row * a.kv.kv_heads + kvh;
  const float* scores = a.scores + (pair * a.group + h0) * slots;
  const float* in = (h0 ? a.acc_out : a.acc_in) + pair * slots;
  float* out = a.acc_out + pair * slots;
  for (; slot < len; slot += step) {  // slots come in whole pages of 16 or more
    f32x4_t w = f32x4_t{0, 0, 0, 0};
#pragma unroll 2
    for (uint32_t h = 0; h < hn; ++h) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(scores + (uint64_t)h * slots + slot);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = w[i] + exp2_fast(x[i] - base[h]) * share[h];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (slot + i < len) out[slot + i] = in[slot + i] + w[i];
  }
}

// Two runs of 16 slots of a tile, as a wave holds them
template <int D>
struct Tile {
  uint32_t n[2];            // slots that count
  u32x4_t k[2][D / 32];     // slot c, d = 32 i + 8 g ..
  uint32_t v[8][D / 32];    // slot 4 g + j % 4 of run j / 4, columns (D / 16) c ..
};

constexpr int kWaves = 4;

// What a workgroup's waves hand over to each other; rows of o are padded, which
// keeps the lanes of a 16-byte store off each other's banks
template <int D>
struct Shared {
  float m[kWaves][16], l[kWaves][16];
  __attribute__((aligned(16))) float o[kWaves][16][D + 4];
  float base[16], share[16];
};

template <int D, bool F32, bool WEIGHTS>
CATENA_DEV void attn_paged_run(const AttnPagedArgs& a) {
  constexpr int KC = D / 32;  // K loads of 8 values, products of S
  constexpr int VC = D / 16;  // columns of V a lane takes
  constexpr int kNonTemporal = 2;
  __shared__ Shared<D> sh;
  const uint32_t lane = threadIdx.x & 63u, c = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t heads = a.group * a.kv.kv_heads, slots = paged_slots(a.kv);
  const uint32_t part_heads = a.group < 16 ? a.group : 16;
  const uint32_t mask = (1u << a.kv.page_shift) - 1u;
  const int koff = (int)(c * D + 8 * g) * 2, voff = (int)(4 * g * D + VC * c) * 2;

  // The rows of a tile, through descriptors that end with those that count:
  // what lies behind the row's end (it may be anything), or in a page that is
  // not there, is not read and comes as 0.
  auto request = [&](Tile<D>& x, const Part& p, uint32_t t) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t slot = 32 * t + 16 * u;
      const bool in = t < p.end && slot < p.len;
      const uint32_t page =
          in ? scalar_word(a.kv.table + (uint64_t)p.row * a.kv.max_pages, slot >> a.kv.page_shift) : 0xFFFFFFFFu;
      const bool here = page < a.kv.num_pages;
      x.n[u] = !here ? 0u : p.len - slot < 16 ? p.len - slot : 16u;
      const uint64_t at = here ? paged_offset(a.kv, page, p.kvh, slot & mask) : 0ull;
      const int bytes = (int)(x.n[u] * D * 2);
      const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kv.k + at), (short)0, bytes, 0x00020000);
      const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kv.v + at), (short)0, bytes, 0x00020000);
#pragma unroll
      for (int i = 0; i < KC; ++i) x.k[u][i] = __builtin_amdgcn_raw_buffer_load_b128(kr, koff, 64 * i, kNonTemporal);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (VC == 8) {
          const u32x4_t w = __builtin_amdgcn_raw_buffer_load_b128(vr, voff, j * D * 2, kNonTemporal);
#pragma unroll
          for (int y = 0; y < 4; ++y) x.v[4 * u + j][y] = w[y];
        } else {
          typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
          const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(vr, voff, j * D * 2, kNonTemporal);
          x.v[4 * u + j][0] = w[0];
          x.v[4 * u + j][1] = w[1];
        }
      }
    }
  };
  bf16x8_t qf[KC];
  float m, l, ease;
  f32x4_t acc[VC];
  auto begin = [&](const Part& p) {
    // Q as the B operand: lane = head c, 8 values of each 32-wide block of d
    const uint16_t* q = a.q + ((uint64_t)p.row * heads + p.kvh * a.group + 16 * p.ht + (c < p.gn ? c : 0)) * D;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      u32x4_t w = *reinterpret_cast<const u32x4_t*>(q + 32 * i + 8 * g);
      if (c >= p.gn) w = u32x4_t{0, 0, 0, 0};
      qf[i] = __builtin_bit_cast(bf16x8_t, w);
    }
    m = kNegInf;
    l = 0.0f;
    ease = ease_of(p.len | 1u);
#pragma unroll
    for (int e = 0; e < VC; ++e) acc[e] = f32x4_t{0, 0, 0, 0};
  };

  auto take = [&](Tile<D>& x, const Part& w, uint32_t t) {
    // scores in base 2: s[j] is slot (g, j) of head c
    float s[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4_t y = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KC; ++i)
        y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x.k[u][i]), qf[i], y, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[4 * u + j] = y[j] * a.scale_log2;
    }
    if (x.n[0] < 16 || x.n[1] < 16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = 4 * g + j % 4 < x.n[j / 4] ? s[j] : kNegInf;
    }
    if constexpr (WEIGHTS) {
      if (c < w.gn && t < w.end) {  // an empty tile's slots are another part's
        float* dst = a.scores + ((uint64_t)w.row * heads + w.kvh * a.group + 16 * w.ht + c) * slots + 32 * t + 4 * g;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (32 * t + 16 * u < w.len)
            *reinterpret_cast<f32x4_t*>(dst + 16 * u) = f32x4_t{s[4 * u], s[4 * u + 1], s[4 * u + 2], s[4 * u + 3]};
      }
    }
    float top = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) top = __builtin_fmaxf(top, s[j]);
    if (__any(top > m + 8.0f)) {
      top = __builtin_fmaxf(top, __shfl_xor(top, 16));
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      const float m2 = __builtin_fmaxf(m, top);
      const float f = exp2_fast(m - anchor(m2));
      m = m2;
      l = l * f;
#pragma unroll
      for (int e = 0; e < VC; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[e][i] = acc[e][i] * f;
    }
    const float base = anchor(m);
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = exp2_fast(s[j] - base);
      l = l + p[j];
      p[j] = p[j] * ease;
    }
    // p's bf16 terms
    constexpr int TERMS = F32 ? 3 : 2;
    bf16x8_t pt[TERMS];
    float least[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) least[j] = p[j] * 0x1p-30f;
#pragma unroll
    for (int y = 0; y < TERMS; ++y) {
      u32x4_t word;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (y + 1 < TERMS) {
          const uint32_t b0 = __float_as_uint(p[2 * j]), b1 = __float_as_uint(p[2 * j + 1]);
          word[j] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
          const float hi0 = __uint_as_float(b0 & 0xFFFF0000u), hi1 = __uint_as_float(b1 & 0xFFFF0000u);
          p[2 * j] = __builtin_fmaxf(p[2 * j] - hi0, least[2 * j]);
          p[2 * j + 1] = __builtin_fmaxf(p[2 * j + 1] - hi1, least[2 * j + 1]);
        } else {
          word[j] = pack_bf16x2(p[2 * j], p[2 * j + 1]);
        }
      }
      pt[y] = __builtin_bit_cast(bf16x8_t, word);
    }
#pragma unroll
    for (int e = 0; e < VC; ++e) {
      // column e of the lane's 8 x VC block
      u32x4_t col;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        col[j] = __builtin_amdgcn_perm(x.v[2 * j + 1][e / 2], x.v[2 * j][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
      const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, col);
#pragma unroll
      for (int y = 0; y < TERMS; ++y)
        acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pt[y], acc[e], 0, 0, 0);
    }
  };

  bool whole = a.blocks == 0;  // units are not cut
  auto finish = [&](const Part& p) {
    // The waves' (m, l, o) to one
    l = l + __shfl_xor(l, 16);
    l = l + __shfl_xor(l, 32);
    __syncthreads();  // the last unit's values have been read
    if (g == 0) {
      sh.m[wave][c] = m;
      sh.l[wave][c] = l;
    }
    if (c < p.gn) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VC; e += 4)
          *reinterpret_cast<f32x4_t*>(&sh.o[wave][c][4 * VC * g + VC * i + e]) =
              f32x4_t{acc[e][i], acc[e + 1][i], acc[e + 2][i], acc[e + 3][i]};
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
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(&sh.o[w][h][d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] + x[i] * f;
      }
      const uint32_t head = p.kvh * a.group + 16 * p.ht + h;
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
      const uint64_t to = (uint64_t)p.row * heads + head, at = to * D + d;
      if constexpr (WEIGHTS) {
        if (d == 0 && whole && a.head_tiles == 1) {
          sh.base[h] = anchor(mm);
          sh.share[h] = 1.0f / ll;
        } else if (d == 0) {
          a.whole_ml[2 * to] = mm;
          a.whole_ml[2 * to + 1] = ll;
        }
      }
      store_o<F32>(a, at, o, ll, p.len);
    }
    if constexpr (WEIGHTS) {
      // weights of whole units that are all of their kv head (of the line's the
      // second kernel adds them, strip by strip): the scores are this workgroup's
      // own, behind two barriers
      if (whole && a.head_tiles == 1) {
        __syncthreads();
        add_weights(a, p.row, p.kvh, 0, p.gn, p.len, 4 * threadIdx.x, 1024, sh.base, sh.share);
      }
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

  // The workgroup's parts one after the other, a wave's tiles of each kWaves
  // apart (one without any takes an empty one).  A tile's rows are requested
  // while the tile before it is worked on, across the border of two parts too.
  uint32_t t = now.beg + wave;
  Tile<D> one, two;
  begin(now);
  request(one, now, t);
  auto step = [&](Tile<D>& x, Tile<D>& y) {
    const bool ends = t + kWaves >= now.end, more = at < last;
    Part next = now;
    uint32_t tn = t + kWaves;  // past the end where nothing is left
    if (ends && more) {
      if (whole) {
        next = unit_from(at);
        at += gridDim.x;
      } else {
        next = part_behind(a, now, last - at);
        at += next.end - next.beg;
      }
      tn = next.beg + wave;
    }
    request(y, next, tn);
    __builtin_amdgcn_sched_barrier(0);
    take(x, now, t);
    __builtin_amdgcn_sched_barrier(0);
    if (ends) {
      finish(now);
      if (!more) return false;
      begin(next);
    }
    now = next;
    t = tn;
    return true;
  };
  while (step(one, two) && step(two, one)) {
  }
}

// Joins the units that were cut, writes 0 for rows without slots, and adds the
// weights that the first kernel could not.  blockIdx.x: the kv head, blockIdx.z:
// rows in turn; blockIdx.y < joins: the o of 1024 / D query heads, a thread four
// columns (pieces 0, for units of few parts), or D / pieces columns of one head, a
// thread some of the parts; else 1024 slots' weights.
template <int D, bool F32>
CATENA_DEV void attn_paged_join(const AttnPagedArgs& a, uint32_t pieces) {
  __shared__ float s_m[16], s_r[16];
  const uint32_t tid = threadIdx.x, heads = a.group * a.kv.kv_heads, kvh = blockIdx.x;
  const FirstRows rows = first_rows(a);
  const Line line = line_of(a, rows);
  if (line.whole && (!a.acc_out || a.head_tiles == 1)) return;
  const uint32_t joins = joins_of<D>(a, pieces);
  if (blockIdx.y < joins) {
    join_o<D, F32>(a, rows, line, pieces);
    return;
  }
  const uint32_t slot0 = (blockIdx.y - joins) * 1024;
  for (uint32_t row = blockIdx.z; row < a.kv.rows; row += gridDim.z) {
    const RowOnLine r = row_on_line(a, rows, row);
    if (slot0 >= r.len) continue;
    for (uint32_t h0 = 0; h0 < a.group; h0 += 16) {
      const uint32_t hn = a.group - h0 < 16 ? a.group - h0 : 16;
      const Parts p = parts_of(line, r, kvh * a.head_tiles + h0 / 16);
      __syncthreads();  // the last heads' values have been read
      // 16 lanes a head, a part each
      for (uint32_t h = tid / 16; h < hn; h += 16) {
        float m = kNegInf, l = 0.0f;
        if (line.whole || p.n == 1) {
          const float* x = a.whole_ml + 2 * ((uint64_t)row * heads + kvh * a.group + h0 + h);
          m = x[0];
          l = x[1];
        } else {
          for (uint32_t i = tid % 16; i < p.n; i += 16) m = __builtin_fmaxf(m, a.part_ml[2 * part_place(a, p, i, h)]);
#pragma unroll
          for (int d = 1; d < 16; d *= 2) m = __builtin_fmaxf(m, __shfl_xor(m, d));
          for (uint32_t i = tid % 16; i < p.n; i += 16) {
            const float* x = a.part_ml + 2 * part_place(a, p, i, h);
            l = l + x[1] * exp2_fast(x[0] - anchor(m));
          }
#pragma unroll
          for (int d = 1; d < 16; d *= 2) l = l + __shfl_xor(l, d);
        }
        if (tid % 16 == 0) {
          s_m[h] = anchor(m);
          s_r[h] = 1.0f / l;
        }
      }
      __syncthreads();
      add_weights(a, row, kvh, h0, hn, r.len, slot0 + 4 * tid, 0x80000000u, s_m, s_r);  // slots < 2^31: once
    }
  }
}

}  // namespace

#define CATENA_ATTN_PAGED(D, OUT, F32)                                                                      \
  extern "C" __global__ __launch_bounds__(256, 2) void catena_attn_paged_d##D##_##OUT(AttnPagedArgs a) {      \
    attn_paged_run<D, F32, false>(a);                                                                      \
  }                                                                                                         \
  extern "C" __global__ __launch_bounds__(256, 2) void catena_attn_paged_weights_d##D##_##OUT(AttnPagedArgs a) { \
    attn_paged_run<D, F32, true>(a);                                                                       \
  }                                                                                                         \
  extern "C" __global__ __launch_bounds__(256) void catena_attn_paged_join_d##D##_##OUT(AttnPagedArgs a,      \
                                                                                        uint32_t pieces) {    \
    attn_paged_join<D, F32>(a, pieces);                                                                       \
  }
CATENA_ATTN_PAGED(128, f32out, true)
CATENA_ATTN_PAGED(128, bf16out, false)
CATENA_ATTN_PAGED(64, f32out, true)
CATENA_ATTN_PAGED(64, bf16out, false)
