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
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) i16x4_t lds_i16x4;

CATENA_DEV uint32_t lane_of(uint32_t x, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)lane); }
CATENA_DEV float anchor(float m) { return m == kNegInf ? 0.0f : m; }

// A uniform word that this kernel does not write, by a scalar load
CATENA_DEV uint32_t scalar_word(const uint32_t* p, uint64_t i) {
  typedef const uint32_t __attribute__((address_space(4))) * word;
  return ((word)(uintptr_t)p)[i];
}

// Where chunk `chunk` (16 bytes) of row `row` of a tile lies in its row
template <int D>
CATENA_DEV uint32_t swizzle_k(uint32_t row, uint32_t chunk) {
  return D == 128 ? chunk ^ (row & 15u) : chunk ^ (row >> 1 & 7u);
}
template <int D>
CATENA_DEV uint32_t swizzle_v(uint32_t row, uint32_t chunk) {
  return D == 128 ? chunk ^ (4 * (row & 3u)) : chunk ^ (4 * (row >> 1 & 1u));
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

template <int D, bool PAGED>
CATENA_DEV void attn_prompt_run(const AttnPromptArgs& a) {
  constexpr int KS = D / 16;   // steps of a score's sum
  constexpr int DB = D / 32;   // blocks of o's columns
  constexpr int kTile = kKeys * D;  // elements of K or V of a tile
  constexpr int kRowsAtOnce = 512 / D;  // rows that one load brings (1 KiB)
  constexpr int kLoads = 16 / kRowsAtOnce;  // loads of a wave's 16 rows
  extern __shared__ __attribute__((aligned(1024))) uint16_t smem[];  // K, V, K, V
  const uint32_t lane = threadIdx.x & 63u, c = lane & 31u, h = lane >> 5;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t kvh = blockIdx.x % a.kv.kv_heads, heads = a.group * a.kv.kv_heads;
  const Unit unit = unit_of(a, blockIdx.x / a.kv.kv_heads, 128);
  if (!unit.any) return;
  // slots in use, and how many of them lie before the new tokens
  uint32_t len = unit.n;
  if (a.lens) len = scalar_word(a.lens, unit.row);
  if (PAGED) len = paged_len(a.kv, len);
  const int32_t old = (int32_t)len - (int32_t)unit.n;  // below 0: the first tokens see nothing

  // the lane's query row
  const uint32_t m_row = unit.tile * 128 + wave * 32 + c, t = m_row / a.group, head = kvh * a.group + m_row % a.group;
  const bool live = t < unit.n;
  const uint64_t q_at = ((uint64_t)(unit.first + (live ? t : 0u)) * heads + (live ? head : kvh * a.group)) * D;
  const int32_t sees = live ? old + (int32_t)t + 1 : 0;  // slots
  bf16x8_t qf[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    u32x4_t w = *reinterpret_cast<const u32x4_t*>(a.q + q_at + 16 * i + 8 * h);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] ^= a.flip;
    qf[i] = __builtin_bit_cast(bf16x8_t, w);
  }
  // tiles: as far as the workgroup's last token sees
  const uint32_t last_t = (unit.tile * 128 + 127) / a.group, t_end = last_t < unit.n ? last_t + 1 : unit.n;
  const int32_t most = old + (int32_t)t_end;
  const uint32_t tiles = most > 0 ? ((uint32_t)most + kKeys - 1) / kKeys : 0u;
  // slots that all of the wave's rows see (rows that are not live see none, and need not)
  const uint32_t t_first = (unit.tile * 128 + wave * 32) / a.group;
  const int32_t all_see = t_first < unit.n ? old + (int32_t)t_first + 1 : 0x7FFFFFFF;

  // Loads: wave w brings slots 16 w .. 16 w + 15 of a tile, a run inside one page
  const uint32_t l_row = lane / (D / 8), l_chunk = lane % (D / 8);
  const uint32_t row_bytes = PAGED ? D * 2 : (uint32_t)(a.stride * 2);
  uint32_t k_off[kLoads], v_off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t r = kRowsAtOnce * i + l_row;  // (16 w does not change the swizzles)
    k_off[i] = r * row_bytes + 16 * swizzle_k<D>(r, l_chunk);
    v_off[i] = r * row_bytes + 16 * swizzle_v<D>(r, l_chunk);
  }
  auto page_of = [&](uint32_t slot) -> uint32_t {
    if constexpr (PAGED) return slot < len ? scalar_word(a.kv.table, (uint64_t)unit.row * a.kv.max_pages + (slot >> a.kv.page_shift)) : 0xFFFFFFFFu;
    return 0;
  };
  auto issue = [&](uint32_t tile, uint32_t buffer) {
    const uint32_t slot = tile * kKeys + 16 * wave;
    uint32_t n = slot < len ? (len - slot < 16 ? len - slot : 16u) : 0u;
    uint64_t at = 0;
    if constexpr (PAGED) {
      const uint32_t page = page_of(slot);
      if (page < a.kv.num_pages)
        at = paged_offset(a.kv, page, kvh, slot & ((1u << a.kv.page_shift) - 1u));
      else
        n = 0;
    } else {
      at = ((uint64_t)unit.first + (n ? slot : 0u)) * a.stride + kvh * D;
    }
    const int bytes = n ? (int)((n - 1) * row_bytes + D * 2) : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kv.k + at), (short)0, bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(a.kv.v + at), (short)0, bytes, 0x00020000);
    uint16_t* dst = smem + buffer * 2 * kTile + 16 * wave * D;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void*)(dst + kRowsAtOnce * i * D), 16, (int)k_off[i], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void*)(dst + kTile + kRowsAtOnce * i * D), 16, (int)v_off[i], 0, 0, 0);
  };

  const float raise = 8.0f / a.scale_log2;
  float m = kNegInf, l = 0.0f;  // the maximum in units of the products; l of the lane's half of the slots
  f32x16_t acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;

  // V's operand: block d of the columns, step s of 16 slots: two transposed reads of 4 slots x 16 columns by
  // 16 lanes each
  const uint32_t v_key = 4 * h + ((lane & 15u) >> 2), v_col = 16 * (lane >> 4 & 1u) + 4 * (lane & 3u);
  auto v_frag = [&](const uint16_t* v, int d, int s) {
    u32x4_t w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t key = 16 * s + 8 * e + v_key, col = 32 * d + v_col;
      const i16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_i16x4*)(v + key * D + 8 * swizzle_v<D>(key, col >> 3) + (col & 7u)));
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 y = __builtin_bit_cast(u32x2, x);
      w[2 * e] = y[0];
      w[2 * e + 1] = y[1];
    }
    return w;
  };

  auto take = [&](uint32_t tile, uint32_t buffer, auto masked) {
    const uint16_t* k = smem + buffer * 2 * kTile;
    const uint16_t* v = k + kTile;
    f32x16_t s[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const uint32_t key = 32 * b + c;
        const bf16x8_t kf = __builtin_bit_cast(
            bf16x8_t, *reinterpret_cast<const u32x4_t*>(k + key * D + 8 * swizzle_k<D>(key, 2 * i + h)));
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[i], s[b], 0, 0, 0);
      }
    }
    if constexpr (masked.value) {
      const int32_t left = sees - (int32_t)(tile * kKeys) - 4 * (int32_t)h;
      uint32_t runs = 0xFu;  // runs of 16 slots whose page exists
      if constexpr (PAGED) {
        runs = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) runs |= (page_of(tile * kKeys + 16 * r) < a.kv.num_pages ? 1u : 0u) << r;
      }
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool seen = 32 * b + 8 * (i / 4) + i % 4 < left && (runs >> (2 * b + i / 8) & 1u);
          s[b][i] = seen ? s[b][i] : kNegInf;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, s[b][i]);
    if (__any(top > m + raise)) {
      top = __builtin_fmaxf(top, __shfl_xor(top, 32));
      const float m2 = __builtin_fmaxf(m, top);
      const float f = __builtin_amdgcn_exp2f((m - anchor(m2)) * a.scale_log2);
      m = m2;
      l = l * f;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = acc[d][i] * f;
    }
    const float base = anchor(m) * a.scale_log2 + kEase;
    bf16x8_t p[4];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        u32x4_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * x + 2 * i], a.scale_log2, -base));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * x + 2 * i + 1], a.scale_log2, -base));
          l = l + e0;
          l = l + e1;
          w[i] = pack_bf16x2(e0, e1);
        }
        p[2 * b + x] = __builtin_bit_cast(bf16x8_t, w);
      }
    bool odd = false;
    if constexpr (masked.value) {
      uint32_t found = 0;
#pragma unroll 4
      for (uint32_t i = lane; i < kTile / 8; i += 64) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(v + 8 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) found |= ((w[j] & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
      }
      odd = __any(found != 0);
    }
    if (!odd) {
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int d = 0; d < DB; ++d)
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, v_frag(v, d, x)), p[x], acc[d], 0, 0, 0);
    } else if constexpr (masked.value) {
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
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(only(0, d, x), p[x], acc[d], 0, 0, 0);
#pragma unroll 1
        for (int kind = 1; kind < 4; ++kind) {
          f32x16_t r;
#pragma unroll
          for (int i = 0; i < 16; ++i) r[i] = 0.0f;
#pragma unroll
          for (int x = 0; x < 4; ++x) r = __builtin_amdgcn_mfma_f32_32x32x16_bf16(only(kind, d, x), p[x], r, 0, 0, 0);
          const float what = kind == 1 ? -kNegInf : kind == 2 ? kNegInf : __builtin_nanf("");
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[d][i] = acc[d][i] + (r[i] > 0.0f ? what : 0.0f);
        }
      }
    }
  };

  auto barrier = [&]() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (tiles > 0) issue(0, 0);
  for (uint32_t i = 0; i < tiles; ++i) {
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0): the wave's rows of this tile are in LDS; lgkmcnt(0): it has read the other buffer
    barrier();
    if (i + 1 < tiles) issue(i + 1, (i + 1) & 1u);
    bool whole = (int32_t)((i + 1) * kKeys) <= all_see;
    if constexpr (PAGED) {
#pragma unroll
      for (int r = 0; r < 4; ++r) whole = whole && page_of(i * kKeys + 16 * r) < a.kv.num_pages;
    }
    if (whole)
      take(i, i & 1u, std::false_type{});
    else
      take(i, i & 1u, std::true_type{});
  }

  l = l + __shfl_xor(l, 32);
  if (!live) return;
  const float by = sees > 0 ? l : 1.0f;
  uint16_t* o = a.o + q_at;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      uint2 w;
      w.x = pack_bf16x2(acc[d][i] / by, acc[d][i + 1] / by);
      w.y = pack_bf16x2(acc[d][i + 2] / by, acc[d][i + 3] / by);
      *reinterpret_cast<uint2*>(o + 32 * d + 8 * (i / 4) + 4 * h) = w;
    }
}

}  // namespace

// grid = kv_heads * tiles of 128 query rows that there may be, heads fastest
#define CATENA_ATTN_PROMPT(D, NAME, PAGED)                                                                   \
  extern "C" __global__ __launch_bounds__(256, 2) void catena_attn_##NAME##_d##D(AttnPromptArgs a) { \
    attn_prompt_run<D, PAGED>(a);                                                                            \
  }
CATENA_ATTN_PROMPT(128, prompt, true)
CATENA_ATTN_PROMPT(64, prompt, true)
CATENA_ATTN_PROMPT(128, packed, false)
CATENA_ATTN_PROMPT(64, packed, false)
