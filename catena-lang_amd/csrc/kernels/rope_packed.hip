// Rotary positions of packed tokens, and their keys and values into the slots of
// a slot map: the batch is one list of tokens, each with its position and its
// place in the pool (catena_kv_admit writes both).
//
// qkv[tokens][(heads + 2 kv_heads) * D] (columns: q heads | k heads | v heads) f32
// or bf16.  Of q and k the first `rot` values of a head turn, in pairs (i, i +
// rot / 2) or (2 i, 2 i + 1), by (cos, sin) = tab[position][i]:
//   y1 = x1 c - x2 s, y2 = x2 c + x1 s  (each operation rounded)
// and everything is rounded to bf16.  A token whose slot is no place of the pool
// or whose position is not in the table writes q (turned by tab[0] there) and the
// copies, nothing else.
//
// 4 bits: of the bf16 values, keys in blocks of 32 share the smallest power of two
// 2^e >= 2^-127 with max |x| <= 6 * 2^e, so that nothing is cut off at the largest
// code; a head's value vector shares max |x| / 6 rounded up to bf16.  Codes are the
// nearest e2m1, of two the even one.  A block with an infinity or NaN has the scale
// NaN.
//
// Bound: HBM for prompts, one launch's latency for a decode step.  A workgroup
// serves one token, a thread 16 values of a head: 8 pairs, or 16 that do not turn, so
// that a pair meets in one thread and both its halves are loads of 16 bytes.  Into 4 bits
// a thread then takes 8 values from LDS (16, with half of the threads idle: 62 us).
// 32 + 2 x 8 heads of 128, 8192 tokens: f32 in, bf16 pages 55 us (303 MB, 5.5 TB/s; 60
// without the loads ahead), bf16 in, 4-bit pages and copies 55 us (211 MB, 3.8 TB/s: v's
// bytes go out one by one, and 140 MB are written for 110); 56 tokens 4.7 us, of which 3.9 on
// the device.
#include "common.h"
#include "paged.h"

namespace {

constexpr uint32_t kThreads = 256;

// Where a token goes: page and place, or nowhere
struct Place {
  uint32_t page, place, pos;
  bool there;
};
CATENA_DEV Place place_of(const RopePackedArgs& a, uint32_t num_pages, uint32_t shift, uint32_t token) {
  const uint32_t pos = a.pos[token];
  const uint64_t slot = a.slots ? a.slots[token] : ~0ull, page = slot >> shift;
  const bool known = pos < a.positions;
  return Place{(uint32_t)page, (uint32_t)slot & ((1u << shift) - 1u), known ? pos : 0u, known && page < num_pages};
}

// Eight values as they lie, and as floats
template <bool WIDE>
struct Eight {
  u32x4_t w[WIDE ? 2 : 1];
};
template <bool WIDE>
CATENA_DEV Eight<WIDE> load8(const void* base, uint64_t at) {
  Eight<WIDE> r;
  const u32x4_t* p = WIDE ? reinterpret_cast<const u32x4_t*>(static_cast<const float*>(base) + at)
                          : reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(base) + at);
  r.w[0] = p[0];
  if constexpr (WIDE) r.w[1] = p[1];
  return r;
}
template <bool WIDE>
CATENA_DEV void floats8(const Eight<WIDE>& r, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (WIDE) {
      x[i] = __uint_as_float(r.w[0][i]);
      x[4 + i] = __uint_as_float(r.w[1][i]);
    } else {
      x[2 * i] = bf16lo(r.w[0][i]);
      x[2 * i + 1] = bf16hi(r.w[0][i]);
    }
  }
}
CATENA_DEV u32x4_t pack8(const float* y) {
  return u32x4_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])};
}

// A thread's 16 values of a head: eight from `first`, eight from `second`
template <bool WIDE>
struct Taken {
  Eight<WIDE> lo, hi;
};
struct Sixteen {
  uint32_t first, second;
  u32x4_t lo, hi;  // rounded
};
// unit: which 16 of the head's D; turns: the head is one of q or k
CATENA_DEV Sixteen places_of(const RopePackedArgs& a, uint32_t unit, bool turns) {
  Sixteen r;
  const bool apart = turns && 16 * unit < a.rot && !a.interleaved;
  r.first = apart ? 8 * unit : 16 * unit;
  r.second = apart ? 8 * unit + a.rot / 2 : 16 * unit + 8;
  return r;
}
template <bool WIDE>
CATENA_DEV Taken<WIDE> take(const RopePackedArgs& a, uint64_t head_at, uint32_t unit, bool turns) {
  const Sixteen r = places_of(a, unit, turns);
  return Taken<WIDE>{load8<WIDE>(a.qkv, head_at + r.first), load8<WIDE>(a.qkv, head_at + r.second)};
}
template <bool WIDE>
CATENA_DEV Sixteen turned(const RopePackedArgs& a, const Taken<WIDE>& t, uint32_t unit, bool turns, uint32_t pos) {
  Sixteen r = places_of(a, unit, turns);
  const bool pairs = turns && 16 * unit < a.rot, apart = pairs && !a.interleaved;
  float x[16], y[16];
  floats8<WIDE>(t.lo, x);
  floats8<WIDE>(t.hi, x + 8);
  if (pairs) {
    const f32x4_t* cs = reinterpret_cast<const f32x4_t*>(a.tab + ((uint64_t)pos * (a.rot / 2) + 8 * unit) * 2);
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4_t w = cs[i];
      c[2 * i] = w[0];
      s[2 * i] = w[1];
      c[2 * i + 1] = w[2];
      s[2 * i + 1] = w[3];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x1 = apart ? x[i] : x[2 * i], x2 = apart ? x[8 + i] : x[2 * i + 1];
      const float t1 = x1 * c[i], t2 = x2 * s[i], t3 = x2 * c[i], t4 = x1 * s[i];
      const float y1 = t1 - t2, y2 = t3 + t4;
      y[i] = y1;
      y[8 + i] = y2;
    }
    if (!apart) {
      float z[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        z[2 * i] = y[i];
        z[2 * i + 1] = y[8 + i];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = z[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[i];
  }
  r.lo = pack8(y);
  r.hi = pack8(y + 8);
  return r;
}
CATENA_DEV void store16(uint16_t* head, const Sixteen& x) {
  *reinterpret_cast<u32x4_t*>(head + x.first) = x.lo;
  *reinterpret_cast<u32x4_t*>(head + x.second) = x.hi;
}

// Every 16 values of a token's heads to a thread in turn: each(head, the token's place, they).  A turn's values are
// asked for before the token's position, or the last turn, is worked on.
template <bool WIDE, class KV, class Each>
CATENA_DEV Place each_unit(const RopePackedArgs& a, const KV& kv, uint32_t token, uint32_t all, const Each& each) {
  const uint32_t D = kv.head_dim, units = D / 16, most = all * units;
  auto ask = [&](uint32_t id) {
    const uint32_t head = id / units;
    return take<WIDE>(a, ((uint64_t)token * all + head) * D, id % units, head < a.heads + kv.kv_heads);
  };
  uint32_t id = threadIdx.x;
  Taken<WIDE> next;
  if (id < most) next = ask(id);
  const Place at = place_of(a, kv.num_pages, kv.page_shift, token);
  while (id < most) {
    const Taken<WIDE> now = next;
    const uint32_t head = id / units, unit = id % units;
    id += kThreads;
    if (id < most) next = ask(id);
    each(head, at, turned<WIDE>(a, now, unit, head < a.heads + kv.kv_heads, at.pos));
  }
  return at;
}

// grid = tokens
template <bool WIDE>
CATENA_DEV void rope_packed(const PagedKv& kv, const RopePackedArgs& a) {
  const uint32_t token = blockIdx.x, D = kv.head_dim, all = a.heads + 2 * kv.kv_heads;
  each_unit<WIDE>(a, kv, token, all, [&](uint32_t head, const Place& at, const Sixteen& x) {
    const bool is_k = head < a.heads + kv.kv_heads;
    if (head < a.heads) {
      store16(a.q + ((uint64_t)token * a.heads + head) * D, x);
      return;
    }
    const uint32_t h = (head - a.heads) % kv.kv_heads;
    if (a.k_out) store16((is_k ? a.k_out : a.v_out) + ((uint64_t)token * kv.kv_heads + h) * D, x);
    if (at.there) store16((is_k ? kv.k : kv.v) + paged_offset(kv, at.page, h, at.place), x);
  });
}

CATENA_DEV uint32_t larger(uint32_t x, uint32_t y) { return x > y ? x : y; }

// Eight bf16 values over `by` and the power of two `unit` as codes
CATENA_DEV uint32_t codes8(const u32x4_t& x, float by, float unit) {
  uint32_t w = 0;
#define CATENA_CODES(j) w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, bf16lo(x[j]) / by, bf16hi(x[j]) / by, unit, j);
  CATENA_CODES(0)
  CATENA_CODES(1)
  CATENA_CODES(2)
  CATENA_CODES(3)
#undef CATENA_CODES
  return w;
}
// The values of four codes' pairs, times unit, rounded to bf16
CATENA_DEV u32x4_t values8(uint32_t code, float unit) {
  u32x4_t r;
#define CATENA_VALUES(j)                                                                             \
  {                                                                                                  \
    typedef float f32x2 __attribute__((ext_vector_type(2)));                                         \
    const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, j);                         \
    r[j] = pack_bf16x2(v[0] * unit, v[1] * unit);                                                    \
  }
  CATENA_VALUES(0)
  CATENA_VALUES(1)
  CATENA_VALUES(2)
  CATENA_VALUES(3)
#undef CATENA_VALUES
  return r;
}
// The largest |x| of eight bf16 values, as bits (an infinity or NaN is above all others)
CATENA_DEV uint32_t top8(const u32x4_t& x) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = larger(top, larger(x[i] << 16 & 0x7FFF0000u, x[i] & 0x7FFF0000u));
  return top;
}

// grid = tokens; LDS: the token's keys and values in bf16
template <bool WIDE>
CATENA_DEV void rope_packed_q4(const PagedKv4& kv, const RopePackedArgs& a) {
  extern __shared__ __attribute__((aligned(16))) uint16_t s_kv[];
  const uint32_t token = blockIdx.x, D = kv.head_dim, all = a.heads + 2 * kv.kv_heads;
  const Place at = each_unit<WIDE>(a, kv, token, all, [&](uint32_t head, const Place&, const Sixteen& x) {
    store16(head < a.heads ? a.q + ((uint64_t)token * a.heads + head) * D : s_kv + (uint64_t)(head - a.heads) * D, x);
  });
  __syncthreads();
  const uint32_t page = 1u << kv.page_shift;
  // Eight values to a thread; whole waves: a head's threads are neighbours in one
  const uint32_t units = D / 8, items = 2 * kv.kv_heads * units;
  for (uint32_t id = threadIdx.x; id < (items + 63) / 64 * 64; id += kThreads) {
    const bool in = id < items;
    const uint32_t vec = in ? id / units : 0u, unit = id % units, h = vec % kv.kv_heads;
    const bool is_k = vec < kv.kv_heads;
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(s_kv + (uint64_t)vec * D + 8 * unit);
    uint32_t top = top8(x);
    top = larger(top, (uint32_t)__shfl_xor((int)top, 1));
    top = larger(top, (uint32_t)__shfl_xor((int)top, 2));
    if (!is_k)
      for (uint32_t step = 4; step < units; step *= 2) top = larger(top, (uint32_t)__shfl_xor((int)top, (int)step));
    const bool odd = top >= 0x7F800000u;  // an infinity or NaN
    float scale;
    uint32_t byte = 0;
    if (is_k) {
      // top = m 2^e, 1 <= m < 2: 2^(e - 2), or 2^(e - 1) where m > 1.5 (a subnormal top, e below 2^-126, gets the least)
      const uint32_t e = top >> 23, up = (top & 0x7FFFFFu) > 0x400000u;
      byte = odd ? 255u : e + up > 2 ? e + up - 2 : 0u;
      scale = __uint_as_float(byte ? byte << 23 : 0x00400000u);
    } else {
      const float s = __uint_as_float(top) / 6.0f;
      scale = __uint_as_float(odd ? 0x7FC00000u : (__float_as_uint(s) + 0xFFFFu) & 0xFFFF0000u);
    }
    const uint32_t some = 0u - (uint32_t)(!odd & (scale > 0.0f));
    const uint32_t code = codes8(x, is_k ? 1.0f : scale, is_k ? scale : 1.0f) & some;
    if (!in) continue;
    if (a.k_out) {
      uint16_t* out = (is_k ? a.k_out : a.v_out) + ((uint64_t)token * kv.kv_heads + h) * D + 8 * unit;
      *reinterpret_cast<u32x4_t*>(out) = values8(code, odd ? __uint_as_float(0x7FC00000u) : scale);
    }
    if (!at.there) continue;
    const uint64_t cells = paged_cells(kv.kv_heads, kv.page_shift, at.page, h);
    if (is_k) {
      *reinterpret_cast<uint32_t*>(kv.k + (cells + at.place) * (D / 2) + 4 * unit) = code;
      if (unit % 4 == 0) kv.k_scale[cells * (D / 32) + (unit / 4) * page + at.place] = (uint8_t)byte;
    } else {
      uint8_t* dst = kv.v + cells * (D / 2) + (uint64_t)(4 * unit) * page + at.place;
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i * page] = (uint8_t)(code >> (8 * i));
      if (unit == 0) kv.v_scale[cells + at.place] = (uint16_t)(__float_as_uint(scale) >> 16);
    }
  }
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void catena_rope_packed_f32in(PagedKv kv, RopePackedArgs a) {
  rope_packed<true>(kv, a);
}
extern "C" __global__ __launch_bounds__(256) void catena_rope_packed_bf16in(PagedKv kv, RopePackedArgs a) {
  rope_packed<false>(kv, a);
}
extern "C" __global__ __launch_bounds__(256) void catena_rope_packed_q4_f32in(PagedKv4 kv, RopePackedArgs a) {
  rope_packed_q4<true>(kv, a);
}
extern "C" __global__ __launch_bounds__(256) void catena_rope_packed_q4_bf16in(PagedKv4 kv, RopePackedArgs a) {
  rope_packed_q4<false>(kv, a);
}

// tab[i - first][j] = (cos, sin) of i * inv_freq[j], times mscale, for positions first ..
// first + n - 1: the angle and its sine in 64 bits, so that far positions lose nothing.
extern "C" __global__ __launch_bounds__(256) void catena_rope_table_f64(const double* __restrict__ inv_freq,
                                                                        float* __restrict__ tab, uint32_t first,
                                                                        uint32_t n, uint32_t half, double mscale) {
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (uint64_t)n * half) return;
  const uint32_t i = (uint32_t)(id / half), j = (uint32_t)(id % half);
  double s, c;
  sincos(((double)first + (double)i) * inv_freq[j], &s, &c);
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  reinterpret_cast<f32x2*>(tab)[id] = f32x2{(float)(c * mscale), (float)(s * mscale)};
}
