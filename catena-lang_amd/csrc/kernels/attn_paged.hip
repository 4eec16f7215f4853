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
// softmax beside the running o.  The slots of a row are cut into `splits` runs,
// one workgroup each, and joined by a second kernel; a run's bounds follow from
// the row's own length, so a short row of a long table is spread as wide.
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
// have time for that (one slot's 32 x D x 16 flop against 4 D bytes).
//
// Rounding: scores and sums in f32.  p goes into the product as bf16 terms,
// each the upper half of what the one before left over: three (all 24 bits) for
// an f32 output, two (2^-16 relative) for a bf16 one; the further products hide
// under the cache's stream.  A term that would be 0 is 2^-126 instead, so that
// an infinity in V gives infinity and not 0 * infinity.
//
// The maximum is raised only where a score passes it by more than 8 in base 2,
// for all lanes of a head at once: until then p stays below 2^8, which costs no
// accuracy, and most tiles need no exchange between lanes.
#include "common.h"
#include "paged.h"

namespace {

constexpr float kNegInf = -__builtin_huge_valf();

// The slots [beg, end) of split s, in whole tiles of 32
struct Run {
  uint32_t beg, end;  // tiles
};
CATENA_DEV Run run_of(uint32_t len, uint32_t splits, uint32_t s) {
  const uint32_t tiles = (len + 31) / 32;
  const uint32_t per = ((tiles + splits - 1) / splits + 3) & ~3u;  // every wave of a run has as many
  const uint32_t beg = s * per;
  return Run{beg < tiles ? beg : tiles, beg + per < tiles ? beg + per : tiles};
}
CATENA_DEV uint32_t runs_of(uint32_t len, uint32_t splits) {
  const uint32_t tiles = (len + 31) / 32;
  const uint32_t per = ((tiles + splits - 1) / splits + 3) & ~3u;
  return per == 0 ? 0 : (tiles + per - 1) / per;
}

CATENA_DEV float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// the reference point of exponents: 0 while no score is above -inf
CATENA_DEV float anchor(float m) { return m == kNegInf ? 0.0f : m; }


struct AttnPagedArgs {
  PagedKv kv;
  const uint16_t* q;      // [rows][heads][D]
  const uint32_t* lens;   // [rows]
  void* o;                // [rows][heads][D], written here where splits == 1
  float* part_o;          // [rows][kv_heads][splits][group][D]
  float* part_ml;         // [rows][kv_heads][splits][group][2]: maximum (base 2), sum
  float* scores;          // [rows][heads][slots] base-2 scores, with weights only
  const float* acc_in;    // [rows][kv_heads][slots]
  float* acc_out;
  uint32_t group, head_tiles, splits;
  float scale_log2;       // scale * log2(e)
};

template <int D, bool F32, bool WEIGHTS>
CATENA_DEV void attn_paged_run(const AttnPagedArgs& a) {
  constexpr int KC = D / 32;  // K loads of 8 values, products of S
  constexpr int VC = D / 16;  // columns of V a lane takes
  const uint32_t lane = threadIdx.x & 63u, c = lane & 15u, g = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = blockIdx.x, split = blockIdx.y;
  const uint32_t ht = unit % a.head_tiles, pair = unit / a.head_tiles;  // pair: (row, kv head)
  const uint32_t row = pair / a.kv.kv_heads, kvh = pair % a.kv.kv_heads;
  const uint32_t heads = a.group * a.kv.kv_heads;
  const uint32_t gn = a.group - 16 * ht < 16 ? a.group - 16 * ht : 16;
  const uint32_t slots = paged_slots(a.kv);
  const uint32_t len = paged_len(a.kv, a.lens[row]);
  const Run run = run_of(len, a.splits, split);
  if (a.splits > 1 && run.beg >= run.end) return;  // the join knows how many runs a length has

  // Q as the B operand: lane = head c, 8 values of each 32-wide block of d
  bf16x8_t qf[KC];
  {
    const uint16_t* q = a.q + ((uint64_t)row * heads + kvh * a.group + 16 * ht + (c < gn ? c : 0)) * D;
#pragma unroll
    for (int i = 0; i < KC; ++i) {
      u32x4_t w = *reinterpret_cast<const u32x4_t*>(q + 32 * i + 8 * g);
      if (c >= gn) w = u32x4_t{0, 0, 0, 0};
      qf[i] = __builtin_bit_cast(bf16x8_t, w);
    }
  }

  float m = kNegInf, l = 0.0f;
  f32x4_t acc[VC];
#pragma unroll
  for (int e = 0; e < VC; ++e) acc[e] = f32x4_t{0, 0, 0, 0};

  const uint32_t* table = a.kv.table + (uint64_t)row * a.kv.max_pages;
  const uint32_t mask = (1u << a.kv.page_shift) - 1u;
  for (uint32_t t = run.beg + wave; t < run.end; t += 4) {
    // two runs of 16 slots: where they live and how many count
    uint64_t at[2];
    uint32_t n[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t slot = 32 * t + 16 * u;
      uint32_t page = slot < len ? table[slot >> a.kv.page_shift] : 0u;
      const bool here = slot < len && page < a.kv.num_pages;
      n[u] = !here ? 0u : len - slot < 16 ? len - slot : 16u;
      if (!here) page = 0;  // read and left out
      at[u] = paged_offset(a.kv, page, kvh, slot & mask);
    }
    // K and V of the tile
    u32x4_t kr[2][KC];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < KC; ++i)
        kr[u][i] = *reinterpret_cast<const u32x4_t*>(a.kv.k + at[u] + c * D + 32 * i + 8 * g);
    uint32_t vr[8][VC / 2];  // slot (j < 4: 4 g + j of the first run, else of the second), columns VC c ..
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint16_t* p = a.kv.v + at[j / 4] + (4 * g + j % 4) * D + VC * c;
      if constexpr (VC == 8) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
        for (int x = 0; x < 4; ++x) vr[j][x] = w[x];
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        vr[j][0] = w.x;
        vr[j][1] = w.y;
      }
    }
    // scores in base 2: s[j] is slot (g, j) of head c
    float s[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      f32x4_t x = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KC; ++i)
        x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kr[u][i]), qf[i], x, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[4 * u + j] = x[j] * a.scale_log2;
    }
    if (n[0] < 16 || n[1] < 16) {
      // what the tile holds past the row's end (or of a page that is not there)
      // may be anything: no score, and zeros in V's place
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = 4 * g + j % 4 < n[j / 4];
        s[j] = in ? s[j] : kNegInf;
#pragma unroll
        for (int x = 0; x < VC / 2; ++x) vr[j][x] = in ? vr[j][x] : 0u;
      }
    }
    if constexpr (WEIGHTS) {
      if (c < gn) {
        float* dst = a.scores + ((uint64_t)row * heads + kvh * a.group + 16 * ht + c) * slots + 32 * t + 4 * g;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (32 * t + 16 * u < len)
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
    }
    // p's bf16 terms
    constexpr int TERMS = F32 ? 3 : 2;
    bf16x8_t pt[TERMS];
#pragma unroll
    for (int x = 0; x < TERMS; ++x) {
      u32x4_t w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (x + 1 < TERMS) {
          const uint32_t b0 = __float_as_uint(p[2 * j]), b1 = __float_as_uint(p[2 * j + 1]);
          w[j] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
          p[2 * j] = __builtin_fmaxf(p[2 * j] - __uint_as_float(b0 & 0xFFFF0000u), 0x1p-126f);
          p[2 * j + 1] = __builtin_fmaxf(p[2 * j + 1] - __uint_as_float(b1 & 0xFFFF0000u), 0x1p-126f);
        } else {
          w[j] = pack_bf16x2(p[2 * j], p[2 * j + 1]);
        }
      }
      pt[x] = __builtin_bit_cast(bf16x8_t, w);
    }
#pragma unroll
    for (int e = 0; e < VC; ++e) {
      // column e of the lane's 8 x VC block
      u32x4_t col;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        col[j] = __builtin_amdgcn_perm(vr[2 * j + 1][e / 2], vr[2 * j][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
      const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, col);
#pragma unroll
      for (int x = 0; x < TERMS; ++x)
        acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pt[x], acc[e], 0, 0, 0);
    }
  }

  // The four waves' (m, l, o) to one
  l = l + __shfl_xor(l, 16);
  l = l + __shfl_xor(l, 32);
  constexpr int OS = D + 4;  // keeps the lanes of a 16-byte store off each other's banks
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ __attribute__((aligned(16))) float s_o[4][16][OS];
  if (g == 0) {
    s_m[wave][c] = m;
    s_l[wave][c] = l;
  }
  if (c < gn) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < VC; e += 4)
        *reinterpret_cast<f32x4_t*>(&s_o[wave][c][4 * VC * g + VC * i + e]) =
            f32x4_t{acc[e][i], acc[e + 1][i], acc[e + 2][i], acc[e + 3][i]};
  }
  __syncthreads();
  for (uint32_t id = threadIdx.x; id < gn * (D / 4); id += 256) {
    const uint32_t h = id / (D / 4), d = id % (D / 4) * 4;
    float mm = kNegInf;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = __builtin_fmaxf(mm, s_m[w][h]);
    float ll = 0.0f;
    f32x4_t o = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2_fast(s_m[w][h] - anchor(mm));
      ll = ll + s_l[w][h] * f;
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(&s_o[w][h][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = o[i] + x[i] * f;
    }
    const uint32_t head = 16 * ht + h;
    if (a.splits > 1 || WEIGHTS) {
      const uint64_t at = ((uint64_t)pair * a.splits + split) * a.group + head;
      if (d == 0) {
        a.part_ml[2 * at] = mm;
        a.part_ml[2 * at + 1] = ll;
      }
      if (a.splits > 1) {
        *reinterpret_cast<f32x4_t*>(a.part_o + at * D + d) = o;
        continue;
      }
    }
    const uint64_t at = ((uint64_t)row * heads + kvh * a.group + head) * D + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = len ? o[i] / ll : 0.0f;
    if constexpr (F32) {
      *reinterpret_cast<f32x4_t*>(static_cast<float*>(a.o) + at) = o;
    } else {
      uint2 w;
      w.x = pack_bf16x2(o[0], o[1]);
      w.y = pack_bf16x2(o[2], o[3]);
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + at) = w;
    }
  }
}

// Joins the runs of a row and adds the weights.  grid.x = (row, kv head);
// blockIdx.y < join_blocks: four query heads' o, else 1024 slots' weights.
template <int D, bool F32>
CATENA_DEV void attn_paged_join(const AttnPagedArgs& a, uint32_t join_blocks) {
  const uint32_t pair = blockIdx.x, row = pair / a.kv.kv_heads, kvh = pair % a.kv.kv_heads;
  const uint32_t len = paged_len(a.kv, a.lens[row]);
  const uint32_t runs = runs_of(len, a.splits);
  const uint32_t heads = a.group * a.kv.kv_heads, slots = paged_slots(a.kv);
  const float* ml = a.part_ml + 2 * (uint64_t)pair * a.splits * a.group;
  if (blockIdx.y < join_blocks) {
    const uint32_t head = blockIdx.y * 4 + threadIdx.x / 64, lane = threadIdx.x & 63u;
    if (head >= a.group) return;
    const float* po = a.part_o + ((uint64_t)pair * a.splits * a.group + head) * D;
    constexpr int PER = D / 64;
    float mm = kNegInf;
    for (uint32_t s = 0; s < runs; ++s) mm = __builtin_fmaxf(mm, ml[2 * ((uint64_t)s * a.group + head)]);
    float ll = 0.0f, o[PER] = {};
    for (uint32_t s = 0; s < runs; ++s) {
      const uint64_t at = (uint64_t)s * a.group + head;
      const float f = exp2_fast(ml[2 * at] - anchor(mm));
      ll = ll + ml[2 * at + 1] * f;
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] = o[i] + po[(uint64_t)s * a.group * D + PER * lane + i] * f;
    }
    const uint64_t at = ((uint64_t)row * heads + kvh * a.group + head) * D + PER * lane;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float x = len ? o[i] / ll : 0.0f;
      if constexpr (F32)
        static_cast<float*>(a.o)[at + i] = x;
      else
        static_cast<uint16_t*>(a.o)[at + i] = (uint16_t)f32_to_bf16_bits(x);
    }
    return;
  }
  const uint32_t slot0 = (blockIdx.y - join_blocks) * 1024;
  if (slot0 >= len) return;
  __shared__ float s_m[256], s_r[256];  // of up to 256 heads of the group at a time
  f32x4_t w = f32x4_t{0, 0, 0, 0};
  const uint32_t slot = slot0 + 4 * threadIdx.x;  // slots come in whole pages of 16 or more
  for (uint32_t h0 = 0; h0 < a.group; h0 += 256) {
    const uint32_t hn = a.group - h0 < 256 ? a.group - h0 : 256;
    if (h0) __syncthreads();
    if (threadIdx.x < hn) {
      const uint32_t head = h0 + threadIdx.x;
      float mm = kNegInf;
      for (uint32_t s = 0; s < runs; ++s) mm = __builtin_fmaxf(mm, ml[2 * ((uint64_t)s * a.group + head)]);
      float ll = 0.0f;
      for (uint32_t s = 0; s < runs; ++s) {
        const uint64_t at = (uint64_t)s * a.group + head;
        ll = ll + ml[2 * at + 1] * exp2_fast(ml[2 * at] - anchor(mm));
      }
      s_m[threadIdx.x] = anchor(mm);
      s_r[threadIdx.x] = 1.0f / ll;
    }
    __syncthreads();
    if (slot < len) {
      const float* sc = a.scores + ((uint64_t)row * heads + kvh * a.group + h0) * slots + slot;
      for (uint32_t h = 0; h < hn; ++h) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(sc + (uint64_t)h * slots);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = w[i] + exp2_fast(x[i] - s_m[h]) * s_r[h];
      }
    }
  }
  if (slot >= len) return;
  const uint64_t at = (uint64_t)pair * slots + slot;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (slot + i < len) a.acc_out[at + i] = a.acc_in[at + i] + w[i];
}

}  // namespace

#define CATENA_ATTN_PAGED(D, OUT, F32)                                                                  \
  extern "C" __global__ __launch_bounds__(256) void catena_attn_paged_d##D##_##OUT(AttnPagedArgs a) {         \
    attn_paged_run<D, F32, false>(a);                                                                         \
  }                                                                                                           \
  extern "C" __global__ __launch_bounds__(256) void catena_attn_paged_weights_d##D##_##OUT(AttnPagedArgs a) { \
    attn_paged_run<D, F32, true>(a);                                                                          \
  }                                                                                                           \
  extern "C" __global__ __launch_bounds__(256) void catena_attn_paged_join_d##D##_##OUT(AttnPagedArgs a,      \
                                                                                        uint32_t join_blocks) { \
    attn_paged_join<D, F32>(a, join_blocks);                                                                  \
  }
CATENA_ATTN_PAGED(128, f32out, true)
CATENA_ATTN_PAGED(128, bf16out, false)
CATENA_ATTN_PAGED(64, f32out, true)
CATENA_ATTN_PAGED(64, bf16out, false)
