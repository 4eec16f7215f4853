// Upkeep of a key-value cache in pages: new rows in, the least weighted rows
// out, pages of one row to another.
#include "common.h"
#include "paged.h"

// ------------------------------------------------------------------ append
//
// qkv[rows * tq][(heads + 2 kv_heads) * D] f32 (columns: q heads | k heads |
// v heads).  Token t of a row goes to slot lens[row] - tq + t at position
// (seen ? seen[row] : lens[row]) - tq + t; pairs (i, i + D/2) of q and k turn
// by (cos, sin) = tab[position][i]:
//   y1 = x1 c - x2 s, y2 = x2 c + x1 s  (each operation rounded)
// q to q_out[rows * tq][heads * D], k and v to the slot's page, all bf16 RNE; a
// tracked cache's weight of the slot starts at 0 and its position is noted.
// A token whose slot or position does not exist, or whose row has fewer of either than
// tq, writes q turned by tab[0] and nothing else; one whose page does not exist writes
// q alone.
//
// Bound: HBM for prompts (4 bytes in, 2 out per value), one launch's latency for
// a decode step.  A thread takes four pairs (two 16-byte loads of x, two of the
// table, two 8-byte stores); a workgroup serves one token, so the page and
// the position are looked up once, by scalar loads.  8 prompts of 500 tokens, 16
// heads of 128: 28.8 us, 5.1 TB/s; one token each 2.9 us.
// grid = (rows * tq, ceil((heads + 2 kv_heads) * D / 8 / 256)).
extern "C" __global__ __launch_bounds__(256) void catena_rope_qkv_paged(
    PagedKv kv, const float* __restrict__ qkv, const float* __restrict__ tab, uint32_t positions,
    const uint32_t* __restrict__ lens, const uint32_t* __restrict__ seen, uint16_t* __restrict__ q_out,
    uint32_t tq, uint32_t heads, float* __restrict__ acc, uint32_t* __restrict__ slot_pos) {
  const uint32_t D = kv.head_dim, quads = D / 8;
  const uint32_t token = blockIdx.x, row = token / tq, t = token % tq;
  const uint32_t id = blockIdx.y * 256 + threadIdx.x;
  const uint32_t head = id / quads, i = id % quads * 4;
  const uint32_t all = heads + 2 * kv.kv_heads;
  if (head >= all) return;
  const uint32_t len = lens[row], count = seen ? seen[row] : len;
  const uint32_t slot = len - tq + t, pos = count - tq + t;
  const bool known = len >= tq && slot < paged_slots(kv) && count >= tq && pos < positions;
  const float* src = qkv + ((uint64_t)token * all + head) * D;
  const f32x4_t x1 = *reinterpret_cast<const f32x4_t*>(src + i);
  const f32x4_t x2 = *reinterpret_cast<const f32x4_t*>(src + D / 2 + i);
  f32x4_t y1 = x1, y2 = x2;
  if (head < heads + kv.kv_heads) {
    const float* cs = tab + ((uint64_t)(known ? pos : 0u) * (D / 2) + i) * 2;
    const f32x4_t a = *reinterpret_cast<const f32x4_t*>(cs), b = *reinterpret_cast<const f32x4_t*>(cs + 4);
    const float c[4] = {a[0], a[2], b[0], b[2]}, s[4] = {a[1], a[3], b[1], b[3]};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float t1 = x1[j] * c[j], t2 = x2[j] * s[j], t3 = x2[j] * c[j], t4 = x1[j] * s[j];
      y1[j] = t1 - t2;
      y2[j] = t3 + t4;
    }
  }
  uint16_t* dst;
  if (head < heads) {
    dst = q_out + ((uint64_t)token * heads + head) * D;
  } else {
    const uint32_t h = (head - heads) % kv.kv_heads;
    uint64_t at;
    if (!known || !paged_place(kv, row, h, slot, &at)) return;
    const bool is_k = head < heads + kv.kv_heads;
    dst = (is_k ? kv.k : kv.v) + at;
    if (is_k && i == 0 && acc) {
      const uint64_t place = ((uint64_t)row * kv.kv_heads + h) * paged_slots(kv) + slot;
      acc[place] = 0.0f;
      slot_pos[place] = pos;
    }
  }
  uint2 w;
  w.x = pack_bf16x2(y1[0], y1[1]);
  w.y = pack_bf16x2(y1[2], y1[3]);
  *reinterpret_cast<uint2*>(dst + i) = w;
  w.x = pack_bf16x2(y2[0], y2[1]);
  w.y = pack_bf16x2(y2[2], y2[3]);
  *reinterpret_cast<uint2*>(dst + D / 2 + i) = w;
}

// ------------------------------------------------------------------ eviction
//
// Keeps min(n, budget) of a row's n slots, per kv head: those of the last
// `recent` positions, then those of the largest accumulated weight, the lower
// slot where two are equal; a NaN weight goes first.  Where more slots than the
// budget are recent, the newest are kept.  The i-th slot given up
// below the budget takes the i-th kept slot from the budget on, so that the
// kept slots are the first ones: attention does not depend on the slots' order,
// and only as many rows move as were given up there.

namespace {

// Larger is kept: the whole order of the rule above but for the slot's number.
CATENA_DEV uint32_t keep_key(float weight, uint32_t pos, uint32_t late) {
  if (pos >= late) return 0xFFFFFFFFu;
  return weight != weight ? 0u : mono_bits(__float_as_uint(weight));
}

// The same where the recent slots alone are more than the budget
CATENA_DEV uint32_t newest_key(uint32_t pos, uint32_t late) {
  const uint32_t after = pos - late;
  return pos < late ? 0u : after < 0xFFFFFFFFu ? after + 1 : after;
}

// Exclusive prefix sum over the workgroup's threads, and the total.  s_wave[2]:
// the caller alternates between the two, so that one barrier is enough.
template <int WAVES>
CATENA_DEV uint32_t block_prefix(uint32_t x, uint32_t* s_wave, uint32_t* total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t in = wave_prefix(x);
  if (lane == 63) s_wave[wave] = in;
  __syncthreads();
  const uint32_t sums = wave_prefix(lane < WAVES ? s_wave[lane] : 0u);
  const uint32_t w = __builtin_amdgcn_readfirstlane(wave);
  *total = (uint32_t)__builtin_amdgcn_readlane((int)sums, WAVES - 1);
  const uint32_t before = w ? (uint32_t)__builtin_amdgcn_readlane((int)sums, (int)w - 1) : 0u;
  return before + in - x;
}

// Moves first, first + step, ... of a (row, kv head), four at a time: a row of K and
// of V (16 bytes a lane), the slot's weight and position.  Sources lie from the
// budget on and are never written, so the order does not matter.
CATENA_DEV void evict_moves(const EvictArgs& a, uint32_t pair, const uint32_t* holes, const uint32_t* sources,
                            uint32_t first, uint32_t end, uint32_t step) {
  constexpr int AT = 4;
  const uint32_t row = pair / a.kv.kv_heads, h = pair % a.kv.kv_heads;
  const uint32_t lane = threadIdx.x % (a.kv.head_dim / 8);
  const uint64_t base = (uint64_t)pair * paged_slots(a.kv);
  for (uint32_t i = first; i < end; i += AT * step) {
    uint32_t to[AT], from[AT];
    uint64_t dst[AT], src[AT];
    bool there[AT];
    u32x4_t k[AT], v[AT];
#pragma unroll
    for (int j = 0; j < AT; ++j) {
      const bool in = i + j * step < end;
      to[j] = in ? holes[i + j * step] : 0xFFFFFFFFu;
      from[j] = in ? sources[i + j * step] : 0xFFFFFFFFu;
    }
#pragma unroll
    for (int j = 0; j < AT; ++j)
      there[j] = paged_place(a.kv, row, h, to[j], &dst[j]) && paged_place(a.kv, row, h, from[j], &src[j]);
#pragma unroll
    for (int j = 0; j < AT; ++j)
      if (there[j]) {
        k[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(a.kv.k + src[j] + 8 * lane));
        v[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(a.kv.v + src[j] + 8 * lane));
      }
#pragma unroll
    for (int j = 0; j < AT; ++j) {
      if (there[j]) {
        *reinterpret_cast<u32x4_t*>(a.kv.k + dst[j] + 8 * lane) = k[j];
        *reinterpret_cast<u32x4_t*>(a.kv.v + dst[j] + 8 * lane) = v[j];
      }
      if (lane == 0 && to[j] != 0xFFFFFFFFu) {
        a.acc_out[base + to[j]] = a.acc_in[base + from[j]];
        a.pos_out[base + to[j]] = a.pos_in[base + from[j]];
      }
    }
  }
}

// What a (row, kv head) keeps: the lists of slots to fill and of slots to fill
// them from, and the weights and positions of the slots that stay in place.  A
// thread has KEYS slots in a row of every THREADS * KEYS; a row that is no longer
// stays in registers, a longer one is read again for each pass.  The budget-th
// largest key is found digit by digit from the top, a histogram in LDS each, until
// a digit's keys are all kept; prefix sums over the threads then order both lists.
// Bound: latency (two dependent loads, a dozen barriers), so short rows take a
// small workgroup: 32 x 8 rows of 5120 slots, 4096 kept, 12.6 us; 8 x 16 of 513 slots,
// 512 kept, 4.0 with the move.
// MANY: recent > budget.  Positions differ, so that only then more slots than the budget
// can be recent, which is counted first.
template <int THREADS, int KEYS, bool MANY>
CATENA_DEV void evict_choose(const EvictArgs& a) {
  constexpr int WAVES = THREADS / 64, DIGIT = THREADS == 256 ? 8 : 12, STEPS = THREADS == 256 ? 4 : 3;
  constexpr uint32_t BINS = 1u << DIGIT, OWN = BINS / THREADS, TILE = THREADS * KEYS;
  constexpr uint32_t LISTS = 128;
  __shared__ uint32_t hist[BINS];
  __shared__ uint32_t s_wave[2][WAVES], s_bin, s_left, s_in_bin, s_holes[LISTS], s_sources[LISTS];
  __shared__ uint64_t s_low[WAVES];
  const uint32_t pair = blockIdx.x, row = pair / a.kv.kv_heads, tid = threadIdx.x, budget = a.budget;
  const uint32_t slots = paged_slots(a.kv);
  const uint64_t base = (uint64_t)pair * slots;

  // the thread's slots of a tile up to `upto`; what is read behind the row's end
  // is table, in whole vectors, and its keys do not count
  f32x4_t w[KEYS / 4];
  u32x4_t p[KEYS / 4];
  uint32_t beg = 0;
  auto load = [&](uint32_t tile, uint32_t upto) {
    beg = tile * TILE + tid * KEYS;
#pragma unroll
    for (int i = 0; i < KEYS / 4; ++i) {
      const bool in = beg + 4 * i < upto;
      w[i] = in ? *reinterpret_cast<const f32x4_t*>(a.acc_in + base + beg + 4 * i) : f32x4_t{0, 0, 0, 0};
      p[i] = in ? *reinterpret_cast<const u32x4_t*>(a.pos_in + base + beg + 4 * i) : u32x4_t{0, 0, 0, 0};
    }
  };
  // a table of one tile is read before the row's length is known
  const bool single = slots <= TILE;
  if (single) load(0, slots);
  const uint32_t n = paged_len(a.kv, a.lens[row]), total_seen = a.seen[row], kept = n < budget ? n : budget;
  const uint32_t late = total_seen - (a.recent < total_seen ? a.recent : total_seen);
  const uint32_t tiles = (n + TILE - 1) / TILE;
  if (!single && tiles == 1) load(0, n);
  if (tid == 0 && pair % a.kv.kv_heads == 0) a.lens_out[row] = kept;
  // the tile's keys; 0, the last of all, behind the row's end
  uint32_t keys[KEYS];
  bool window = false;  // recent slots alone are kept
  auto rate = [&]() {
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const uint32_t pos = p[i / 4][i % 4];
      const uint32_t key = MANY && window ? newest_key(pos, late) : keep_key(w[i / 4][i % 4], pos, late);
      keys[i] = beg + i < n ? key : 0u;
    }
  };
  // the slots below the budget as they are; the moves overwrite those given up
  auto copy = [&]() {
#pragma unroll
    for (int i = 0; i < KEYS / 4; ++i) {
      const uint32_t j = beg + 4 * i;
      if (j + 4 <= kept) {
        if (a.acc_out != a.acc_in) *reinterpret_cast<f32x4_t*>(a.acc_out + base + j) = w[i];
        if (a.pos_out != a.pos_in) *reinterpret_cast<u32x4_t*>(a.pos_out + base + j) = p[i];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < kept) {
            if (a.acc_out != a.acc_in) a.acc_out[base + j + e] = w[i][e];
            if (a.pos_out != a.pos_in) a.pos_out[base + j + e] = p[i][e];
          }
      }
    }
  };
  if (n <= budget) {
    for (uint32_t tile = 0; tile < tiles; ++tile) {
      if (tiles > 1) load(tile, n);
      copy();
    }
    if (tid == 0 && !a.at_once) a.count[pair] = 0;
    return;
  }
  if constexpr (MANY) {
    uint32_t mine = 0, all;
#pragma unroll 1
    for (uint32_t tile = 0; tile < tiles; ++tile) {
      if (tiles > 1) load(tile, n);
#pragma unroll
      for (int i = 0; i < KEYS; ++i) mine += beg + i < n && p[i / 4][i % 4] >= late;
    }
    block_prefix<WAVES>(mine, s_wave[1], &all);
    window = all > budget;
  }
  if (tiles == 1) rate();

  // One slot too many, as behind every step of a full cache: the smallest key, the
  // higher slot of equal ones, is given up, and the last slot takes its place.
  if (n - budget == 1) {
    uint64_t low = ~0ull;
#pragma unroll 1
    for (uint32_t tile = 0; tile < tiles; ++tile) {
      if (tiles > 1) load(tile, n), rate();
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        const uint64_t x = ((uint64_t)keys[i] << 32) | ~(beg + i);
        if (beg + i < n) low = x < low ? x : low;
      }
      copy();
    }
    const uint32_t hi = ~wave_umax(~(uint32_t)(low >> 32));
    const uint32_t lo = ~wave_umax((uint32_t)(low >> 32) == hi ? ~(uint32_t)low : 0u);
    if (tid % 64 == 0) s_low[tid / 64] = ((uint64_t)hi << 32) | lo;
    __syncthreads();
    low = s_low[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) low = s_low[i] < low ? s_low[i] : low;
    const uint32_t to = ~(uint32_t)low;
    if (to < budget && tid < a.kv.head_dim / 8) evict_moves(a, pair, &to, &budget, 0, 1, 1);
    if (tid == 0 && !a.at_once) a.count[pair] = 0;
    return;
  }

  uint32_t prefix = 0, left = budget, shift = 32, total;
  bool ties = true;  // more keys in the prefix's range than are kept
#pragma unroll 1
  for (int step = 0; step < STEPS && ties; ++step) {
    const uint32_t known = step == 0 ? 0u : 0xFFFFFFFFu << shift;
    const uint32_t bits = shift < DIGIT ? shift : DIGIT, bins = 1u << bits;
    shift -= bits;
#pragma unroll
    for (uint32_t b = 0; b < OWN; ++b) hist[tid + b * THREADS] = 0;
    __syncthreads();
#pragma unroll 1
    for (uint32_t tile = 0; tile < tiles; ++tile) {
      if (tiles > 1) load(tile, n), rate();
      if (beg < n) {
#pragma unroll
        for (int i = 0; i < KEYS; ++i)
          if ((keys[i] & known) == prefix) atomicAdd(&hist[(keys[i] >> shift) & (bins - 1)], 1u);
      }
    }
    __syncthreads();
    // the thread's bins from the top: the keys above them, then bin by bin (a
    // digit of fewer bits leaves the upper bins empty)
    uint32_t own[OWN], mine = 0;
#pragma unroll
    for (uint32_t b = 0; b < OWN; ++b) {
      own[b] = hist[BINS - 1 - (tid * OWN + b)];
      mine += own[b];
    }
    uint32_t over = block_prefix<WAVES>(mine, s_wave[step & 1], &total);
    if (over < left && over + mine >= left) {
#pragma unroll
      for (uint32_t b = 0; b < OWN; ++b) {
        if (over < left && over + own[b] >= left) {
          s_bin = BINS - 1 - (tid * OWN + b);
          s_left = left - over;
          s_in_bin = own[b];
        }
        over += own[b];
      }
    }
    __syncthreads();
    prefix |= s_bin << shift;
    left = s_left;
    ties = s_in_bin != left;
  }

  // Kept: keys above the prefix's range, and in it all or, of that very key, the
  // first `left`.  Both lists in the order of slots; few moves stay in LDS for
  // this workgroup.
  // (What lies behind the row's end has the lowest key and the highest slots: it
  // is counted among equals, never kept.)
  const uint32_t range = 0xFFFFFFFFu << shift;
  const bool here = a.at_once != 0;
  uint32_t* holes = here ? s_holes : a.holes + (uint64_t)pair * a.most;
  uint32_t* sources = here ? s_sources : a.sources + (uint64_t)pair * a.most;
  uint32_t equal_before = 0, holes_before = 0, sources_before = 0;
#pragma unroll 1
  for (uint32_t tile = 0; tile < tiles; ++tile) {
    if (tiles > 1) load(tile, n), rate();
    uint32_t passed = 0;
    if (ties) {
      uint32_t equal = 0;
      if (beg < n) {
#pragma unroll
        for (int i = 0; i < KEYS; ++i) equal += (keys[i] & range) == prefix;
      }
      if (tile) __syncthreads();  // the last tile's sums have been read
      passed = equal_before + block_prefix<WAVES>(equal, s_wave[0], &total);
      equal_before += total;
    }
    uint32_t kept_bits = 0;  // a bit a slot
    if (beg < n) {
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        const uint32_t key = keys[i] & range;
        const bool same = key == prefix, keep = key > prefix || (same && (!ties || passed < left));
        passed += same;
        kept_bits |= keep ? 1u << i : 0u;
      }
    }
    // given up below the budget, kept from it on
    const uint32_t below = beg >= budget ? 0u : budget - beg >= KEYS ? (1u << KEYS) - 1u : (1u << (budget - beg)) - 1u;
    uint32_t given = ~kept_bits & below, taken = kept_bits & ~below;
    if (tile) __syncthreads();
    // a tile's counts fit 16 bits each
    const uint32_t before =
        block_prefix<WAVES>(((uint32_t)__popc(taken) << 16) | (uint32_t)__popc(given), s_wave[1], &total);
    uint32_t hole = holes_before + (before & 0xFFFFu), src = sources_before + (before >> 16);
    holes_before += total & 0xFFFFu;
    sources_before += total >> 16;
    for (; given; given &= given - 1) holes[hole++] = beg + (uint32_t)__ffs((int)given) - 1;
    for (; taken; taken &= taken - 1) sources[src++] = beg + (uint32_t)__ffs((int)taken) - 1;
    copy();
  }
  if (here) {
    __syncthreads();
    const uint32_t lanes = a.kv.head_dim / 8;
    evict_moves(a, pair, s_holes, s_sources, tid / lanes, holes_before, THREADS / lanes);
  } else if (tid == 0) {
    a.count[pair] = holes_before;
  }
}

}  // namespace

// One workgroup per (row, kv head)
extern "C" __global__ __launch_bounds__(256) void catena_kv_evict_choose_1k(EvictArgs a) {
  evict_choose<256, 4, false>(a);
}
extern "C" __global__ __launch_bounds__(256) void catena_kv_evict_choose_1k_many_recent(EvictArgs a) {
  evict_choose<256, 4, true>(a);
}
extern "C" __global__ __launch_bounds__(1024) void catena_kv_evict_choose_8k(EvictArgs a) {
  evict_choose<1024, 8, false>(a);
}
extern "C" __global__ __launch_bounds__(1024) void catena_kv_evict_choose_8k_many_recent(EvictArgs a) {
  evict_choose<1024, 8, true>(a);
}

// grid = (pairs, ceil(most / 64)); 64 moves a workgroup.  Bound: HBM, 8 D bytes a
// move: the 32 x 8 rows' 1024 slots too many, heads of 128, 47.6 us at 4.5 TB/s, the
// rate of a copy.  (Four moves in flight a lane: two or eight take longer, and so do
// non-temporal stores.)
extern "C" __global__ __launch_bounds__(256) void catena_kv_evict_move(EvictArgs a) {
  const uint32_t pair = blockIdx.x, lanes = a.kv.head_dim / 8, first = blockIdx.y * 64, n = a.count[pair];
  if (first >= n) return;
  evict_moves(a, pair, a.holes + (uint64_t)pair * a.most, a.sources + (uint64_t)pair * a.most,
              first + threadIdx.x / lanes, n - first < 64 ? n : first + 64, 256 / lanes);
}

// ------------------------------------------------------------------ reorder
//
// Row r goes on as row p = parents[r] was: the pages that p has filled are
// shared (their numbers copied), the one it has partly filled is copied into r's
// spare page, whose place as spare r's own partly filled page takes.  Pages
// past it stay r's own.  Nothing that is read here is written: the tables are
// two, and a spare page is in no table.  A row that is its own parent keeps its
// pages.  A row whose parent does not exist, has another length than the row
// or one past the table is given up: length 0, no pages, its spare kept.  Where the
// parent's partly filled page is none of the pool's, r's is none either: neither its
// spare page nor its own has those rows.
//
// Bound: HBM, two passes over the used part of a page for each (row, head, pool); a
// launch where that is little.  64 rows x 8 heads of 128, 32 pools, 49 slots each: 65.6
// us, 5.5 TB/s; 4 rows 2.4 us.
// grid = (rows, kv_heads, pools): one (row, head, pool)'s slots of the last page;
// the workgroups of head 0 and pool 0 write the row's table.

namespace {
CATENA_DEV void kv_reorder(const ReorderArgs& a, uint16_t* const* pools) {
  const PagedKv& kv = a.kv;
  const uint32_t r = blockIdx.x, h = blockIdx.y, mask = (1u << kv.page_shift) - 1u;
  const uint32_t p = a.parents[r];
  const uint32_t n = p < kv.rows ? a.lens[p] : 0u;
  const bool good = p < kv.rows && n == a.lens[r] && n <= paged_slots(kv);
  const uint32_t last = n >> kv.page_shift, used = n & mask;
  const bool partly = good && p != r && used != 0;
  const uint32_t* mine = kv.table + (uint64_t)r * kv.max_pages;
  const uint32_t* theirs = kv.table + (uint64_t)(good ? p : r) * kv.max_pages;
  const uint32_t from = theirs[partly ? last : 0u], to = a.spare[r];
  const bool copies = partly && from < kv.num_pages;
  if (a.tables && h == 0 && blockIdx.z == 0) {
    uint32_t* out = a.table_out + (uint64_t)r * kv.max_pages;
    for (uint32_t j = threadIdx.x; j < kv.max_pages; j += 256)
      out[j] = !good ? 0xFFFFFFFFu : j < last ? theirs[j] : j == last && partly ? (copies ? to : from) : mine[j];
    if (threadIdx.x == 0) {
      a.lens_out[r] = good ? n : 0u;
      a.spare_out[r] = copies ? mine[last] : to;
    }
  }
  if (!copies || blockIdx.z >= a.n_pools) return;
  if (to >= kv.num_pages) return;
  uint16_t* pool = pools[blockIdx.z];
  const u32x4_t* src = reinterpret_cast<const u32x4_t*>(pool + paged_offset(kv, from, h, 0));
  u32x4_t* dst = reinterpret_cast<u32x4_t*>(pool + paged_offset(kv, to, h, 0));
  const uint32_t chunks = used * (kv.head_dim / 8);
  for (uint32_t i = threadIdx.x; i < chunks; i += 256) dst[i] = src[i];
}
}  // namespace

// The pools' pointers are kernel arguments: up to 8 (a few layers) or up to 128,
// whose 1 KiB takes 0.5 us longer to hand over.
extern "C" __global__ __launch_bounds__(256) void catena_kv_reorder_8(ReorderArgs a, ReorderPools<8> pools) {
  kv_reorder(a, pools.p);
}
extern "C" __global__ __launch_bounds__(256) void catena_kv_reorder_128(ReorderArgs a, ReorderPools<128> pools) {
  kv_reorder(a, pools.p);
}
