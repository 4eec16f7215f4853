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
// A token whose slot or position does not exist writes q turned by tab[0] and
// nothing else; one whose page does not exist writes q alone.
//
// Bound: HBM for prompts (4 bytes in, 2 out per value), one launch's latency for
// a decode step.  A thread takes four pairs (two 16-byte loads of x, two of the
// table, two 8-byte stores); a workgroup serves one token, so the page and
// the position are looked up once, by scalar loads.
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
// slot where two are equal; a NaN weight goes first.  The i-th slot given up
// below the budget takes the i-th kept slot from the budget on, so that the
// kept slots are the first ones: attention does not depend on the slots' order,
// and only as many rows move as were given up there.

namespace {

// Larger is kept: the whole order of the rule above but for the slot's number.
CATENA_DEV uint32_t keep_key(float weight, uint32_t pos, uint32_t late) {
  if (pos >= late) return 0xFFFFFFFFu;
  return weight != weight ? 0u : mono_bits(__float_as_uint(weight));
}

// Exclusive prefix sum over the workgroup's 1024 threads, and the total
CATENA_DEV uint32_t block_prefix(uint32_t x, uint32_t* s_wave, uint32_t* total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  uint32_t in = x;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t y = __shfl_up(in, d);
    if (lane >= (uint32_t)d) in += y;
  }
  __syncthreads();  // s_wave is free again
  if (lane == 63) s_wave[wave] = in;
  __syncthreads();
  uint32_t before = 0, sum = 0;
#pragma unroll
  for (uint32_t w = 0; w < 16; ++w) {
    const uint32_t v = s_wave[w];
    before += w < wave ? v : 0u;
    sum += v;
  }
  *total = sum;
  return before + in - x;
}

}  // namespace

// What a (row, kv head) keeps: the lists of slots to fill and of slots to fill
// them from, and the weights and positions of the slots that stay in place.
// The budget-th largest key is found digit by digit (12, 12 and 8 bits, a
// histogram in LDS each), then a thread walks a run of slots of its own.
// One workgroup of 1024 per (row, kv head); lists: count[pairs], holes
// [pairs][most], sources[pairs][most].
extern "C" __global__ __launch_bounds__(1024) void catena_kv_evict_choose(
    PagedKv kv, const uint32_t* lens, const uint32_t* seen, const float* acc_in, const uint32_t* pos_in,
    uint32_t* lens_out, float* acc_out, uint32_t* pos_out, uint32_t* count, uint32_t* holes, uint32_t* sources,
    uint32_t most, uint32_t budget, uint32_t recent) {
  __shared__ uint32_t hist[4096];
  __shared__ uint32_t s_wave[16], s_bin, s_left;
  const uint32_t pair = blockIdx.x, row = pair / kv.kv_heads, tid = threadIdx.x;
  const uint32_t n = paged_len(kv, lens[row]), kept = n < budget ? n : budget;
  const uint64_t base = (uint64_t)pair * paged_slots(kv);
  const float* acc = acc_in + base;
  const uint32_t* pos = pos_in + base;
  if (tid == 0 && pair % kv.kv_heads == 0) lens_out[row] = kept;
  const bool moved = acc_out != acc_in, moved_pos = pos_out != pos_in;
  if (n <= budget) {
    for (uint32_t j = tid; j < n; j += 1024) {
      if (moved) acc_out[base + j] = acc[j];
      if (moved_pos) pos_out[base + j] = pos[j];
    }
    if (tid == 0) count[pair] = 0;
    return;
  }
  const uint32_t total_seen = seen[row], late = total_seen - (recent < total_seen ? recent : total_seen);
  // the budget-th largest key: its bits from the top
  uint32_t prefix = 0, left = budget;
#pragma unroll 1
  for (int step = 0; step < 3; ++step) {
    const uint32_t shift = step == 0 ? 20 : step == 1 ? 8 : 0, bins = step == 2 ? 256 : 4096;
    const uint32_t above = step == 0 ? 0u : 0xFFFFFFFFu << (step == 1 ? 20 : 8);  // bits already known
    for (uint32_t b = tid; b < bins; b += 1024) hist[b] = 0;
    __syncthreads();
    for (uint32_t j = tid; j < n; j += 1024) {
      const uint32_t key = keep_key(acc[j], pos[j], late);
      if ((key & above) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // thread t's bins from the top: the keys above them, then bin by bin
    const uint32_t per = bins / 1024 ? bins / 1024 : 1;
    uint32_t mine = 0;
    for (uint32_t b = 0; b < per; ++b) {
      const uint32_t at = tid * per + b;
      if (at < bins) mine += hist[bins - 1 - at];
    }
    uint32_t total;
    uint32_t over = block_prefix(mine, s_wave, &total);
    if (over < left && over + mine >= left) {
      for (uint32_t b = 0; b < per; ++b) {
        const uint32_t bin = bins - 1 - (tid * per + b), c = hist[bin];
        if (over + c >= left) {
          s_bin = bin;
          s_left = left - over;
          break;
        }
        over += c;
      }
    }
    __syncthreads();
    prefix |= s_bin << shift;
    left = s_left;
  }
  // Slots of that very key: the first `left` of them are kept.  A thread's run
  // of slots, so that one prefix sum orders them all.
  const uint32_t per = (n + 1023) / 1024, beg = tid * per < n ? tid * per : n, end = beg + per < n ? beg + per : n;
  uint32_t equal = 0;
  for (uint32_t j = beg; j < end; ++j) equal += keep_key(acc[j], pos[j], late) == prefix;
  uint32_t total;
  const uint32_t equal0 = block_prefix(equal, s_wave, &total);
  uint32_t seen_eq = equal0, n_hole = 0, n_src = 0;
  for (uint32_t j = beg; j < end; ++j) {
    const uint32_t key = keep_key(acc[j], pos[j], late);
    const bool keep = key > prefix || (key == prefix && seen_eq++ < left);
    n_hole += !keep && j < budget;
    n_src += keep && j >= budget;
  }
  uint32_t holes_all, src_all;
  uint32_t hole = block_prefix(n_hole, s_wave, &holes_all), src = block_prefix(n_src, s_wave, &src_all);
  seen_eq = equal0;
  for (uint32_t j = beg; j < end; ++j) {
    const uint32_t key = keep_key(acc[j], pos[j], late);
    const bool keep = key > prefix || (key == prefix && seen_eq++ < left);
    if (j < budget) {
      if (!keep) {
        holes[(uint64_t)pair * most + hole++] = j;
      } else {
        if (moved) acc_out[base + j] = acc[j];
        if (moved_pos) pos_out[base + j] = pos[j];
      }
    } else if (keep) {
      sources[(uint64_t)pair * most + src++] = j;
    }
  }
  if (tid == 0) count[pair] = holes_all;
}

// The moves: a row of K and of V (16 bytes a lane), the slot's weight and
// position.  Sources lie from the budget on and are never written, so the order
// does not matter.  grid = (pairs, ceil(most / 64)); 64 moves a workgroup.
extern "C" __global__ __launch_bounds__(256) void catena_kv_evict_move(
    PagedKv kv, const float* acc_in, const uint32_t* pos_in, float* acc_out, uint32_t* pos_out,
    const uint32_t* count, const uint32_t* holes, const uint32_t* sources, uint32_t most) {
  const uint32_t pair = blockIdx.x, row = pair / kv.kv_heads, h = pair % kv.kv_heads;
  const uint32_t n = count[pair], lanes = kv.head_dim / 8;
  const uint32_t lane = threadIdx.x % lanes, first = blockIdx.y * 64 + threadIdx.x / lanes;
  const uint32_t end = blockIdx.y * 64 + 64 < n ? blockIdx.y * 64 + 64 : n;
  const uint64_t base = (uint64_t)pair * paged_slots(kv), list = (uint64_t)pair * most;
  for (uint32_t i = first; i < end; i += 256 / lanes) {
    const uint32_t to = holes[list + i], from = sources[list + i];
    uint64_t dst, src;
    if (paged_place(kv, row, h, to, &dst) && paged_place(kv, row, h, from, &src)) {
      const u32x4_t k = *reinterpret_cast<const u32x4_t*>(kv.k + src + 8 * lane);
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(kv.v + src + 8 * lane);
      *reinterpret_cast<u32x4_t*>(kv.k + dst + 8 * lane) = k;
      *reinterpret_cast<u32x4_t*>(kv.v + dst + 8 * lane) = v;
    }
    if (lane == 0) {
      acc_out[base + to] = acc_in[base + from];
      pos_out[base + to] = pos_in[base + from];
    }
  }
}

// ------------------------------------------------------------------ reorder
//
// Row r goes on as row p = parents[r] was: the pages that p has filled are
// shared (their numbers copied), the one it has partly filled is copied into r's
// spare page, whose place as spare r's own partly filled page takes.  Pages
// past it stay r's own.  Nothing that is read here is written: the tables are
// two, and a spare page is in no table.  A row that is its own parent keeps its
// pages.  A row whose parent does not exist, has another length than the row
// or one past the table is given up: length 0, no pages, its spare kept.
//
// grid = (rows, kv_heads, pools): one (row, head, pool)'s slots of the last page;
// the workgroups of head 0 and pool 0 write the row's table.
struct ReorderPools {
  uint16_t* p[128];
};
extern "C" __global__ __launch_bounds__(256) void catena_kv_reorder(
    PagedKv kv, ReorderPools pools, uint32_t n_pools, uint32_t tables, const uint32_t* lens, const uint32_t* parents,
    const uint32_t* spare, uint32_t* table_out, uint32_t* lens_out, uint32_t* spare_out) {
  const uint32_t r = blockIdx.x, h = blockIdx.y, mask = (1u << kv.page_shift) - 1u;
  const uint32_t p = parents[r];
  const uint32_t n = p < kv.rows ? lens[p] : 0u;
  const bool good = p < kv.rows && n == lens[r] && n <= paged_slots(kv);
  const uint32_t last = n >> kv.page_shift, used = n & mask;
  const bool copies = good && p != r && used != 0;
  const uint32_t* mine = kv.table + (uint64_t)r * kv.max_pages;
  const uint32_t* theirs = kv.table + (uint64_t)(good ? p : r) * kv.max_pages;
  if (tables && h == 0 && blockIdx.z == 0) {
    uint32_t* out = table_out + (uint64_t)r * kv.max_pages;
    for (uint32_t j = threadIdx.x; j < kv.max_pages; j += 256)
      out[j] = !good ? 0xFFFFFFFFu : j < last ? theirs[j] : j == last && copies ? spare[r] : mine[j];
    if (threadIdx.x == 0) {
      lens_out[r] = good ? n : 0u;
      spare_out[r] = copies ? mine[last] : spare[r];
    }
  }
  if (!copies || blockIdx.z >= n_pools) return;
  const uint32_t from = theirs[last], to = spare[r];
  if (from >= kv.num_pages || to >= kv.num_pages) return;
  uint16_t* pool = pools.p[blockIdx.z];
  const u32x4_t* src = reinterpret_cast<const u32x4_t*>(pool + paged_offset(kv, from, h, 0));
  u32x4_t* dst = reinterpret_cast<u32x4_t*>(pool + paged_offset(kv, to, h, 0));
  const uint32_t chunks = used * (kv.head_dim / 8);
  for (uint32_t i = threadIdx.x; i < chunks; i += 256) dst[i] = src[i];
}
