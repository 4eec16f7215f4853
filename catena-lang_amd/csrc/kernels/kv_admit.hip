// Pages for the tokens of a step over requests of different lengths: who is
// admitted, which pages a row gets, where its tokens go; and pages given back.
//
// Free pages are a stack, free_pages[0 .. count).  A request's row has lens[r]
// slots in the pages table[r][0 .. held[r]); it asks for want[r] more slots:
//   t_r = want[r] where lens[r] + want[r] fits the table, else 0
//   p_r = max(0, pages of lens[r] + t_r - held[r]) where t_r > 0, else 0
// With T, P the sums of t, p over the rows up to r, r is admitted where T_r <=
// max_tokens and (p_r = 0 or P_r <= count).  Both sums grow, so the admitted rows
// that need pages are the first ones that do, and the pages P_r - p_r .. P_r - 1
// below the top of the stack are r's own.  So no row waits for another: every
// workgroup takes the sums itself, from the rows' words in L2, and then its share
// of the tokens; one launch.
//
// Bound: latency: the rows' words, two sums over a workgroup's 1024 rows, a token's row
// by halving, its page, one after the other.  A step of 64 rows 4.7 us (4.0 on the
// device), 64 prompts among 1024 rows, 131072 places 5.7 (5.6); as tensor operations 420.
#include "common.h"
#include "paged.h"

namespace {

constexpr uint32_t kThreads = 256, kRows = 1024;  // rows summed at a time, four a thread

// a + b, or the largest word
CATENA_DEV uint32_t add_sat(uint32_t a, uint32_t b) {
  const uint32_t c = a + b;
  return c < a ? 0xFFFFFFFFu : c;
}
// Inclusive sums over the wave, cut off at the largest word
CATENA_DEV uint32_t wave_prefix_sat(uint32_t x) {
#define CATENA_DPP_SAT(ctrl, rows) x = add_sat(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, (ctrl), (rows), 0xF, false))
  CATENA_DPP_SAT(0x111, 0xF);
  CATENA_DPP_SAT(0x112, 0xF);
  CATENA_DPP_SAT(0x114, 0xF);
  CATENA_DPP_SAT(0x118, 0xF);
  CATENA_DPP_SAT(0x142, 0xA);
  CATENA_DPP_SAT(0x143, 0xC);
#undef CATENA_DPP_SAT
  return x;
}

// Sums of two values over the workgroup's threads before this one, and over all
struct Two {
  uint32_t a, b;
};
CATENA_DEV Two block_before(Two x, Two* s_wave, Two* all) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const Two in = {wave_prefix_sat(x.a), wave_prefix_sat(x.b)};
  __syncthreads();  // the last sums have been read
  if (lane == 63) s_wave[wave] = in;
  // the lane before this one: its inclusive sum (a difference would not do where sums are cut off)
  Two before = {(uint32_t)__shfl_up((int)in.a, 1), (uint32_t)__shfl_up((int)in.b, 1)};
  if (lane == 0) before = Two{0, 0};
  __syncthreads();
  Two sum = {0, 0};
#pragma unroll
  for (uint32_t w = 0; w < kThreads / 64; ++w) {
    if (w == wave) before = Two{add_sat(before.a, sum.a), add_sat(before.b, sum.b)};
    sum = Two{add_sat(sum.a, s_wave[w].a), add_sat(sum.b, s_wave[w].b)};
  }
  *all = sum;
  return before;
}

// Number of the first n (a power of two) ascending words that are <= x, less one;
// s[0] <= x
CATENA_DEV uint32_t last_at_most(const uint32_t* s, uint32_t n, uint32_t x) {
  uint32_t at = 0;
  for (uint32_t step = n / 2; step > 0; step /= 2)
    if (s[at + step] <= x) at += step;
  return at;
}

// (no page for a place that is not on the stack, which no admitted row asks for)
CATENA_DEV uint32_t free_page(const AdmitArgs& a, uint32_t count, uint32_t at) {
  return at < count ? a.free_pages[at] : 0xFFFFFFFFu;
}

}  // namespace

// grid: workgroups that share the tokens
extern "C" __global__ __launch_bounds__(256) void catena_kv_admit(AdmitArgs a) {
  __shared__ Two s_wave[kThreads / 64];
  __shared__ uint32_t s_start[kRows], s_page[kRows], s_len[kRows], s_held[kRows], s_seen[kRows];
  const uint32_t tid = threadIdx.x;
  const uint64_t slots = (uint64_t)a.max_pages << a.page_shift;
  const uint32_t mask = (1u << a.page_shift) - 1u;
  const uint32_t given = *a.free_count, count = given < a.num_pages ? given : a.num_pages;
  uint32_t tokens = 0, pages = 0;      // admitted in the chunks before
  uint32_t asked_t = 0, asked_p = 0;   // asked for there
  const uint32_t* counted = a.seen ? a.seen : a.lens;
  for (uint32_t r0 = 0; r0 < a.rows; r0 += kRows) {
    uint32_t len[4], held[4], seen[4], t[4], p[4];
    Two sum = {0, 0}, all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = r0 + 4 * tid + i, in = 0u - (uint32_t)(r < a.rows), at = r < a.rows ? r : a.rows - 1;
      len[i] = a.lens[at] & in;
      held[i] = a.held[at] & in;
      t[i] = a.want[at] & in;
      seen[i] = counted[at] & in;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t to = (uint64_t)len[i] + t[i];
      t[i] = to > slots ? 0u : t[i];
      const uint32_t need = (uint32_t)((to + mask) >> a.page_shift);
      p[i] = (t[i] > 0) & (need > held[i]) ? need - held[i] : 0u;
      sum = Two{add_sat(sum.a, t[i]), add_sat(sum.b, p[i])};
    }
    Two before = block_before(sum, s_wave, &all);
    before = Two{add_sat(before.a, asked_t), add_sat(before.b, asked_p)};
    asked_t = add_sat(asked_t, all.a);
    asked_p = add_sat(asked_p, all.b);
    uint32_t first[4];
    sum = Two{0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      first[i] = before.b;
      before = Two{add_sat(before.a, t[i]), add_sat(before.b, p[i])};
      // (by a mask: as a branch, the compiler of ROCm 7.2 left out the zeroing of a
      // thread's first row where pages ran out; the built code was read to see it)
      const uint32_t fits = 0u - (uint32_t)((before.a <= a.max_tokens) & (before.a != 0xFFFFFFFFu) &
                                            ((p[i] == 0) | (before.b <= count)));
      t[i] &= fits;
      p[i] &= fits;
      sum = Two{sum.a + t[i], sum.b + p[i]};
    }
    before = block_before(sum, s_wave, &all);
    uint32_t start = tokens + before.a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = 4 * tid + i, r = r0 + at;
      s_start[at] = r < a.rows ? start : 0xFFFFFFFFu;
      s_page[at] = first[i];
      s_len[at] = len[i];
      s_held[at] = held[i];
      s_seen[at] = seen[i];
      if (blockIdx.x == 0 && r < a.rows) {
        a.starts[r] = start;
        a.lens_out[r] = len[i] + t[i];
        a.held_out[r] = held[i] + p[i];
        if (a.seen_out) a.seen_out[r] = seen[i] + t[i];
      }
      start += t[i];
    }
    __syncthreads();
    // the chunk's tokens, in workgroups' turns of 256 of all
    const uint32_t end = tokens + all.a;
    const uint64_t turn = (uint64_t)gridDim.x * kThreads;
    uint64_t k = (uint64_t)blockIdx.x * kThreads + tid;
    if (k < tokens) k += (tokens - k + turn - 1) / turn * turn;
    for (; k < end; k += turn) {
      const uint32_t at = last_at_most(s_start, kRows, (uint32_t)k), back = (uint32_t)k - s_start[at];
      const uint32_t slot = s_len[at] + back, entry = slot >> a.page_shift, have = s_held[at];
      uint32_t* row = a.table + (uint64_t)(r0 + at) * a.max_pages;
      uint32_t page;
      if (entry < have) {
        page = row[entry];
      } else {
        // a page's first new token enters it; the row's first one also those before its own
        const uint32_t top = count - 1 - s_page[at];
        page = free_page(a, count, top - (entry - have));
        if (back == 0)
          for (uint32_t e = have; e < entry; ++e) row[e] = free_page(a, count, top - (e - have));
        if (back == 0 || (slot & mask) == 0) row[entry] = page;
      }
      a.token_pos[k] = s_seen[at] + back;
      a.slot_map[k] = page < a.num_pages ? ((uint64_t)page << a.page_shift) + (slot & mask) : ~0ull;
    }
    tokens = end;
    pages += all.b;
    __syncthreads();  // the rows' words have been read
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.starts[a.rows] = tokens;
    *a.free_count_out = count - pages;
  }
  for (uint64_t k = (uint64_t)tokens + (uint64_t)blockIdx.x * kThreads + tid; k < a.max_tokens;
       k += (uint64_t)gridDim.x * kThreads) {
    a.token_pos[k] = 0;
    a.slot_map[k] = ~0ull;
  }
}

// Rows that have ended: their pages on top of the stack, in the order of rows and
// table entries.  grid: workgroups that share the pages
extern "C" __global__ __launch_bounds__(256) void catena_kv_release(ReleaseArgs a) {
  __shared__ Two s_wave[kThreads / 64];
  __shared__ uint32_t s_start[kRows];
  const uint32_t tid = threadIdx.x;
  const uint32_t given = *a.free_count, count = given < a.num_pages ? given : a.num_pages, room = a.num_pages - count;
  uint32_t pages = 0;
  for (uint32_t r0 = 0; r0 < a.rows; r0 += kRows) {
    uint32_t n[4];
    Two sum = {0, 0}, all;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = r0 + 4 * tid + i;
      const bool in = r < a.rows;
      const uint32_t at = in ? r : a.rows - 1;
      const uint32_t ended = (uint32_t)(a.finished[at] == 0) - 1u, held = a.held[at];  // all bits of one that has ended
      n[i] = (0u - (uint32_t)in) & ended & (held < a.max_pages ? held : a.max_pages);
      sum.a = add_sat(sum.a, n[i]);
      if (in & (blockIdx.x == 0)) {
        a.lens_out[r] = ~ended & a.lens[r];
        a.held_out[r] = ~ended & held;
      }
    }
    uint32_t start = add_sat(pages, block_before(sum, s_wave, &all).a);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s_start[4 * tid + i] = r0 + 4 * tid + i < a.rows ? start : 0xFFFFFFFFu;
      start = add_sat(start, n[i]);
    }
    __syncthreads();
    const uint32_t end = add_sat(pages, all.a);
    const uint64_t turn = (uint64_t)gridDim.x * kThreads;
    uint64_t k = (uint64_t)blockIdx.x * kThreads + tid;
    if (k < pages) k += (pages - k + turn - 1) / turn * turn;
    for (; k < end; k += turn) {
      const uint32_t at = last_at_most(s_start, kRows, (uint32_t)k);
      uint32_t* entry = a.table + (uint64_t)(r0 + at) * a.max_pages + ((uint32_t)k - s_start[at]);
      if (k < room) a.free_pages[count + k] = *entry;
      *entry = 0xFFFFFFFFu;
    }
    pages = end;
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) *a.free_count_out = count + (pages < room ? pages : room);
}
