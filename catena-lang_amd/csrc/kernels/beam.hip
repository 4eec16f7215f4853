// Beam search's selection over beams and vocabulary.
//
//   score(w, v) = scores[w] + (logits[w][v] - log sum_u exp(logits[w][u]))
//
// over the beams w and tokens v of a group; the beams' best W of the W * V
// continuations, larger score first; equal scores: the lower beam, then the
// larger logit, then the lower token.  A done beam offers one continuation, the
// end token at its own score.  A continuation whose score is not finite is not
// offered, so a beam whose logits hold NaN or +inf (or nothing above -inf)
// offers none.
//
// Bound: the logits are read once, 4 bytes each, so HBM; for one request the
// latency of two launches.  First kernel: a workgroup keeps a run of a row's
// logits in registers, takes their maximum, the sum of their exponentials and
// their W largest.  Second kernel: a workgroup per group joins the runs of
// its rows and takes the W largest of their lists.  Per
// logit the first one issues a maximum, a subtraction, a product, an exponential
// (four times an add), an add and a comparison; exponentials by exp2, keys only
// for logits that reach the bound, loads without address arithmetic: 32 beams x 8
// x 128000 in 22.0 us (6.0 TB/s), against 38 with keys for all and exponentials
// in two steps.
//
// Accuracy, in units of u = 2^-24: an exponential is off by 2.3 |x - m| (the
// difference, its product with log2 e, and log2 e itself are f32) and 2, a thread's sum
// of 16 by 5.  Their mean under the row's probabilities is what the log sum is off by:
// that of |x - m| is the entropy less (log sum - m), so at most ln V, 18 for the most
// tokens: 3e-6 at most, and it does not fall with V where the terms are alike (one logit
// 8.59 above 127999 equal ones: 4e-7).  Further sums, and scores, are f64.  Within a beam
// the logits decide; scores of two beams are told apart down to twice that.
// (Exponentials in f64 as well, by a polynomial of degree 11: 43.5 us instead of 26.6 for
// the 32 x 8 rows with their join.)
#include "common.h"

namespace {

constexpr uint32_t LIST = 1024;      // candidates it can sort at once
constexpr float kNegInf = -__builtin_huge_valf();
constexpr int kNonTemporal = 2;
constexpr float kLog2e = 1.44269502f;

// Orders offered logits (larger first, lower token where equal); 0: not offered
CATENA_DEV uint32_t offer(float x) { return x > kNegInf ? mono_bits(__float_as_uint(x)) : 0u; }
CATENA_DEV float offered(uint32_t mono) {
  return __uint_as_float((mono & 0x80000000u) ? (mono & 0x7FFFFFFFu) : ~mono);
}
CATENA_DEV uint64_t with_token(uint32_t mono, uint32_t token) { return mono ? ((uint64_t)mono << 32) | ~token : 0ull; }

// The largest of the wave's values; the lower halves meet only where the upper
// ones are equal
CATENA_DEV uint64_t wave_max64(uint64_t x) {
  const uint32_t hi = wave_umax((uint32_t)(x >> 32));
  const uint64_t have = __ballot((uint32_t)(x >> 32) == hi);
  uint32_t lo;
  if ((have & (have - 1)) == 0)
    lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, __ffsll((unsigned long long)have) - 1);
  else
    lo = wave_umax((uint32_t)(x >> 32) == hi ? (uint32_t)x : 0u);
  return ((uint64_t)hi << 32) | lo;
}

// The sum of the wave's values in f64: within rows of 16 lanes, then rows to rows
CATENA_DEV double wave_sum64(double x) {
#define CATENA_DPP_ADD64(ctrl, rows)                                                                        \
  {                                                                                                         \
    const uint64_t b = (uint64_t)__double_as_longlong(x);                                                     \
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, (ctrl), (rows), 0xF, false); \
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), (ctrl), (rows), 0xF, false);   \
    x = x + __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));                                     \
  }
  CATENA_DPP_ADD64(0x111, 0xF);
  CATENA_DPP_ADD64(0x112, 0xF);
  CATENA_DPP_ADD64(0x114, 0xF);
  CATENA_DPP_ADD64(0x118, 0xF);
  CATENA_DPP_ADD64(0x142, 0xA);
  CATENA_DPP_ADD64(0x143, 0xC);
#undef CATENA_DPP_ADD64
  const uint64_t b = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), 63);
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}

// A bound that at least `beams` of the wave's 64 values reach (of those that are
// not 0; 0 where there are fewer), near the largest such one
CATENA_DEV uint32_t wave_bound(uint32_t x, uint32_t beams) {
  uint32_t bound = 0;
#pragma unroll
  for (int b = 31; b >= 14; --b) {
    const uint32_t t = bound | (1u << b);
    if ((uint32_t)__popcll(__ballot(x >= t)) >= beams) bound = t;
  }
  return bound;
}

// Run blockIdx.y of row blockIdx.x: part_m its maximum, part_s the sum of
// exp(logit - maximum), best[W] its largest (with_token, 0 where there are
// fewer).  The W-th largest of one wave's 64 lane maxima, cut to 18 bits, is a
// bound that W logits reach: what reaches the largest such bound of the four
// waves is listed and sorted by counting.  Where more do than the list holds
// (equal logits), the W are taken one after the other.
template <int PER>
CATENA_DEV void beam_runs(const float* __restrict__ logits, const uint32_t* __restrict__ done,
                          float* __restrict__ part_m, double* __restrict__ part_s, uint64_t* __restrict__ best,
                          uint32_t vocab, uint32_t beams) {
  __shared__ float s_max[4];
  __shared__ double s_sum[4];
  __shared__ uint32_t s_bound[4], s_count;
  __shared__ uint64_t s_key[LIST + 8], s_wave[4];
  const uint32_t row = blockIdx.x, run = blockIdx.y, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  if (done && done[row]) return;
  const uint32_t first = run * 256 * PER + tid;
  const int bytes = (int)(vocab * 4u);  // at most 2^28
  const __amdgpu_buffer_rsrc_t x =
      __builtin_amdgcn_make_buffer_rsrc((void*)(logits + (uint64_t)row * vocab), (short)0, bytes, 0x00020000);
  float v[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k)
    v[k] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(x, (int)(first * 4), 1024 * k, kNonTemporal));
  if (first - tid + 256 * PER > vocab) {
#pragma unroll
    for (int k = 0; k < PER; ++k) v[k] = first + 256 * k < vocab ? v[k] : kNegInf;
  }
  if (tid == 0) s_count = 0;

  float top = v[0];
#pragma unroll
  for (int k = 1; k < PER; ++k) top = __builtin_fmaxf(top, v[k]);  // of the numbers: a NaN shows in the sum
  const uint32_t mine = offer(top);
  // the maximum, and the wave's bound
  const uint32_t wmax = wave_umax(mine);
  uint32_t bound = wave_bound(mine, beams);
  if (lane == 0) {
    s_max[wave] = wmax ? offered(wmax) : kNegInf;
    s_bound[wave] = bound;
  }
  __syncthreads();
  const float m = __builtin_fmaxf(__builtin_fmaxf(s_max[0], s_max[1]), __builtin_fmaxf(s_max[2], s_max[3]));
  bound = max(max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3])), 1u);
  // nothing to refer to while nothing is above -inf
  const float c = m == kNegInf ? 0.0f : m;
  float sum[4] = {};
#pragma unroll
  for (int k = 0; k < PER; ++k) sum[k % 4] = sum[k % 4] + __builtin_amdgcn_exp2f((v[k] - c) * kLog2e);
  const double total = wave_sum64((double)((sum[0] + sum[1]) + (sum[2] + sum[3])));
  if (lane == 0) s_sum[wave] = total;
  if (mine >= bound) {
    const float least = bound == 1u ? -__FLT_MAX__ : offered(bound);
    uint32_t which = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) which |= v[k] >= least ? 1u << k : 0u;
    while (which) {
      const uint32_t one = (uint32_t)__ffs((int)which) - 1;
      which &= which - 1;
      float value = v[0];
#pragma unroll
      for (int k = 1; k < PER; ++k) value = one == (uint32_t)k ? v[k] : value;
      const uint32_t at = atomicAdd(&s_count, 1u);
      if (at < LIST) s_key[at] = with_token(offer(value), first + 256 * one);
    }
  }
  __syncthreads();
  const uint64_t part = (uint64_t)row * gridDim.y + run;
  if (tid == 0) {
    part_m[part] = m;
    part_s[part] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
  }
  const uint32_t n = s_count;
  uint64_t* out = best + part * beams;
  if (n <= LIST) {
    if (tid < 8) s_key[n + tid] = 0;  // eight at a time
    __syncthreads();
    for (uint32_t i = tid; i < n; i += 256) {
      const uint64_t key = s_key[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; j += 8)
#pragma unroll
        for (int e = 0; e < 8; ++e) rank += s_key[j + e] > key;
      if (rank < beams) out[rank] = key;
    }
    if (tid >= n && tid < beams) out[tid] = 0;
    return;
  }
  uint64_t last = ~0ull;
  for (uint32_t r = 0; r < beams; ++r) {
    uint64_t b = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const uint64_t key = with_token(offer(v[k]), first + 256 * k);
      if (key < last && key > b) b = key;
    }
    b = wave_max64(b);
    if (lane == 0) s_wave[wave] = b;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) b = s_wave[w] > b ? s_wave[w] : b;
    if (tid == 0) out[r] = b;
    last = b;
    __syncthreads();
  }
}

// The `beams` largest of n keys (and of those in best, where there are any) into
// best in order, by one wave: PER keys a lane in registers (the keys are sorted lists of
// `beams`; shifted, so that a lane has entries of several ranks and few keys reach
// the bound that half the lanes' largest do).  Those that reach the
// wave's bound are listed and sorted by counting; where they are more than the
// list holds, the largest is taken out time after time.
constexpr uint32_t WLIST = 128;
// Each of the list's count keys to its place, by the number of larger ones; behind
// them the list has eight zeros
template <int PER>
CATENA_DEV void place(const uint64_t* list, uint32_t count, uint64_t* best, uint32_t beams) {
  const uint32_t lane = threadIdx.x & 63u;
  uint64_t mine[PER];
  uint32_t above[PER] = {};
#pragma unroll
  for (int i = 0; i < PER; ++i) mine[i] = lane + 64 * i < count ? list[lane + 64 * i] : 0ull;
  for (uint32_t j = 0; j < count; j += 8)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint64_t x = list[j + e];
#pragma unroll
      for (int i = 0; i < PER; ++i) above[i] += x > mine[i];
    }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (mine[i] && above[i] < beams) best[above[i]] = mine[i];
}

template <int PER>
CATENA_DEV void largest_of(const uint64_t* keys, uint32_t n, bool more, uint64_t* best, uint32_t beams,
                           uint64_t* list) {
  const uint32_t lane = threadIdx.x & 63u;
  uint64_t k[PER + 1];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t at = 64 * i + ((lane + 5 * i) & 63u);
    k[i] = at < n ? keys[at] : 0ull;
  }
  k[PER] = more && lane < beams ? best[lane] : 0ull;
  uint64_t mine = 0;
#pragma unroll
  for (int i = 0; i <= PER; ++i) mine = k[i] > mine ? k[i] : mine;
  // (few keys are sorted sooner than bounded)
  const uint32_t least = !more && n <= 32 ? 1u : max(wave_bound((uint32_t)(mine >> 32), beams), 1u);
  uint32_t count = 0;
#pragma unroll
  for (int i = 0; i <= PER; ++i) {
    const bool in = (uint32_t)(k[i] >> 32) >= least;
    const uint64_t have = __ballot(in);
    const uint32_t at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0));
    if (in && at < WLIST) list[at] = k[i];
    count += (uint32_t)__popcll(have);
  }
  if (count <= WLIST && lane < 8) list[count + lane] = 0;  // eight at a time
  __builtin_amdgcn_wave_barrier();
  if (count <= WLIST) {
    if (count <= 64) {
      place<1>(list, count, best, beams);
    } else {
      place<2>(list, count, best, beams);
    }
    if (lane >= count && lane < beams) best[lane] = 0;
    return;
  }
  uint64_t kept = 0;
  for (uint32_t r = 0; r < beams; ++r) {
    const uint64_t top = wave_max64(mine);
    if (lane == r) kept = top;
    if (mine == top) {
      mine = 0;
#pragma unroll
      for (int i = 0; i <= PER; ++i) mine = k[i] < top && k[i] > mine ? k[i] : mine;
    }
  }
  if (lane < beams) best[lane] = kept;
}

}  // namespace

extern "C" __global__ __launch_bounds__(256) void catena_beam_runs_8(
    const float* logits, const uint32_t* done, float* part_m, double* part_s, uint64_t* best, uint32_t vocab,
    uint32_t beams) {
  beam_runs<8>(logits, done, part_m, part_s, best, vocab, beams);
}
extern "C" __global__ __launch_bounds__(256) void catena_beam_runs_16(
    const float* logits, const uint32_t* done, float* part_m, double* part_s, uint64_t* best, uint32_t vocab,
    uint32_t beams) {
  beam_runs<16>(logits, done, part_m, part_s, best, vocab, beams);
}
// Group blockIdx.x: a wave joins a row's runs (their log sum in f64) and takes
// the W largest of their lists; then the first wave takes the W largest of all
// rows', as f64 scores in ordered integers whose last ten bits give way to the
// entry's number, so that no two are equal and a lower beam goes first.  (Merging
// the rows' lists entry by entry takes 0.2 us each: 4, 8, 16, 32 beams 4.2, 5.5,
// 8.7, 16.6 us against 3.7, 4.6, 6.4, 11.4.)  W <= 32; 64 threads a beam, up to 16.
// A place that no offered continuation fills: its own beam as parent, token 0,
// score -inf, not done.
extern "C" __global__ __launch_bounds__(1024) void catena_beam_join(
    const float* __restrict__ part_m, const double* __restrict__ part_s, const uint64_t* __restrict__ best,
    const float* scores, const uint32_t* done, uint32_t* tokens, uint32_t* parents, float* scores_out,
    uint32_t* done_out, uint32_t runs, uint32_t beams, uint32_t eos) {
  __shared__ uint64_t s_best[32][32];  // with_token, then the scores as ordered integers
  __shared__ uint32_t s_token[32][32];
  __shared__ uint64_t s_list[16][WLIST + 8];
  __shared__ uint32_t s_done[32];
  __shared__ uint64_t s_key[32 * 32], s_won[32];
  const uint32_t group = blockIdx.x, lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (uint32_t w = wave; w < beams; w += blockDim.x / 64) {
    const uint32_t row = group * beams + w;
    // a done beam's parts were not written: read all the same, so that nothing
    // waits for the flag, and not used
    const double score = (double)scores[row];
    const bool over = done && done[row] != 0;
    const float* pm = part_m + (uint64_t)row * runs;
    const double* ps = part_s + (uint64_t)row * runs;
    const uint64_t* keys = best + (uint64_t)row * runs * beams;
    const uint32_t n = runs * beams;
    // a run of nothing above -inf adds 0 (or its NaN)
    float m = lane < runs ? pm[lane] : kNegInf;
    double sum = lane < runs ? ps[lane] : 0.0;
    if (n <= 64) {
      largest_of<1>(keys, n, false, s_best[w], beams, s_list[wave]);
    } else if (n <= 256) {
      largest_of<4>(keys, n, false, s_best[w], beams, s_list[wave]);
    } else {
      for (uint32_t i = 0; i < n; i += 1024)
        largest_of<16>(keys + i, n - i < 1024 ? n - i : 1024, i != 0, s_best[w], beams, s_list[wave]);
    }
    const float mine = m;
    for (uint32_t r = lane + 64; r < runs; r += 64) m = __builtin_fmaxf(m, pm[r]);
    const uint32_t top = wave_umax(offer(m));
    m = top ? offered(top) : kNegInf;
    sum = lane < runs ? sum * exp((double)mine - (double)m) : 0.0;
    for (uint32_t r = lane + 64; r < runs; r += 64) sum = sum + ps[r] * exp((double)pm[r] - (double)m);
    sum = wave_sum64(sum);
    const double shift = over ? score : score - ((double)m + log(sum));
    // the row's continuations: 0 where it has no more, or offers none
    if (lane == 0) s_done[w] = over;
    if (lane < beams) {
      const uint64_t b = over ? (lane == 0 ? 1ull : 0ull) : s_best[w][lane];
      const double s = over ? shift : (double)offered((uint32_t)(b >> 32)) + shift;
      const uint64_t bits = (uint64_t)__double_as_longlong(s + 0.0);  // -0 as +0
      s_token[w][lane] = over ? eos : ~(uint32_t)b;
      const uint64_t key = (bits >> 63) ? ~bits : bits | (1ull << 63);
      s_best[w][lane] = key;
      s_key[w * beams + lane] =
          b == 0 || !(shift - shift == 0.0) ? 0ull : (key & ~1023ull) | (1023u - (32 * w + lane));
    }
  }
  __syncthreads();
  if (wave != 0) return;
  const uint32_t n = beams * beams;
  if (n <= 64)
    largest_of<1>(s_key, n, false, s_won, beams, s_list[0]);
  else if (n <= 256)
    largest_of<4>(s_key, n, false, s_won, beams, s_list[0]);
  else
    largest_of<16>(s_key, n, false, s_won, beams, s_list[0]);
  __builtin_amdgcn_wave_barrier();
  if (lane >= beams) return;
  const uint32_t out = group * beams + lane;
  const uint64_t won = s_won[lane];
  const bool filled = won != 0;
  const uint32_t place = 1023u - (uint32_t)(won & 1023u), w = place / 32, token = filled ? s_token[w][place % 32] : 0u;
  const uint64_t score = s_best[w][place % 32];
  const uint64_t bits = (score >> 63) ? score & ~(1ull << 63) : ~score;
  tokens[out] = token;
  parents[out] = filled ? group * beams + w : out;
  scores_out[out] = filled ? (float)__longlong_as_double((long long)bits) : kNegInf;
  if (done_out) done_out[out] = filled && (s_done[w] != 0 || token == eos);
}
