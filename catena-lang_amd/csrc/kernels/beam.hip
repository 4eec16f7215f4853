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
// its rows and merges the W sorted lists.
//
// Scores of different beams meet in 64 bits: within a beam the logits decide, but
// between beams the sums may lie closer than 32 bits can tell.  Exponentials and
// a thread's sum of 16 are f32 (each off by 2^-23 of itself), sums of those and
// all that follows f64.
#include "common.h"

namespace {

constexpr int PER = 16;             // logits a thread holds
constexpr uint32_t RUN = 256 * PER;  // and a workgroup
constexpr uint32_t LIST = 1024;      // candidates it can sort at once
constexpr float kNegInf = -__builtin_huge_valf();

// Orders offered logits (larger first, lower token where equal); 0: not offered
CATENA_DEV uint32_t offer(float x) { return x > kNegInf ? mono_bits(__float_as_uint(x)) : 0u; }
CATENA_DEV float offered(uint32_t mono) {
  return __uint_as_float((mono & 0x80000000u) ? (mono & 0x7FFFFFFFu) : ~mono);
}
CATENA_DEV uint64_t with_token(uint32_t mono, uint32_t token) { return mono ? ((uint64_t)mono << 32) | ~token : 0ull; }

// The largest of the wave's values
CATENA_DEV uint64_t wave_max64(uint64_t x) {
  const uint32_t hi = wave_umax((uint32_t)(x >> 32));
  const uint32_t lo = wave_umax((uint32_t)(x >> 32) == hi ? (uint32_t)x : 0u);
  return ((uint64_t)hi << 32) | lo;
}

}  // namespace

// Run blockIdx.y of row blockIdx.x: part_m its maximum, part_s the sum of
// exp(logit - maximum), best[W] its largest (with_token, 0 where there are fewer).
// The W-th largest of one wave's 64 lane maxima is a bound that W logits reach:
// what reaches the largest such bound of the four waves is listed and
// sorted by counting.  Where more do than the list holds (equal logits), the W
// are taken one after the other.
extern "C" __global__ __launch_bounds__(256) void catena_beam_runs(
    const float* __restrict__ logits, const uint32_t* __restrict__ done, float* __restrict__ part_m,
    double* __restrict__ part_s, uint64_t* __restrict__ best, uint32_t vocab, uint32_t beams) {
  __shared__ float s_max[4];
  __shared__ double s_sum[4];
  __shared__ uint32_t s_bound[4], s_count;
  __shared__ uint64_t s_key[LIST], s_wave[4];
  const uint32_t row = blockIdx.x, run = blockIdx.y, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  if (done && done[row]) return;
  const float* x = logits + (uint64_t)row * vocab;
  const uint32_t first = run * RUN + tid;
  float v[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) v[k] = first + 256 * k < vocab ? x[first + 256 * k] : kNegInf;
  if (tid == 0) s_count = 0;

  float top = v[0];
#pragma unroll
  for (int k = 1; k < PER; ++k) top = __builtin_fmaxf(top, v[k]);  // of the numbers: a NaN shows in the sum
  const uint32_t mine = offer(top);
  // the maximum, and the wave's bound
  uint32_t bound = 0;
#pragma unroll 1
  for (int b = 31; b >= 0; --b) {
    const uint32_t t = bound | (1u << b);
    if ((uint32_t)__popcll(__ballot(mine >= t)) >= beams) bound = t;
  }
  const uint32_t wmax = wave_umax(mine);
  if (lane == 0) {
    s_max[wave] = wmax ? offered(wmax) : kNegInf;
    s_bound[wave] = bound;
  }
  __syncthreads();
  const float m = __builtin_fmaxf(__builtin_fmaxf(s_max[0], s_max[1]), __builtin_fmaxf(s_max[2], s_max[3]));
  bound = max(max(max(s_bound[0], s_bound[1]), max(s_bound[2], s_bound[3])), 1u);
  // exp(x - m) = 2^(x log2e - m log2e), the product's rounding made good by a
  // second one; no reference point while nothing is above -inf
  const float ref = m == kNegInf ? 0.0f : m;
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const float d = v[k] - ref;
    const float hi = d * 1.44269502f;
    const float lo = __builtin_fmaf(d, 1.44269502f, -hi) + d * 1.92596303e-8f;
    float e = __builtin_amdgcn_exp2f(hi);
    if (d > -__builtin_huge_valf()) e = __builtin_fmaf(e, lo * 0.693147182f, e);
    sum = sum + e;
  }
  double total = (double)sum;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) total = total + __shfl_xor(total, d);
  if (lane == 0) s_sum[wave] = total;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const uint32_t key = offer(v[k]);
    if (key >= bound) {
      const uint32_t at = atomicAdd(&s_count, 1u);
      if (at < LIST) s_key[at] = with_token(key, first + 256 * k);
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
    for (uint32_t i = tid; i < n; i += 256) {
      const uint64_t key = s_key[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; ++j) rank += s_key[j] > key;
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

// Group blockIdx.x: a wave joins a row's runs (its log sum in f64) and takes the
// W largest of their lists, each lane at the head of lists of its own; then the
// first wave merges the rows' lists, lane w at the head of beam w's.
// W <= 32.  A place that no offered continuation fills: its own beam as
// parent, token 0, score -inf, not done.
extern "C" __global__ __launch_bounds__(1024) void catena_beam_join(
    const float* __restrict__ part_m, const double* __restrict__ part_s, const uint64_t* __restrict__ best,
    const float* scores, const uint32_t* done, uint32_t* tokens, uint32_t* parents, float* scores_out,
    uint32_t* done_out, uint32_t runs, uint32_t beams, uint32_t eos) {
  __shared__ uint64_t s_best[32][32];
  __shared__ double s_shift[32];
  __shared__ uint32_t s_done[32];
  const uint32_t group = blockIdx.x, lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (uint32_t w = wave; w < beams; w += 16) {
    const uint32_t row = group * beams + w;
    const double score = (double)scores[row];
    if (done && done[row]) {
      if (lane == 0) {
        s_done[w] = 1;
        s_shift[w] = score;
      }
      continue;
    }
    const float* pm = part_m + (uint64_t)row * runs;
    const double* ps = part_s + (uint64_t)row * runs;
    float m = kNegInf;
    for (uint32_t r = lane; r < runs; r += 64) m = __builtin_fmaxf(m, pm[r]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = __builtin_fmaxf(m, __shfl_xor(m, d));
    const double ref = m == kNegInf ? 0.0 : (double)m;
    double sum = 0.0;
    for (uint32_t r = lane; r < runs; r += 64) sum = sum + ps[r] * exp((double)pm[r] - ref);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) sum = sum + __shfl_xor(sum, d);
    if (lane == 0) {
      s_done[w] = 0;
      s_shift[w] = score - (ref + log(sum));
    }
    const uint64_t* lists = best + (uint64_t)row * runs * beams;
    uint64_t last = ~0ull;
    uint64_t head = 0;  // the largest of this lane's lists below `last`
    bool stale = true;
    for (uint32_t r = 0; r < beams; ++r) {
      if (stale) {
        head = 0;
        for (uint32_t q = lane; q < runs; q += 64) {
          const uint64_t* list = lists + (uint64_t)q * beams;
          for (uint32_t i = 0; i < beams; ++i) {
            const uint64_t key = list[i];
            if (key < last) {
              head = key > head ? key : head;
              break;
            }
          }
        }
      }
      const uint64_t top = wave_max64(head);
      if (lane == 0) s_best[w][r] = top;
      last = top;
      stale = head == top;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  const uint32_t w = lane;
  const bool here = w < beams;
  const double shift = here ? s_shift[w] : 0.0;
  const bool over = here && s_done[w] != 0;
  const bool offers = here && shift - shift == 0.0;  // finite
  uint32_t at = 0;
  for (uint32_t r = 0; r < beams; ++r) {
    // this beam's next continuation as an ordered integer: 0 where it has none
    uint64_t key = 0;
    uint32_t token = 0;
    double s = 0.0;
    if (offers && at < (over ? 1u : beams)) {
      if (over) {
        s = shift;
        token = eos;
        key = 1;
      } else if (s_best[w][at]) {
        const uint64_t b = s_best[w][at];
        s = (double)offered((uint32_t)(b >> 32)) + shift;
        token = ~(uint32_t)b;
        key = 1;
      }
      if (key) {
        const uint64_t bits = (uint64_t)__double_as_longlong(s + 0.0);  // -0 as +0
        key = (bits >> 63) ? ~bits : bits | (1ull << 63);
      }
    }
    const uint64_t top = wave_max64(key);
    const uint32_t out = group * beams + r;
    if (top == 0) {
      if (lane == 0) {
        tokens[out] = 0;
        parents[out] = out;
        scores_out[out] = kNegInf;
        if (done_out) done_out[out] = 0;
      }
      continue;
    }
    const uint32_t winner = (uint32_t)__ffsll((unsigned long long)__ballot(key == top)) - 1;
    if (lane == winner) {
      tokens[out] = token;
      parents[out] = group * beams + w;
      scores_out[out] = (float)s;
      if (done_out) done_out[out] = over || token == eos;
      ++at;
    }
  }
}
