// Kernel ABI of beam search's selection (beam.hip).  Arguments are checked
// before the device is looked for.
#include <cstdint>

#include "internal.h"

using namespace catena;

namespace {
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

struct BeamPlan {
  uint32_t per, runs;  // logits a thread holds; runs a row
  uint64_t rows, sums, maxima, bytes;  // best[rows][runs][beams] u64 comes first
};

int beam_plan(uint32_t groups, uint32_t beams, uint32_t vocab, BeamPlan* p) {
  if (beams == 0 || vocab == 0) return fail(CATENA_ERR_INVALID_ARGUMENT, "%u beams over %u tokens", beams, vocab);
  if (beams > 32 || vocab > (1u << 26))
    return fail(CATENA_ERR_UNSUPPORTED, "beam selection of %u beams over %u tokens", beams, vocab);
  p->rows = (uint64_t)groups * beams;
  // (a grid's first side, whose threads may not pass 32 bits)
  if (p->rows > 0xFFFFFFull) return fail(CATENA_ERR_UNSUPPORTED, "too many beams");
  // 16 logits a thread; 8 while that gives less than a workgroup for each CU
  // (4 x 32000: 4.3 us against 4.7; 256 x 128000: 31.8 against 22.7)
  p->per = p->rows * ((vocab + 4095) / 4096) < 256 ? 8 : 16;
  p->runs = (vocab + 256 * p->per - 1) / (256 * p->per);
  const uint64_t parts = p->rows * p->runs;
  p->sums = parts * beams * 8;
  p->maxima = p->sums + parts * 8;
  p->bytes = p->maxima + parts * 4;
  return CATENA_OK;
}
}  // namespace

extern "C" {

int catena_mi355x_beam_select_plan(uint32_t groups, uint32_t beams, uint32_t vocab, uint64_t* workspace_bytes) {
  if (!workspace_bytes) return fail(CATENA_ERR_INVALID_ARGUMENT, "null output");
  BeamPlan p;
  const int st = beam_plan(groups, beams, vocab, &p);
  if (!st) *workspace_bytes = p.bytes;
  return st;
}

int catena_mi355x_beam_select_f32(const float* logits, const float* scores, const uint32_t* done, uint32_t* tokens,
                                  uint32_t* parents, float* scores_out, uint32_t* done_out, uint32_t groups,
                                  uint32_t beams, uint32_t vocab, uint32_t eos, void* workspace,
                                  uint64_t workspace_bytes) {
  BeamPlan p;
  int st = beam_plan(groups, beams, vocab, &p);
  if (st) return st;
  if (groups == 0) return CATENA_OK;
  if (!logits || !scores || !tokens || !parents || !scores_out)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "null operand");
  const void* words[] = {logits, scores, done, tokens, parents, scores_out, done_out};
  for (const void* w : words)
    if (!aligned(w, 4)) return fail(CATENA_ERR_INVALID_ARGUMENT, "misaligned operand");
  if (eos == 0xFFFFFFFFu ? done != nullptr : eos >= vocab)
    return fail(CATENA_ERR_INVALID_ARGUMENT, "end token %u of %u", eos, vocab);
  if (!workspace || workspace_bytes < p.bytes || !aligned(workspace, 16))
    return fail(CATENA_ERR_INVALID_ARGUMENT, "beam selection needs %llu bytes of 16-byte aligned workspace",
                (unsigned long long)p.bytes);
  st = ensure_init();
  if (st) return st;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  uint64_t* best = reinterpret_cast<uint64_t*>(ws);
  double* part_s = reinterpret_cast<double*>(ws + p.sums);
  float* part_m = reinterpret_cast<float*>(ws + p.maxima);
  uint32_t runs = p.runs;
  void* args[] = {&logits, &done, &part_m, &part_s, &best, &vocab, &beams};
  st = launch(p.per == 8 ? KernelId::BeamRuns8 : KernelId::BeamRuns16, dim3((unsigned)p.rows, runs), dim3(256), 0, args);
  if (st) return st;
  void* jargs[] = {&part_m, &part_s, &best, &scores, &done, &tokens, &parents, &scores_out, &done_out, &runs, &beams, &eos};
  return launch(KernelId::BeamJoin, dim3(groups), dim3(64 * (beams < 16 ? beams : 16)), 0, jargs);
}

}  // extern "C"
