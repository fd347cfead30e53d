// C ABI of the operators on logits and beams: argument checks, then one
// launcher each. No call synchronises the device.
#include <cmath>
#include <string>

#include "kernels.cuh"
#include "status.h"

namespace {

#define CK(expr)                                                     \
  do {                                                               \
    cudaError_t _e = (expr);                                         \
    if (_e != cudaSuccess) return rnet_status::fail_cuda(_e, #expr); \
  } while (0)
#define NEED(cond, msg) \
  if (!(cond)) return rnet_status::fail(RNET_ERR_ARG, msg)

unsigned* ew() { return rnet_status::device_error_word(); }

bool aligned(const void* p, size_t n) { return ((size_t)p & (n - 1)) == 0; }

size_t elem(int dtype) { return dtype == RNET_DTYPE_BF16 ? 2 : 4; }

// Whether the bytes up to the last of `rows` rows can be counted.
bool pitch_fits(int rows, long long ld) { return rows == 0 || ld <= (1LL << 60) / rows; }

// Bytes that `rows` rows with a pitch of ld elements span.
size_t span(int rows, long long ld, int vocab, int dtype) {
  return rows > 0 ? ((size_t)(rows - 1) * (size_t)ld + (size_t)vocab) * elem(dtype) : 0;
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
  const size_t x = (size_t)a, y = (size_t)b;
  return na && nb && x < y + nb && y < x + na;
}

const std::string TOPK_RANGE = "top_k must be 1.." + std::to_string(RNET_TOPK_MAX);
const std::string BEAM_RANGE = "beams must be 1.." + std::to_string(RNET_BEAMS_MAX);

}  // namespace

extern "C" {

int rnet_topk_logits_forward(const void* logits, int dtype, long long ld, float temperature,
                             float* top_logits, int* top_idx, float* lse, int rows, int vocab,
                             int top_k, void* stream) {
  NEED(logits && top_logits && top_idx, "topk_logits_forward: null pointer");
  NEED(dtype == RNET_DTYPE_F32 || dtype == RNET_DTYPE_BF16,
       "topk_logits_forward: dtype must be RNET_DTYPE_F32 or RNET_DTYPE_BF16");
  NEED(rows >= 0 && vocab > 0, "topk_logits_forward: bad size");
  NEED(vocab <= RNET_SELECT_VOCAB_MAX, "topk_logits_forward: vocab above 2^30");
  NEED(ld >= vocab, "topk_logits_forward: row pitch below vocab");
  NEED(pitch_fits(rows, ld), "topk_logits_forward: row pitch too large");
  NEED(top_k >= 1 && top_k <= RNET_TOPK_MAX && top_k <= vocab,
       "topk_logits_forward: " + TOPK_RANGE + " and not above vocab");
  NEED(temperature >= 1e-4f && temperature <= 1e4f,
       "topk_logits_forward: temperature must be within 1e-4 and 1e4");
  NEED(aligned(logits, elem(dtype)) && aligned(top_logits, 4) && aligned(top_idx, 4) &&
           aligned(lse, 4),
       "topk_logits_forward: a pointer is not aligned to its element size");
  CK(rnet_k::topk_logits(logits, dtype == RNET_DTYPE_BF16, ld, temperature, top_logits, top_idx,
                         lse, rows, vocab, top_k, ew(), (cudaStream_t)stream));
  return RNET_OK;
}

int rnet_distill_topk_forward(const void* logits, int dtype, long long ld, const int* teacher_idx,
                              const float* teacher_logits, const float* teacher_lse,
                              const int* targets, const float* row_weight, float temperature,
                              float soft_weight, float hard_weight, float grad_scale,
                              float* row_loss, float* loss, void* dlogits, long long ld_dlogits,
                              int rows, int vocab, int top_k, void* stream) {
  NEED(logits && teacher_idx && teacher_logits && row_loss, "distill_topk_forward: null pointer");
  NEED(dtype == RNET_DTYPE_F32 || dtype == RNET_DTYPE_BF16,
       "distill_topk_forward: dtype must be RNET_DTYPE_F32 or RNET_DTYPE_BF16");
  NEED(rows >= 0 && vocab > 0, "distill_topk_forward: bad size");
  NEED(ld >= vocab && (!dlogits || ld_dlogits >= vocab),
       "distill_topk_forward: row pitch below vocab");
  NEED(pitch_fits(rows, ld) && (!dlogits || pitch_fits(rows, ld_dlogits)),
       "distill_topk_forward: row pitch too large");
  if (vocab > RNET_DISTILL_VOCAB_MAX)
    return rnet_status::fail(RNET_ERR_UNSUPPORTED,
                             "distill_topk_forward: vocab above " +
                                 std::to_string(RNET_DISTILL_VOCAB_MAX));
  NEED(top_k >= 1 && top_k <= RNET_TOPK_MAX, "distill_topk_forward: " + TOPK_RANGE);
  NEED(temperature >= 1e-4f && temperature <= 1e4f,
       "distill_topk_forward: temperature must be within 1e-4 and 1e4");
  NEED(std::isfinite(soft_weight) && std::isfinite(hard_weight) && std::isfinite(grad_scale),
       "distill_topk_forward: weights and grad_scale must be finite");
  NEED(hard_weight == 0.0f || targets, "distill_topk_forward: hard_weight needs targets");
  NEED(aligned(logits, elem(dtype)) && aligned(dlogits, elem(dtype)) && aligned(teacher_idx, 4) &&
           aligned(teacher_logits, 4) && aligned(teacher_lse, 4) && aligned(targets, 4) &&
           aligned(row_weight, 4) && aligned(row_loss, 4) && aligned(loss, 4),
       "distill_topk_forward: a pointer is not aligned to its element size");
  NEED((dlogits == logits && ld == ld_dlogits) ||
           !overlap(logits, span(rows, ld, vocab, dtype), dlogits,
                    dlogits ? span(rows, ld_dlogits, vocab, dtype) : 0),
       "distill_topk_forward: dlogits overlaps the logits without being them");
  CK(rnet_k::distill_topk(logits, dtype == RNET_DTYPE_BF16, ld, teacher_idx, teacher_logits,
                          teacher_lse, targets, row_weight, temperature, soft_weight, hard_weight,
                          grad_scale, row_loss, loss, dlogits, ld_dlogits, rows, vocab, top_k,
                          ew(), (cudaStream_t)stream));
  return RNET_OK;
}

int rnet_beam_select(const void* logits, int dtype, long long ld, const float* scores_in,
                     const int* finished_in, int eos, float* scores, int* tokens, int* parents,
                     int* finished, int batch, int beams, int vocab, void* stream) {
  NEED(logits && scores_in && scores && tokens && parents, "beam_select: null pointer");
  NEED(dtype == RNET_DTYPE_F32 || dtype == RNET_DTYPE_BF16,
       "beam_select: dtype must be RNET_DTYPE_F32 or RNET_DTYPE_BF16");
  NEED(batch >= 0 && vocab > 0, "beam_select: bad size");
  NEED(beams >= 1 && beams <= RNET_BEAMS_MAX, "beam_select: " + BEAM_RANGE);
  NEED((long long)batch * beams <= 0x7fffffffLL, "beam_select: batch * beams too large");
  NEED(vocab <= RNET_SELECT_VOCAB_MAX, "beam_select: vocab above 2^30");
  NEED(ld >= vocab, "beam_select: row pitch below vocab");
  NEED(pitch_fits(batch * beams, ld), "beam_select: row pitch too large");
  NEED(eos >= -1 && eos < vocab, "beam_select: eos must be -1 (none) or a token");
  NEED(!finished_in || (eos >= 0 && finished),
       "beam_select: finished beams need an eos token and the finished output");
  NEED(aligned(logits, elem(dtype)) && aligned(scores_in, 4) && aligned(finished_in, 4) &&
           aligned(scores, 4) && aligned(tokens, 4) && aligned(parents, 4) && aligned(finished, 4),
       "beam_select: a pointer is not aligned to its element size");
  CK(rnet_k::beam_select(logits, dtype == RNET_DTYPE_BF16, ld, scores_in, finished_in, eos, scores,
                         tokens, parents, finished, batch, beams, vocab, ew(),
                         (cudaStream_t)stream));
  return RNET_OK;
}

int rnet_beam_reorder(const void* src, void* dst, size_t row_bytes, size_t row_pitch, size_t outer,
                      size_t outer_pitch, const int* parents, int batch, int beams, void* stream) {
  NEED(src && dst && parents, "beam_reorder: null pointer");
  NEED(batch >= 0 && batch <= 65535 && outer <= 65535,
       "beam_reorder: batch must be 0..65535 and outer at most 65535");
  NEED(beams >= 1 && beams <= RNET_BEAMS_MAX, "beam_reorder: " + BEAM_RANGE);
  NEED(row_bytes % 4 == 0 && row_pitch % 4 == 0 && outer_pitch % 4 == 0 && aligned(src, 4) &&
           aligned(dst, 4) && aligned(parents, 4),
       "beam_reorder: rows, pitches and pointers must be multiples of 4 bytes");
  NEED(row_bytes <= ((size_t)1 << 38), "beam_reorder: row too long");
  const size_t rows = (size_t)batch * beams;
  NEED(row_pitch >= row_bytes, "beam_reorder: row pitch below the row");
  NEED(rows == 0 || row_pitch <= ((size_t)1 << 62) / rows, "beam_reorder: row pitch too large");
  const size_t plane = rows ? (rows - 1) * row_pitch + row_bytes : 0;
  NEED(outer <= 1 || (outer_pitch >= plane && outer_pitch <= ((size_t)1 << 62) / outer),
       "beam_reorder: outer pitch below a plane of rows");
  const size_t bytes = outer ? (outer - 1) * outer_pitch + plane : 0;
  NEED(src == dst || !overlap(src, bytes, dst, bytes),
       "beam_reorder: dst overlaps src without being it");
  CK(rnet_k::beam_reorder(src, dst, row_bytes, row_pitch, outer, outer_pitch, parents, batch,
                          beams, ew(), (cudaStream_t)stream));
  return RNET_OK;
}

int rnet_beam_backtrack(const int* tokens, const int* parents, const float* scores, int eos,
                        float length_alpha, int* sequences, int* lengths, float* ranked_scores,
                        int n_steps, int batch, int beams, void* stream) {
  NEED(tokens && parents && scores && sequences && lengths && ranked_scores,
       "beam_backtrack: null pointer");
  NEED(n_steps >= 1 && n_steps <= (1 << 30) && batch >= 0, "beam_backtrack: bad size");
  NEED(beams >= 1 && beams <= RNET_BEAMS_MAX, "beam_backtrack: " + BEAM_RANGE);
  NEED((long long)batch * beams <= 0x7fffffffLL, "beam_backtrack: batch * beams too large");
  NEED(std::isfinite(length_alpha), "beam_backtrack: length_alpha must be finite");
  NEED(aligned(tokens, 4) && aligned(parents, 4) && aligned(scores, 4) && aligned(sequences, 4) &&
           aligned(lengths, 4) && aligned(ranked_scores, 4),
       "beam_backtrack: a pointer is not aligned to its element size");
  const size_t bytes = (size_t)n_steps * batch * beams * sizeof(int);
  NEED(!overlap(sequences, bytes, tokens, bytes) && !overlap(sequences, bytes, parents, bytes),
       "beam_backtrack: sequences overlap the records");
  CK(rnet_k::beam_backtrack(tokens, parents, scores, eos, length_alpha, sequences, lengths,
                            ranked_scores, n_steps, batch, beams, ew(), (cudaStream_t)stream));
  return RNET_OK;
}

}  // extern "C"
