// C ABI of the vocabulary losses (lz_losses.cu): token log-probabilities, a
// clipped policy loss, a preference loss and distillation from a teacher's
// top logits. Mirrored by the ctypes structure in results_b200/ops/losses.py.
#pragma once
#include <cuda_runtime.h>

#define LZ_LOSS_LOGP 0     /* log-probability of one token per row */
#define LZ_LOSS_POLICY 1   /* clipped policy loss with a KL term */
#define LZ_LOSS_DISTILL 2  /* KL from a teacher's top logits */

#define LZ_LOSS_MAX_TOP 1024

// Doubles in front of the per-row parts of `work` (1 / denominator; ticket and
// number of rows that count) and per row.
#define LZ_LOSS_WORK_HEAD 2
#define LZ_LOSS_WORK_ROW 5

#ifdef __cplusplus
extern "C" {
#endif

struct LzLossArgs {
  // logits of row r: logits + (r / inner) * outer_stride + (r % inner) * inner_stride
  // (elements); the vocabulary itself is contiguous
  const void* logits;
  long long outer_stride, inner_stride, inner;
  long long rows, vocab;
  void* grad;            // [rows][vocab] contiguous, logits' type; null: no gradient
  const void* ids;       // LOGP, POLICY: token of each row; DISTILL: [rows][top]
  const void* teacher;   // DISTILL: [rows][top] logits
  const float* old_logp; // POLICY, [rows]
  const float* advantages;
  const float* ref_logp; // null: no KL term
  const float* weights;  // [rows]; null: every row counts once
  const float* denom_ptr;  // device scalar, or null
  const float* upstream;     // backward: device scalar; null: 1
  const float* row_upstream; // backward of LOGP: [rows]
  float* loss;           // scalar (POLICY, DISTILL)
  float* logp;           // [rows] (LOGP, POLICY)
  float* kl;             // [rows] (POLICY with ref_logp, DISTILL)
  unsigned char* clipped;  // [rows] (POLICY)
  // [HEAD + ROW rows], 16-byte aligned: head, then per row its sum (four
  // floats), the slope of the loss in its log-probability (LOGP: that itself, in
  // 64 bits, since sums of many are taken of it), a CTA's loss, and its
  // place in the order in which rows are taken (int)
  double* work;
  double denom;          // denominator; < 0: the sum of the weights
  float inv_temperature, clip_low, clip_high, kl_coef;
  int kind, dtype, ids64, top, teacher_dtype, device;
  int fresh;             // backward: 1 when `grad` does not hold the gradient for upstream 1 yet
  unsigned long long capture;  // of the forward pass (set by it): the id of the graph capture that it ran in, 0 for none
  unsigned long long wait_ns;  // bound of every wait in the kernels; 0: 4 s, 1: nothing is waited for
};

#define LZ_LOSS_APART 1  /* nothing ran: the forward pass ran in another capture */

// Statistics, outputs and (grad != null) the gradient for upstream 1.
int lz_loss_forward(struct LzLossArgs* a, cudaStream_t stream);
// The gradient for another upstream value, from the statistics in `work`. Without `fresh` it
// returns LZ_LOSS_APART where one of the two passes can run again without the other (either was
// captured into a graph, or each into one of its own): `grad` is then the wrong memory to hand out,
// since it is only written for upstream 1 by the forward pass, and any time that runs again.
int lz_loss_backward(const struct LzLossArgs* a, cudaStream_t stream);

// Preference loss from the rows' log-probabilities (the `work` that lz_loss_forward
// of LOGP left, ids as there):
// sequences are [offsets[i], offsets[i+1]) or `length` rows each; the first
// `pairs` are the chosen ones. Writes loss, rewards [2 pairs] and, in work, the slopes.
struct LzPairArgs {
  const double* logp_work;
  const void* ids;
  const void* offsets;   // [2 pairs + 1] or null
  const float* ref_logp; // [2 pairs] or null
  float *loss, *rewards;
  double* work;          // ticket, losses of the pairs [pairs], slopes of the rows (float [rows])
  long long rows, pairs, length;
  double beta, smoothing;
  int normalized, ids64, offsets64, device;
};
int lz_loss_pairs(const struct LzPairArgs* a, cudaStream_t stream);

#ifdef __cplusplus
}
#endif
