/* C ABI of libfmhip.so, token-level entry points: distillation from a teacher's listed columns and
 * sampling. The conventions (device pointers, dense rows, caller-owned buffers, no allocation and
 * no synchronisation, status codes, fm_last_error, fixed-order reductions) are those of fm_hip.h. */
#ifndef FM_HIP_TOKENS_H_
#define FM_HIP_TOKENS_H_

#include "fm_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------ KL from a teacher's list
 * KL(teacher || student) where the teacher is known at k columns of each row only (a stored or a
 * remote teacher; fm_kl_fwd_topk and fm_topk write such lists). With z = student / temperature,
 * p = softmax(z) over all v columns, and q the teacher's probabilities of its listed columns:
 *   FM_TAIL_DROP, FM_TAIL_RENORM   row_loss = sum_j q_j (log q_j - log p_j)
 *   FM_TAIL_BUCKET                 the same + q_r (log q_r - log p_r): everything unlisted is one
 *                                  more outcome, q_r = max(0, 1 - sum q), p_r = the student's
 *                                  probability of all unlisted columns (summed, not 1 - sum p)
 * idx: [n, k] int32 or int64 (index_bits). A negative entry is an empty slot; a row whose slot 0
 * is empty is skipped: loss 0, gradient 0, not counted by the mean, its logits not read. A column
 * that a row lists more than once counts once, with the sum of its probabilities. A column >= v
 * makes the row's loss and gradient NaN, and so does a NaN or +inf among the logits, or nothing but -inf. With FM_TAIL_BUCKET and every column listed, q_r = 0.
 * teacher: [n, k] of teacher_dtype.
 *   FM_TEACHER_LOGITS  q = softmax(teacher / temperature) over the row's slots (FM_TAIL_RENORM), or
 *                      exp(teacher / temperature - teacher_lse[row]) (the other two; teacher_lse:
 *                      fp32 [n], the log-sum-exp of the teacher's whole row / temperature)
 *   FM_TEACHER_PROBS   q = teacher (already at the temperature), divided by its sum for FM_TAIL_RENORM
 * The listed columns and the row's loss are computed in 64 bits (the loss is a small difference),
 * the sweep over the row in fp32.
 * row_loss: fp32 [n]. stats: fp32 [n, 4] for fm_kl_topk_bwd (base-2 exponent and the sum of weights
 * against it, of the whole row, then of its unlisted columns; a negative sum goes with the largest logit itself,
 * where masks with the lowest values leave nothing else). loss, n_valid: fp32 device scalars; loss = sum of
 * row_loss (FM_REDUCE_SUM) or that / n_valid (FM_REDUCE_MEAN), n_valid = max(1, rows not skipped);
 * both may be NULL for FM_REDUCE_NONE, which writes neither. 1 <= k <= 1024, k may exceed v;
 * n < 2^22, v < 2^30 (FM_ERR_UNSUPPORTED past those). */
enum fm_teacher { FM_TEACHER_LOGITS = 0, FM_TEACHER_PROBS = 1 };
enum fm_tail { FM_TAIL_RENORM = 0, FM_TAIL_DROP = 1, FM_TAIL_BUCKET = 2 };

int fm_kl_topk_fwd(const void* student, const void* idx, const void* teacher, const float* teacher_lse,
                   float* row_loss, float* stats, float* loss, float* n_valid, int64_t n, int64_t v,
                   int k, int dtype, int index_bits, int teacher_dtype, int teacher_kind, int tail,
                   double temperature, int reduction, fm_stream_t stream);

/* The same and the gradient wrt the undivided student logits for an upstream gradient of 1, from
 * one launch over the rows: dstudent [n, v] of dtype (it may be the student buffer itself),
 *   dstudent_j = (p_j sum(q) - q_j) / temperature [/ n_valid],  unlisted columns of FM_TAIL_BUCKET:
 *   (p_j - q_r p_j / p_r) / temperature [/ n_valid].
 * Sum or mean only. What a row has beyond the registers and LDS of a workgroup is read twice.
 * fm_scale_inplace applies another upstream gradient. stats may be NULL. */
int fm_kl_topk_loss_grad(const void* student, const void* idx, const void* teacher, const float* teacher_lse,
                         float* row_loss, float* stats, float* loss, float* n_valid, void* dstudent, int64_t n,
                         int64_t v, int k, int dtype, int index_bits, int teacher_dtype, int teacher_kind,
                         int tail, double temperature, int reduction, fm_stream_t stream);

/* That gradient from the saved stats, with any upstream gradient: multiplied by grad_out[row]
 * (grad_per_row != 0) or grad_out[0], divided by *n_valid; NULL counts as 1 for either. dstudent is a
 * buffer of its own. */
int fm_kl_topk_bwd(const void* student, const void* idx, const void* teacher, const float* teacher_lse,
                   const float* stats, const float* n_valid, const float* grad_out, int grad_per_row,
                   void* dstudent, int64_t n, int64_t v, int k, int dtype, int index_bits, int teacher_dtype,
                   int teacher_kind, int tail, double temperature, fm_stream_t stream);

/* ------------------------------------------------------------------ sampling
 * One token per row of logits [n, v] from one uniform number per row. With T the temperature,
 * m the row's maximum and e_j = exp((x_j - m) / T), and the order "value descending, index ascending":
 *   top_k   > 0 (and below v): only the first top_k of the order stay;
 *   top_p   < 1: rank r stays iff the mass before it is below top_p times the mass top_k left
 *           (rank 0 always stays);
 *   min_p   > 0: only e_j >= min_p stay (values above 1 count as 1);
 *   token   = the first column (ascending) whose running sum of the e that stay exceeds u times their
 *           sum; logprob = log(e_token / sum).
 * T == 0 takes the first maximum (logprob 0), whatever the filters. A row that has no distribution --
 * it holds a NaN or +inf or nothing but -inf, or T is negative, infinite or NaN -- gets token -1 and
 * logprob NaN. u counts as at most the largest fp32 below 1 and at least 0 (NaN: 0). top_p or min_p
 * NaN: off. Logits of -inf are never taken.
 * u: fp32 [n]. temperature, top_p, min_p: fp32 [n] or NULL for the number behind them for every row;
 * top_k: int32 [n] or NULL likewise. token: int64 [n]; logprob: fp32 [n] or NULL. logits may have any
 * alignment of their type. Weights are computed in 64 bits, rounded to multiples of 2^-fx (fx = 63 - log2 v
 * rounded up, at most 50; where nothing cuts, the sums of 512 to 2048 columns are) and summed as integers: a
 * row's token and logprob are the same bits whatever rows come with it. v <= 2^20, n < 2^22 (FM_ERR_UNSUPPORTED
 * past those). */
int fm_sample(const void* logits, const float* u, const float* temperature, const int32_t* top_k,
              const float* top_p, const float* min_p, float temperature0, int top_k0, float top_p0,
              float min_p0, int64_t* token, float* logprob, int64_t n, int64_t v, int dtype,
              fm_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FM_HIP_TOKENS_H_ */
