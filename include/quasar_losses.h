/* quasar_losses.h - log-probabilities of given tokens and the losses made of
 * them, over device-resident rows of logits (libquasar_cuda, sm_100a).
 *
 * What follows a pick when a model is scored or trained on the picked tokens:
 * the log-probability of each row's token at the sampling temperature, the
 * clipped policy loss and the paired preference loss, each with its gradient
 * into the logits. (No counterpart in the reference, which only samples.)
 *
 * Conventions are those of quasar_sampler.h: pointers named d_* are device
 * pointers on the current device, `stream` is a cudaStream_t (NULL = the
 * legacy default stream), calls are asynchronous on it and return a status
 * after the launch. No call allocates, synchronises or keeps anything between
 * calls: every buffer, scratch included, is the caller's, so calls that use
 * different buffers may overlap and every call can be captured into a graph.
 * A kernel's waits for its own copies and sums end after 2^32 cycles (about
 * 2 s; they take microseconds). Where one does, the status is still that of the
 * launch: rows whose sums were not complete by then come out NaN, and so do all
 * gradients of the CTA that gave up.
 * Outputs are apart from inputs and from each other but where it says may be.
 * Results do not depend on the run: no sum is formed by atomics.
 *
 * Rows. Row r of `rows` holds V logits at d_logits + r*ld (elements of dtype,
 * ld >= V, 1 <= V <= QUASAR_MAX_VOCAB, any alignment that the type has).
 * d_targets[r] is its token:
 *   target < 0      the row takes no part: its logits do not count (some
 *                   of them may be read), its outputs are 0 and its
 *                   gradient is a row of zeros;
 *   target >= V     the row's outputs and its gradient are NaN (the gradient
 *                   zeros in a row of weight 0, in a pair that takes no part
 *                   and outside of the sequences).
 * A logit of -inf has probability 0 (as banned tokens do). A row whose logits
 * are all -inf has no distribution: its log-probability is -inf, its entropy
 * 0 and its gradient zeros. NaN or +inf in a row that takes part makes that
 * row's outputs NaN.
 *
 * With z = l / temperature, M = max l, S = sum exp((l - M) / temperature):
 *   p_v      = exp((l_v - M) / temperature) / S
 *   logprob  = (l_target - M) / temperature - ln S
 *   entropy  = -sum p ln p
 * Sums over a row are kept in 32 bits by each thread and warp (V / 512 terms a
 * lane and CTA) and joined in 64 bits, where a row has more than 32 warps of up
 * to two of them added in 32; the policy loss of many long rows rounds each
 * CTA's sums to 32 bits before it joins a row's CTAs. From them
 * log-probabilities, entropies and row losses are formed in 64 bits and rounded
 * once; sums over sequences and rows are 64-bit sums of these rounded values.
 * Gradients, and the ratio and KL factor in them, are formed in 32 bits and
 * rounded once to dtype. So log-probabilities are good to about 4e-7 of 1 +
 * |logprob| (2^20 equal logits: 2e-5), entropies to 4e-6 of 1 + H (where one
 * logit holds most of a row: 2e-5).
 * A row whose derivatives by log-probability and entropy are both 0 (a clipped
 * ratio) has a gradient of zeros, whatever its logits. Where a derivative by the
 * log-probability is infinite, or so large that its products pass the fp32
 * range, the gradient is infinite with its sign where they do, and 0 where p is
 * 0 (an infinite derivative by the entropy defines nothing where p is not 0). */
#ifndef QUASAR_LOSSES_H
#define QUASAR_LOSSES_H

#include "quasar_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of logits and of gradients into them. */
#define QUASAR_F32  0
#define QUASAR_F16  1
#define QUASAR_BF16 2

/* What the gradient needs of a row's softmax. */
typedef struct {
    float max;   /* M (-inf: no finite logit) */
    float sum;   /* S */
} quasar_logprob_stat;

/* Log-probability of each row's target.
 *   temperature   > 0 and finite.
 *   d_logprob     [rows] out.
 *   d_entropy     [rows] out, or NULL (computing it costs about one more
 *                 multiply-add per logit).
 *   d_stats       [rows] out for quasar_token_logprobs_grad, or NULL. */
int quasar_token_logprobs(const void *d_logits, int dtype, int64_t ld, int rows, int V,
                          const int32_t *d_targets, float temperature,
                          float *d_logprob, float *d_entropy, quasar_logprob_stat *d_stats,
                          void *stream);

/* Gradient into the logits of sum_r (g_logprob[r] * logprob[r] +
 * g_entropy[r] * entropy[r]), with the stats (and entropies) that
 * quasar_token_logprobs gave for the same logits, targets and temperature:
 *   grad_v = (g_logprob * ([v == target] - p_v)
 *             - g_entropy * p_v * (ln p_v + entropy)) / temperature
 *   d_entropy, d_grad_entropy   [rows], both or neither NULL.
 *   d_grad        [rows][grad_ld] of dtype, every row of it written; may be
 *                 d_logits itself (with grad_ld == ld: in place), and must not
 *                 overlap it otherwise. Rows of d_grad with the 16-byte phase
 *                 of the logits' rows are written with 16-byte stores, others
 *                 element by element. */
int quasar_token_logprobs_grad(const void *d_logits, int dtype, int64_t ld, int rows, int V,
                               const int32_t *d_targets, float temperature,
                               const quasar_logprob_stat *d_stats, const float *d_entropy,
                               const float *d_grad_logprob, const float *d_grad_entropy,
                               void *d_grad, int64_t grad_ld, void *stream);

typedef struct {
    float temperature;    /* > 0: the temperature the tokens were sampled at */
    float clip_low;       /* >= 0: the ratio is clipped to [1 - clip_low, 1 + clip_high] */
    float clip_high;      /* >= 0 */
    float kl_coef;        /* weight of the KL term (nonzero needs d_ref_logprob) */
    float entropy_coef;   /* weight of the entropy bonus */
    float grad_scale;     /* multiplies the gradient, not the loss (loss scaling for 16-bit types) */
} quasar_policy_params;

/* Clipped policy loss of the rows' tokens and its gradient into the logits.
 * With ratio = exp(logprob - old_logprob) and u = ref_logprob - logprob:
 *   row_loss = -min(ratio * A, clip(ratio) * A) + kl_coef * (exp(u) - u - 1)
 *              - entropy_coef * entropy
 *   loss     = sum_r weight_r * row_loss_r
 * The gradient takes ratio, KL term and entropy as functions of the logits
 * (old and ref log-probabilities, advantages and weights are constants); a
 * ratio at a border counts as not clipped, and an advantage of 0 takes nothing
 * of a ratio, an infinite one either. Ratio and KL factor may pass the fp32
 * range (up to e^176) as long as their products with weight and grad_scale do
 * not.
 *   d_old_logprob, d_advantage   [rows].
 *   d_ref_logprob   [rows], or NULL with kl_coef == 0.
 *   d_weight        [rows], or NULL for 1/rows each. A row of weight 0 takes
 *                   no part, like one with a negative target.
 *   d_logprob       [rows] out; may be d_old_logprob or d_ref_logprob.
 *   d_entropy       [rows] out, or NULL.
 *   d_row_loss      [rows] out (not multiplied by the weight).
 *   d_loss          [1] out.
 *   d_grad          [rows][grad_ld] of dtype out as for
 *                   quasar_token_logprobs_grad (in place allowed), or NULL.
 * rows == 0 writes a loss of 0. */
int quasar_policy_loss(const void *d_logits, int dtype, int64_t ld, int rows, int V,
                       const int32_t *d_targets, const float *d_old_logprob, const float *d_advantage,
                       const float *d_ref_logprob, const float *d_weight,
                       const quasar_policy_params *params,
                       float *d_logprob, float *d_entropy, float *d_row_loss, float *d_loss,
                       void *d_grad, int64_t grad_ld, void *stream);

typedef struct {
    float temperature;       /* > 0 */
    float beta;              /* scale of the paired log ratio */
    float label_smoothing;   /* in [0, 1]: share of the loss with the pair turned round */
    float grad_scale;        /* multiplies the gradient, not the loss */
    int32_t length_normalize; /* nonzero: a sequence's score is the mean, not the sum, over its tokens */
    int32_t reserved;        /* set to 0 */
} quasar_preference_params;

/* Preference loss over pairs of packed sequences and its gradient into the
 * logits. Sequence s holds rows [d_cu_seqlens[s], d_cu_seqlens[s+1]); pair i
 * is sequences 2i (chosen) and 2i + 1 (rejected). Its rows with a target >= 0
 * count (a prompt's rows have target -1). With score_s the sum (or mean) of
 * the sequence's log-probabilities less ref_logprob_s:
 *   x         = beta * (score_chosen - score_rejected)
 *   pair_loss = -(1 - label_smoothing) * ln sigmoid(x) - label_smoothing * ln sigmoid(-x)
 *   loss      = sum_i weight_i * pair_loss_i
 *   d_cu_seqlens    [2*pairs + 1], from >= 0 up to <= rows, not falling. A
 *                   sequence may be empty (its score is 0 less the
 *                   reference's). Rows before the first and behind the last
 *                   sequence have a gradient of zeros. A pair whose
 *                   offsets fall or leave [0, rows] has a loss of NaN (and so
 *                   has the whole, unless the pair's weight is 0) and its
 *                   rows get no gradient.
 *   d_ref_logprob   [2*pairs] the reference model's scores (sums, or means
 *                   with length_normalize), or NULL for 0.
 *   d_pair_weight   [pairs], or NULL for 1/pairs each. A pair of weight 0
 *                   takes no part in loss and gradient.
 *   d_logprob       [rows] out, per token.
 *   d_seq_logprob   [2*pairs] out: the sums over the sequences; may be
 *                   d_ref_logprob.
 *   d_pair_loss     [pairs] out;  d_loss [1] out.
 *   d_stats         [rows] out;  d_row_grad [rows] out: the derivative of the
 *                   loss by each token's log-probability, times grad_scale.
 *   d_grad          [rows][grad_ld] of dtype out as for
 *                   quasar_token_logprobs_grad (in place allowed), or NULL.
 * pairs == 0 writes a loss of 0 and zero gradients. */
int quasar_preference_loss(const void *d_logits, int dtype, int64_t ld, int rows, int V,
                           const int32_t *d_targets, const int32_t *d_cu_seqlens, int pairs,
                           const float *d_ref_logprob, const float *d_pair_weight,
                           const quasar_preference_params *params,
                           float *d_logprob, float *d_seq_logprob, float *d_pair_loss, float *d_loss,
                           quasar_logprob_stat *d_stats, float *d_row_grad,
                           void *d_grad, int64_t grad_ld, void *stream);

/* ---- self-test ------------------------------------------------------------ */

/* quasar_policy_loss with waits of about wait_cycles (0 to 2^32, rounded down to
 * a power of two), of which one CTA's loads stop after `chunks` chunks where the
 * call takes the streaming kernel (many long rows, with d_grad): waits run out
 * there. Used by the GPU tests to see that what was not computed comes out NaN. */
int quasar_selftest_stalled_policy_loss(int64_t wait_cycles, int chunks,
                                        const void *d_logits, int dtype, int64_t ld, int rows, int V,
                                        const int32_t *d_targets, const float *d_old_logprob, const float *d_advantage,
                                        const float *d_ref_logprob, const float *d_weight,
                                        const quasar_policy_params *params,
                                        float *d_logprob, float *d_entropy, float *d_row_loss, float *d_loss,
                                        void *d_grad, int64_t grad_ld, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* QUASAR_LOSSES_H */
