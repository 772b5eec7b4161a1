// token_loss.cuh - launchers of the token log-probability, policy-loss and
// preference-loss kernels (token_loss.cu); the C entries are in losses.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/quasar_losses.h"

namespace qs {
namespace loss {

struct Args {
    const void* logits;
    int64_t ld;
    int rows, V;
    const int32_t* targets;
    float k;       // log2(e) / temperature: exp((l - M) / T) = 2^((l - M) * k)
    // streaming kernel's self-test, else 0: its waits end after 2^(high 8 bits)
    // cycles, and one CTA's loads stop after (low 24 bits) - 1 chunks. (In what
    // was padding: beyond 216 bytes of arguments a launch takes 0.4 us longer.)
    uint32_t selftest;
    double inv_t;  // 1 / temperature

    float* logprob;
    float* entropy;
    quasar_logprob_stat* stats;

    // policy loss (adv != NULL)
    const float* old_lp;
    const float* adv;
    const float* ref_lp;
    const float* weight;
    double mean;  // the weight of a row with weight == NULL
    double clip_lo, clip_hi, kl, ec;
    float* row_loss;
    double scale;  // gradient scale

    // preference loss: zeroed by the statistics kernel, filled by the pair kernel;
    // to the gradient kernel a sign that rows of g_lp 0 take no part, whatever
    // their target
    float* row_grad;

    // gradient (policy: NULL for none)
    void* grad;
    int64_t grad_ld;
    const float* g_lp;       // gradient kernel: per-row derivatives
    const float* g_ent;      // ... or NULL
    const float* ent_in;     // entropies the statistics kernel gave (with g_ent)
    const quasar_logprob_stat* stats_in;
};
static_assert(sizeof(Args) == 216, "see selftest");

struct PairArgs {
    const float* logprob;
    const int32_t* targets;
    const int32_t* cu;
    int pairs, rows;
    const float* ref;
    double beta, eps, scale;
    int mean;
    const float* weight;
    float *seq, *pair_loss, *row_grad;
};

// Log-probabilities (and, with args.adv, the policy loss and its gradient).
cudaError_t launch_rows(const Args& a, int dtype, cudaStream_t st);
// The gradient into the logits from given per-row derivatives.
cudaError_t launch_grad(const Args& a, int dtype, cudaStream_t st);
// Sequence sums, pair losses, their weighted sum and the rows' derivatives.
cudaError_t launch_pairs(const PairArgs& p, float* loss, cudaStream_t st);
// out[0] = sum of w[i] * x[i] (w NULL: 1/n each), in index order by blocks.
cudaError_t launch_weighted_sum(const float* x, const float* w, int n, float* out, cudaStream_t st);

}  // namespace loss
}  // namespace qs
