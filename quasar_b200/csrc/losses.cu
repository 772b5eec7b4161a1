// losses.cu - the C entries of include/quasar_losses.h: argument checks and
// launch order.
#include <math.h>
#include <string.h>

#include "../../include/quasar_losses.h"
#include "ptx.cuh"
#include "token_loss.cuh"

namespace {

size_t type_size(int dtype) { return dtype == QUASAR_F32 ? 4 : 2; }

bool check_rows(const void* d_logits, int dtype, int64_t ld, int rows, int V, const int32_t* d_targets, float temperature) {
    if (dtype != QUASAR_F32 && dtype != QUASAR_F16 && dtype != QUASAR_BF16) return false;
    if (rows < 0 || V < 1 || V > QUASAR_MAX_VOCAB || ld < V) return false;
    // 1/temperature has to be a float too
    if (!(temperature > 0.0f) || !isfinite(temperature) || !isfinite(2.0f / temperature)) return false;
    if (rows == 0) return true;
    if (ld > INT64_MAX / 4 / rows) return false;
    return d_logits && d_targets && (uintptr_t)d_logits % type_size(dtype) == 0 && (uintptr_t)d_targets % 4 == 0;
}

// A gradient of the logits' shape: in place, or apart from them.
bool check_grad(const void* d_logits, int dtype, int64_t ld, int rows, int V, const void* d_grad, int64_t grad_ld) {
    if (grad_ld < V) return false;
    if (rows == 0) return true;
    if (grad_ld > INT64_MAX / 4 / rows || !d_grad || (uintptr_t)d_grad % type_size(dtype) != 0) return false;
    if (d_grad == d_logits) return grad_ld == ld || rows == 1;
    const uintptr_t l0 = (uintptr_t)d_logits, l1 = l0 + ((size_t)(rows - 1) * ld + V) * type_size(dtype);
    const uintptr_t g0 = (uintptr_t)d_grad, g1 = g0 + ((size_t)(rows - 1) * grad_ld + V) * type_size(dtype);
    return g1 <= l0 || l1 <= g0;
}

qs::loss::Args row_args(const void* d_logits, int64_t ld, int rows, int V, const int32_t* d_targets, float temperature) {
    qs::loss::Args a;
    memset(&a, 0, sizeof a);
    a.logits = d_logits;
    a.ld = ld;
    a.rows = rows;
    a.V = V;
    a.targets = d_targets;
    a.inv_t = 1.0 / (double)temperature;
    a.k = (float)(1.4426950408889634074 * a.inv_t);
    return a;
}

// A failed launch's error is this call's status, and not the next call's last error.
int status(cudaError_t e) {
    if (e == cudaSuccess) return QUASAR_OK;
    cudaGetLastError();
    return QUASAR_ECUDA;
}

int policy_loss(uint32_t selftest, const void* d_logits, int dtype, int64_t ld, int rows, int V, const int32_t* d_targets,
                const float* d_old_logprob, const float* d_advantage, const float* d_ref_logprob,
                const float* d_weight, const quasar_policy_params* params, float* d_logprob, float* d_entropy,
                float* d_row_loss, float* d_loss, void* d_grad, int64_t grad_ld, void* stream) {
    if (!params || !d_loss) return QUASAR_EINVAL;
    if (!check_rows(d_logits, dtype, ld, rows, V, d_targets, params->temperature)) return QUASAR_EINVAL;
    if (!(params->clip_low >= 0.0f) || !(params->clip_high >= 0.0f) || !isfinite(params->kl_coef) ||
        !isfinite(params->entropy_coef) || !isfinite(params->grad_scale))
        return QUASAR_EINVAL;
    if (d_grad && !check_grad(d_logits, dtype, ld, rows, V, d_grad, grad_ld)) return QUASAR_EINVAL;
    const cudaStream_t st = (cudaStream_t)stream;
    if (rows > 0) {
        if (!d_old_logprob || !d_advantage || !d_logprob || !d_row_loss) return QUASAR_EINVAL;
        if (params->kl_coef != 0.0f && !d_ref_logprob) return QUASAR_EINVAL;
        qs::loss::Args a = row_args(d_logits, ld, rows, V, d_targets, params->temperature);
        a.logprob = d_logprob;
        a.entropy = d_entropy;
        a.old_lp = d_old_logprob;
        a.adv = d_advantage;
        a.ref_lp = d_ref_logprob;
        a.weight = d_weight;
        a.mean = 1.0 / rows;
        a.clip_lo = params->clip_low;
        a.clip_hi = params->clip_high;
        a.kl = params->kl_coef;
        a.ec = params->entropy_coef;
        a.row_loss = d_row_loss;
        a.scale = params->grad_scale;
        a.grad = d_grad;
        a.grad_ld = grad_ld;
        a.selftest = selftest;
        const int rc = status(qs::loss::launch_rows(a, dtype, st));
        if (rc != QUASAR_OK) return rc;
    }
    return status(qs::loss::launch_weighted_sum(d_row_loss, d_weight, rows, d_loss, st));
}

}  // namespace

extern "C" {

int quasar_token_logprobs(const void* d_logits, int dtype, int64_t ld, int rows, int V, const int32_t* d_targets,
                          float temperature, float* d_logprob, float* d_entropy, quasar_logprob_stat* d_stats,
                          void* stream) {
    if (!check_rows(d_logits, dtype, ld, rows, V, d_targets, temperature)) return QUASAR_EINVAL;
    if (rows == 0) return QUASAR_OK;
    if (!d_logprob) return QUASAR_EINVAL;
    qs::loss::Args a = row_args(d_logits, ld, rows, V, d_targets, temperature);
    a.logprob = d_logprob;
    a.entropy = d_entropy;
    a.stats = d_stats;
    return status(qs::loss::launch_rows(a, dtype, (cudaStream_t)stream));
}

int quasar_token_logprobs_grad(const void* d_logits, int dtype, int64_t ld, int rows, int V, const int32_t* d_targets,
                               float temperature, const quasar_logprob_stat* d_stats, const float* d_entropy,
                               const float* d_grad_logprob, const float* d_grad_entropy, void* d_grad, int64_t grad_ld,
                               void* stream) {
    if (!check_rows(d_logits, dtype, ld, rows, V, d_targets, temperature)) return QUASAR_EINVAL;
    if (!check_grad(d_logits, dtype, ld, rows, V, d_grad, grad_ld)) return QUASAR_EINVAL;
    if (rows == 0) return QUASAR_OK;
    if (!d_stats || !d_grad_logprob || !d_entropy != !d_grad_entropy) return QUASAR_EINVAL;
    qs::loss::Args a = row_args(d_logits, ld, rows, V, d_targets, temperature);
    a.stats_in = d_stats;
    a.ent_in = d_entropy;
    a.g_lp = d_grad_logprob;
    a.g_ent = d_grad_entropy;
    a.grad = d_grad;
    a.grad_ld = grad_ld;
    return status(qs::loss::launch_grad(a, dtype, (cudaStream_t)stream));
}

int quasar_policy_loss(const void* d_logits, int dtype, int64_t ld, int rows, int V, const int32_t* d_targets,
                       const float* d_old_logprob, const float* d_advantage, const float* d_ref_logprob,
                       const float* d_weight, const quasar_policy_params* params, float* d_logprob, float* d_entropy,
                       float* d_row_loss, float* d_loss, void* d_grad, int64_t grad_ld, void* stream) {
    return policy_loss(0, d_logits, dtype, ld, rows, V, d_targets, d_old_logprob, d_advantage, d_ref_logprob,
                       d_weight, params, d_logprob, d_entropy, d_row_loss, d_loss, d_grad, grad_ld, stream);
}

int quasar_selftest_stalled_policy_loss(int64_t wait_cycles, int chunks, const void* d_logits, int dtype, int64_t ld,
                                        int rows, int V, const int32_t* d_targets, const float* d_old_logprob,
                                        const float* d_advantage, const float* d_ref_logprob, const float* d_weight,
                                        const quasar_policy_params* params, float* d_logprob, float* d_entropy,
                                        float* d_row_loss, float* d_loss, void* d_grad, int64_t grad_ld, void* stream) {
    if (wait_cycles < 0 || wait_cycles > qs::WAIT_CYCLES || chunks < 0) return QUASAR_EINVAL;
    uint32_t bits = 0;
    while ((2ll << bits) <= wait_cycles) bits++;
    const uint32_t most = 0xFFFFFEu, stop = (uint32_t)chunks < most ? (uint32_t)chunks : most;
    return policy_loss(bits << 24 | (stop + 1), d_logits, dtype, ld, rows, V, d_targets, d_old_logprob, d_advantage, d_ref_logprob,
                       d_weight, params, d_logprob, d_entropy, d_row_loss, d_loss, d_grad, grad_ld, stream);
}

int quasar_preference_loss(const void* d_logits, int dtype, int64_t ld, int rows, int V, const int32_t* d_targets,
                           const int32_t* d_cu_seqlens, int pairs, const float* d_ref_logprob,
                           const float* d_pair_weight, const quasar_preference_params* params, float* d_logprob,
                           float* d_seq_logprob, float* d_pair_loss, float* d_loss, quasar_logprob_stat* d_stats,
                           float* d_row_grad, void* d_grad, int64_t grad_ld, void* stream) {
    if (!params || !d_loss || pairs < 0) return QUASAR_EINVAL;
    if (!check_rows(d_logits, dtype, ld, rows, V, d_targets, params->temperature)) return QUASAR_EINVAL;
    if (!isfinite(params->beta) || !(params->label_smoothing >= 0.0f && params->label_smoothing <= 1.0f) ||
        !isfinite(params->grad_scale))
        return QUASAR_EINVAL;
    if (d_grad && !check_grad(d_logits, dtype, ld, rows, V, d_grad, grad_ld)) return QUASAR_EINVAL;
    if (rows > 0 && (!d_logprob || !d_stats || !d_row_grad)) return QUASAR_EINVAL;
    if (pairs > 0 && (!d_cu_seqlens || !d_seq_logprob || !d_pair_loss)) return QUASAR_EINVAL;
    if (pairs > INT32_MAX / 4) return QUASAR_EINVAL;
    const cudaStream_t st = (cudaStream_t)stream;
    qs::loss::Args a = row_args(d_logits, ld, rows, V, d_targets, params->temperature);
    int rc = QUASAR_OK;
    if (rows > 0) {
        a.logprob = d_logprob;
        a.stats = d_stats;
        a.row_grad = d_row_grad;
        rc = status(qs::loss::launch_rows(a, dtype, st));
    }
    if (rc == QUASAR_OK) {
        qs::loss::PairArgs p;
        memset(&p, 0, sizeof p);
        p.logprob = d_logprob;
        p.targets = d_targets;
        p.cu = d_cu_seqlens;
        p.pairs = pairs;
        p.rows = rows;
        p.ref = d_ref_logprob;
        p.beta = params->beta;
        p.eps = params->label_smoothing;
        p.scale = params->grad_scale;
        p.mean = params->length_normalize != 0;
        p.weight = d_pair_weight;
        p.seq = d_seq_logprob;
        p.pair_loss = d_pair_loss;
        p.row_grad = d_row_grad;
        rc = status(qs::loss::launch_pairs(p, d_loss, st));
    }
    if (rc == QUASAR_OK && rows > 0 && d_grad) {
        a.stats_in = d_stats;
        a.g_lp = d_row_grad;
        a.grad = d_grad;
        a.grad_ld = grad_ld;
        rc = status(qs::loss::launch_grad(a, dtype, st));
    }
    return rc;
}

}  // extern "C"
