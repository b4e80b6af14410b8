// learn_api.cpp - the C ABI of the operators that train a draft head: the layer norm with its backward pass and
// distillation.  Checks of arguments and the launches.
//
// A descriptor is looked at before the sampler is: what is wrong with a call is said the same way
// with or without a device.
#include <cmath>
#include <cstdint>

#include "../../include/lily_sampler.h"
#include "operators.h"
#include "operators_check.h"

using namespace lily;

namespace {

int check_layer_size(uint32_t rows, uint32_t d) {
    if (rows == 0u || d == 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows and d must be positive");
    }
    if (d > LILY_NORM_MAX_D) {
        return api_fail(LILY_ERR_RANGE, "a norm takes rows of up to %u elements", LILY_NORM_MAX_D);
    }
    if (rows > MAX_THREADS / norm_shape(d).threads) {
        return api_fail(LILY_ERR_RANGE, "a norm takes up to %u rows of %u elements", MAX_THREADS / norm_shape(d).threads, d);
    }
    return LILY_OK;
}

int check_layer(const lily_layer* n) {
    if (n == nullptr || n->x_dev == nullptr || n->out_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "layer, x and out are required");
    }
    if (int rc = check_layer_size(n->rows, n->d)) {
        return rc;
    }
    if (n->x_dtype > LILY_BF16 || n->stream_dtype > LILY_BF16 || n->weight_dtype > LILY_BF16) {
        return api_fail(LILY_ERR_INVALID_ARG, "x, residual, weight and bias are LILY_F32 or LILY_BF16");
    }
    if (n->out_dtype > LILY_E4M3) {
        return api_fail(LILY_ERR_INVALID_ARG, "out is LILY_F32, LILY_BF16 or LILY_E4M3");
    }
    if ((n->out_dtype == LILY_E4M3) != (n->scales_dev != nullptr)) {
        return api_fail(LILY_ERR_INVALID_ARG, "scales come with an E4M3 out, and only there");
    }
    if ((n->scale_block != 0u && n->scale_block != LILY_BLOCK) || (n->scale_block != 0u && n->out_dtype != LILY_E4M3)) {
        return api_fail(LILY_ERR_INVALID_ARG, "scale_block is 0 or, with an E4M3 out, LILY_BLOCK");
    }
    if (n->sum_dev != nullptr && n->residual_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "a sum needs a residual");
    }
    if (!(std::isfinite(n->eps) && n->eps >= 0.0f)) {
        return api_fail(LILY_ERR_INVALID_ARG, "eps must be finite and >= 0");
    }
    const uint32_t blocks = (n->d + LILY_BLOCK - 1u) / LILY_BLOCK;
    if (n->rows > 1u && (n->x_stride < n->d || n->out_stride < n->d || (n->residual_dev != nullptr && n->residual_stride < n->d) ||
                         (n->sum_dev != nullptr && n->sum_stride < n->d) || (n->scale_block != 0u && n->scales_stride < blocks))) {
        return api_fail(LILY_ERR_INVALID_ARG, "a stride is shorter than its row");
    }
    const Span x = span(n->x_dev, n->rows, n->d, n->x_stride, n->x_dtype);
    const Span res = span(n->residual_dev, n->rows, n->d, n->residual_stride, n->stream_dtype);
    const Span sum = span(n->sum_dev, n->rows, n->d, n->sum_stride, n->stream_dtype);
    const Span out = span(n->out_dev, n->rows, n->d, n->out_stride, n->out_dtype);
    const Span w = span(n->weight_dev, 1, n->d, n->d, n->weight_dtype);
    const Span bias = span(n->bias_dev, 1, n->d, n->d, n->weight_dtype);
    const Span scales = n->scale_block == 0u ? span(n->scales_dev, 1, n->rows, n->rows, LILY_F32)
                                             : span(n->scales_dev, n->rows, blocks, n->scales_stride, LILY_F32);
    const Span mean = span(n->mean_dev, 1, n->rows, n->rows, LILY_F32);
    const Span rstd = span(n->rstd_dev, 1, n->rows, n->rows, LILY_F32);
    if (int rc = check_places({&x, &res, &sum, &out, &w, &bias, &scales, &mean, &rstd})) {
        return rc;
    }
    for (const Span* o : {&sum, &out}) {
        for (const Span* i : {&x, &res}) {
            if (overlap(*o, *i) && !same(*o, *i)) {
                return api_fail(LILY_ERR_INVALID_ARG, "an output overlaps an input without being it");
            }
        }
    }
    const Span* outputs[] = {&sum, &out, &scales, &mean, &rstd};
    for (int a = 0; a < 5; ++a) {
        if (overlap(*outputs[a], w) || overlap(*outputs[a], bias)) {
            return api_fail(LILY_ERR_INVALID_ARG, "an output overlaps weight or bias");
        }
        if (a >= 2 && (overlap(*outputs[a], x) || overlap(*outputs[a], res))) {
            return api_fail(LILY_ERR_INVALID_ARG, "scales, mean or rstd overlap an input");
        }
        for (int b = a + 1; b < 5; ++b) {
            if (overlap(*outputs[a], *outputs[b])) {
                return api_fail(LILY_ERR_INVALID_ARG, "two outputs overlap");
            }
        }
    }
    return LILY_OK;
}

int check_layer_grad(const lily_layer_grad* n) {
    if (n == nullptr || n->grad_dev == nullptr || n->h_dev == nullptr || n->mean_dev == nullptr || n->rstd_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "layer_grad, grad, h, mean and rstd are required");
    }
    if (n->grad_x_dev == nullptr && n->grad_weight_dev == nullptr && n->grad_bias_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "nothing is asked for");
    }
    if (int rc = check_layer_size(n->rows, n->d)) {
        return rc;
    }
    if (n->grad_dtype > LILY_BF16 || n->h_dtype > LILY_BF16 || n->weight_dtype > LILY_BF16 || n->grad_x_dtype > LILY_BF16) {
        return api_fail(LILY_ERR_INVALID_ARG, "grad, h, weight, past and grad_x are LILY_F32 or LILY_BF16");
    }
    if (n->past_dev != nullptr && n->grad_x_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "past needs a grad_x");
    }
    if (n->accumulate > 1u) {
        return api_fail(LILY_ERR_INVALID_ARG, "accumulate is 0 or 1");
    }
    if (n->rows > 1u && (n->grad_stride < n->d || n->h_stride < n->d || (n->past_dev != nullptr && n->past_stride < n->d) ||
                         (n->grad_x_dev != nullptr && n->grad_x_stride < n->d))) {
        return api_fail(LILY_ERR_INVALID_ARG, "a stride is shorter than d");
    }
    const Span grad = span(n->grad_dev, n->rows, n->d, n->grad_stride, n->grad_dtype);
    const Span h = span(n->h_dev, n->rows, n->d, n->h_stride, n->h_dtype);
    const Span mean = span(n->mean_dev, 1, n->rows, n->rows, LILY_F32);
    const Span rstd = span(n->rstd_dev, 1, n->rows, n->rows, LILY_F32);
    const Span w = span(n->weight_dev, 1, n->d, n->d, n->weight_dtype);
    const Span past = span(n->past_dev, n->rows, n->d, n->past_stride, n->grad_x_dtype);
    const Span gx = span(n->grad_x_dev, n->rows, n->d, n->grad_x_stride, n->grad_x_dtype);
    const Span gw = span(n->grad_weight_dev, 1, n->d, n->d, LILY_F32);
    const Span gb = span(n->grad_bias_dev, 1, n->d, n->d, LILY_F32);
    if (int rc = check_places({&grad, &h, &mean, &rstd, &w, &past, &gx, &gw, &gb})) {
        return rc;
    }
    for (const Span* i : {&grad, &h, &past}) {
        if (overlap(gx, *i) && !same(gx, *i)) {
            return api_fail(LILY_ERR_INVALID_ARG, "grad_x overlaps an input without being it");
        }
    }
    for (const Span* i : {&mean, &rstd, &w}) {
        if (overlap(gx, *i)) {
            return api_fail(LILY_ERR_INVALID_ARG, "grad_x overlaps mean, rstd or the weights");
        }
    }
    for (const Span* o : {&gw, &gb}) {
        for (const Span* i : {&grad, &h, &mean, &rstd, &w, &past, &gx}) {
            if (overlap(*o, *i)) {
                return api_fail(LILY_ERR_INVALID_ARG, "a gradient of weight or bias overlaps another array");
            }
        }
    }
    if (overlap(gw, gb)) {
        return api_fail(LILY_ERR_INVALID_ARG, "the gradients of weight and bias overlap");
    }
    return LILY_OK;
}

int check_distillation(const lily_distillation* d, bool backward) {
    if (d == nullptr || d->logits_dev == nullptr || d->ids_dev == nullptr || d->values_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "distillation, logits, ids and values are required");
    }
    if (backward && (d->stats_dev == nullptr || d->grad_dev == nullptr)) {
        return api_fail(LILY_ERR_INVALID_ARG, "the backward pass requires stats and grad");
    }
    if (backward && d->loss_dev != nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "the backward pass has no loss");
    }
    if (!backward && d->loss_dev == nullptr && d->stats_dev == nullptr && d->grad_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "nothing is asked for");
    }
    if (d->rows == 0u || d->vocab == 0u || d->k == 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows, vocab and k must be positive");
    }
    if (d->vocab > (1u << 24)) {
        return api_fail(LILY_ERR_RANGE, "distillation takes vocabularies up to 2^24");
    }
    if (d->k > LILY_SAMPLE_K_CAP) {
        return api_fail(LILY_ERR_RANGE, "a teacher's list holds up to %u entries", LILY_SAMPLE_K_CAP);
    }
    if (d->logits_dtype > LILY_BF16 || d->values_dtype > LILY_BF16 || d->grad_dtype > LILY_BF16) {
        return api_fail(LILY_ERR_INVALID_ARG, "logits, values and grad are LILY_F32 or LILY_BF16");
    }
    if (d->teacher > LILY_TEACHER_PROBS || d->rest > 1u) {
        return api_fail(LILY_ERR_INVALID_ARG, "teacher is LILY_TEACHER_LOGITS or LILY_TEACHER_PROBS, rest 0 or 1");
    }
    if ((d->teacher == LILY_TEACHER_LOGITS && d->rest != 0u) != (d->teacher_lse_dev != nullptr)) {
        return api_fail(LILY_ERR_INVALID_ARG, "teacher_lse comes with logits and rest, and only there");
    }
    // (below 2^-126 log2(e) / T is none of f32's)
    if (!(std::isfinite(d->temperature) && d->temperature >= 0x1p-126f) || !std::isfinite(d->grad_scale)) {
        return api_fail(LILY_ERR_INVALID_ARG, "temperature must be finite and at least 2^-126, grad_scale finite");
    }
    if (d->rows > 1u && (d->logits_stride < d->vocab || d->ids_stride < d->k || d->values_stride < d->k ||
                         (d->grad_dev != nullptr && d->grad_stride < d->vocab))) {
        return api_fail(LILY_ERR_INVALID_ARG, "a stride is shorter than its row");
    }
    const Span z = span(d->logits_dev, d->rows, d->vocab, d->logits_stride, d->logits_dtype);
    const Span ids = span(d->ids_dev, d->rows, d->k, d->ids_stride, LILY_F32);
    const Span values = span(d->values_dev, d->rows, d->k, d->values_stride, d->values_dtype);
    const Span counts = span(d->counts_dev, 1, d->rows, d->rows, LILY_F32);
    const Span tl = span(d->teacher_lse_dev, 1, d->rows, d->rows, LILY_F32);
    const Span weights = span(d->row_weights_dev, 1, d->rows, d->rows, LILY_F32);
    const Span loss = span(d->loss_dev, 1, d->rows, d->rows, LILY_F32);
    const Span stats = span(d->stats_dev, 1, d->rows * 4ull, d->rows * 4ull, LILY_F32);
    const Span grad = span(d->grad_dev, d->rows, d->vocab, d->grad_stride, d->grad_dtype);
    if (int rc = check_places({&z, &ids, &values, &counts, &tl, &weights, &loss, &stats, &grad})) {
        return rc;
    }
    if (overlap(grad, z) && !same(grad, z)) {
        return api_fail(LILY_ERR_INVALID_ARG, "grad overlaps the logits without being them");
    }
    for (const Span* o : {&grad, &loss, &stats}) {
        for (const Span* i : {&ids, &values, &counts, &tl, &weights}) {
            if (overlap(*o, *i)) {
                return api_fail(LILY_ERR_INVALID_ARG, "an output overlaps an input");
            }
        }
    }
    if (overlap(loss, z) || overlap(stats, z) || overlap(grad, loss) || overlap(grad, stats) || overlap(loss, stats)) {
        return api_fail(LILY_ERR_INVALID_ARG, "loss, stats and another array overlap");
    }
    return LILY_OK;
}

int distill(lily_sampler_t* s, const lily_distillation* d, bool backward) {
    if (int rc = check_distillation(d, backward)) {
        return rc;
    }
    if (int rc = need_sampler(s)) {
        return rc;
    }
    ON_DEVICE(sampler_device(s));
    ProjectWorkspace ws;
    sampler_project_workspace(s, &ws);
    HIP_TRY(launch_distill(sampler_stream(s), *d, backward, ws));
    return LILY_OK;
}

}  // namespace

extern "C" {

int lily_layer_norm(lily_sampler_t* s, const lily_layer* layer) {
    if (int rc = check_layer(layer)) {
        return rc;
    }
    if (int rc = need_sampler(s)) {
        return rc;
    }
    ON_DEVICE(sampler_device(s));
    HIP_TRY(launch_layer_norm(sampler_stream(s), *layer));
    return LILY_OK;
}

int lily_layer_norm_backward(lily_sampler_t* s, const lily_layer_grad* grad) {
    if (int rc = check_layer_grad(grad)) {
        return rc;
    }
    if (int rc = need_sampler(s)) {
        return rc;
    }
    ON_DEVICE(sampler_device(s));
    ProjectWorkspace ws;
    sampler_project_workspace(s, &ws);
    HIP_TRY(launch_layer_norm_backward(sampler_stream(s), *grad, ws));
    return LILY_OK;
}

int lily_distill(lily_sampler_t* s, const lily_distillation* d) { return distill(s, d, false); }

int lily_distill_backward(lily_sampler_t* s, const lily_distillation* d) { return distill(s, d, true); }

}  // extern "C"
