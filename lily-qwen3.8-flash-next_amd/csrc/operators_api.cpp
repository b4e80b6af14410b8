// operators_api.cpp - the C ABI of the operators around the head: checks of arguments and one launch.
//
// A descriptor is looked at before the sampler is: what is wrong with a call is said the same way
// with or without a device.
#include <cmath>
#include <cstdint>

#include "../../include/lily_sampler.h"
#include "api_internal.h"
#include "device_scope.h"
#include "operand_span.h"
#include "operators.h"

using namespace lily;

namespace {

#define HIP_TRY(call)                                                                         \
    do {                                                                                      \
        hipError_t e_ = (call);                                                               \
        if (e_ != hipSuccess) {                                                               \
            return api_fail(LILY_ERR_HIP, "%s: %s", #call, hipGetErrorString(e_));            \
        }                                                                                     \
    } while (0)
#define ON_DEVICE(device)                 \
    DeviceScope device_scope_(device);    \
    HIP_TRY(device_scope_.err)

constexpr uint32_t MAX_THREADS = 0xffffffffu;   // of a launch

int check_norm(const lily_norm* n) {
    if (n == nullptr || n->x_dev == nullptr || n->out_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "norm, x and out are required");
    }
    if (n->rows == 0u || n->d == 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows and d must be positive");
    }
    if (n->d > LILY_NORM_MAX_D) {
        return api_fail(LILY_ERR_RANGE, "a norm takes rows of up to %u elements", LILY_NORM_MAX_D);
    }
    if (n->rows > MAX_THREADS / norm_shape(n->d).threads) {
        return api_fail(LILY_ERR_RANGE, "a norm takes up to %u rows of %u elements", MAX_THREADS / norm_shape(n->d).threads, n->d);
    }
    if (n->x_dtype > LILY_BF16 || n->stream_dtype > LILY_BF16 || n->weight_dtype > LILY_BF16) {
        return api_fail(LILY_ERR_INVALID_ARG, "x, residual and weight are LILY_F32 or LILY_BF16");
    }
    if (n->out_dtype > LILY_E4M3) {
        return api_fail(LILY_ERR_INVALID_ARG, "out is LILY_F32, LILY_BF16 or LILY_E4M3");
    }
    if ((n->out_dtype == LILY_E4M3) != (n->scales_dev != nullptr)) {
        return api_fail(LILY_ERR_INVALID_ARG, "scales come with an E4M3 out, and only there");
    }
    if (n->sum_dev != nullptr && n->residual_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "a sum needs a residual");
    }
    if (!(std::isfinite(n->eps) && n->eps >= 0.0f) || !std::isfinite(n->weight_offset)) {
        return api_fail(LILY_ERR_INVALID_ARG, "eps must be finite and >= 0, weight_offset finite");
    }
    if (n->weight_dev == nullptr && n->weight_offset != 0.0f) {
        return api_fail(LILY_ERR_INVALID_ARG, "weight_offset needs weights");
    }
    const bool one = n->rows == 1u;
    if (!one && (n->x_stride < n->d || n->out_stride < n->d || (n->residual_dev != nullptr && n->residual_stride < n->d) ||
                 (n->sum_dev != nullptr && n->sum_stride < n->d))) {
        return api_fail(LILY_ERR_INVALID_ARG, "a stride is shorter than d");
    }
    const Span x = span(n->x_dev, n->rows, n->d, n->x_stride, n->x_dtype);
    const Span res = span(n->residual_dev, n->rows, n->d, n->residual_stride, n->stream_dtype);
    const Span sum = span(n->sum_dev, n->rows, n->d, n->sum_stride, n->stream_dtype);
    const Span out = span(n->out_dev, n->rows, n->d, n->out_stride, n->out_dtype);
    const Span w = span(n->weight_dev, 1, n->d, n->d, n->weight_dtype);
    const Span scales = span(n->scales_dev, 1, n->rows, n->rows, LILY_F32);
    for (const Span* s : {&x, &res, &sum, &out, &w, &scales}) {
        if (!fits(*s)) {
            return api_fail(LILY_ERR_RANGE, "rows and strides reach beyond the address space");
        }
        if (s->rows != 0u && (s->at % size_of(s->dtype) != 0u)) {
            return api_fail(LILY_ERR_INVALID_ARG, "an array does not start at a multiple of its element's size");
        }
    }
    for (const Span* o : {&sum, &out}) {
        for (const Span* i : {&x, &res}) {
            if (overlap(*o, *i) && !same(*o, *i)) {
                return api_fail(LILY_ERR_INVALID_ARG, "an output overlaps an input without being it");
            }
        }
        if (overlap(*o, w) || overlap(*o, scales)) {
            return api_fail(LILY_ERR_INVALID_ARG, "an output overlaps the weights or the scales");
        }
    }
    for (const Span* i : {&x, &res, &w}) {
        if (overlap(scales, *i)) {
            return api_fail(LILY_ERR_INVALID_ARG, "the scales overlap an input");
        }
    }
    if (overlap(sum, out)) {
        return api_fail(LILY_ERR_INVALID_ARG, "sum and out overlap");
    }
    return LILY_OK;
}

int check_projection(const lily_projection* p) {
    if (p == nullptr || p->x_dev == nullptr || p->weight_dev == nullptr || p->out_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "projection, x, weight and out are required");
    }
    if (p->rows == 0u || p->n == 0u || p->d == 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows, n and d must be positive");
    }
    if (p->dtype != LILY_BF16 && p->dtype != LILY_E4M3) {
        return api_fail(LILY_ERR_INVALID_ARG, "x and weight are LILY_BF16 or LILY_E4M3");
    }
    if (p->bias_dtype > LILY_BF16 || p->residual_dtype > LILY_BF16 || p->out_dtype > LILY_BF16) {
        return api_fail(LILY_ERR_INVALID_ARG, "bias, residual and out are LILY_F32 or LILY_BF16");
    }
    if (p->activation > LILY_ACT_RELU) {
        return api_fail(LILY_ERR_INVALID_ARG, "unknown activation %u", p->activation);
    }
    const uint64_t e = size_of(p->dtype);
    if (p->d * e % 16u != 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "d must be a multiple of 16 bytes: of 8 in bf16, of 16 in E4M3");
    }
    if (p->d > 0xffffff80u / e || p->rows > (1u << 24) || p->n > (1u << 26)) {
        return api_fail(LILY_ERR_RANGE, "a product takes up to 2^24 rows, 2^26 outputs and rows of 2^32 - 128 bytes");
    }
    // (the smallest tile that many rows may get: 256 threads for 64 x 64)
    if (((p->rows + 63ull) / 64u) * ((p->n + 63ull) / 64u) > MAX_THREADS / 256u) {
        return api_fail(LILY_ERR_RANGE, "a product has up to 2^24 - 1 tiles of 64 x 64 outputs");
    }
    if ((p->rows > 1u && (p->x_stride < p->d || p->out_stride < p->n || (p->residual_dev != nullptr && p->residual_stride < p->n))) ||
        (p->n > 1u && p->weight_stride < p->d)) {
        return api_fail(LILY_ERR_INVALID_ARG, "a stride is shorter than its row");
    }
    const Span x = span(p->x_dev, p->rows, p->d, p->x_stride, p->dtype);
    const Span w = span(p->weight_dev, p->n, p->d, p->weight_stride, p->dtype);
    const Span out = span(p->out_dev, p->rows, p->n, p->out_stride, p->out_dtype);
    const Span res = span(p->residual_dev, p->rows, p->n, p->residual_stride, p->residual_dtype);
    const Span bias = span(p->bias_dev, 1, p->n, p->n, p->bias_dtype);
    const Span xs = span(p->x_scales_dev, 1, p->rows, p->rows, LILY_F32);
    const Span ws = span(p->weight_scales_dev, 1, p->n, p->n, LILY_F32);
    if (!aligned(x) || !aligned(w)) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows of x and weight must start at multiples of 16 bytes");
    }
    if ((p->rows > 1u && x.stride > (1u << 23)) || (p->n > 1u && w.stride > (1u << 23))) {
        return api_fail(LILY_ERR_RANGE, "rows of x and weight lie at most 2^23 bytes apart");
    }
    for (const Span* s : {&x, &w, &out, &res, &bias, &xs, &ws}) {
        if (!fits(*s)) {
            return api_fail(LILY_ERR_RANGE, "rows and strides reach beyond the address space");
        }
        if (s->rows != 0u && (s->at % size_of(s->dtype) != 0u)) {
            return api_fail(LILY_ERR_INVALID_ARG, "an array does not start at a multiple of its element's size");
        }
    }
    for (const Span* i : {&x, &w, &bias, &xs, &ws}) {
        if (overlap(out, *i)) {
            return api_fail(LILY_ERR_INVALID_ARG, "out overlaps an operand");
        }
    }
    if (overlap(out, res) && !same(out, res)) {
        return api_fail(LILY_ERR_INVALID_ARG, "out overlaps the residual without being it");
    }
    return LILY_OK;
}

int need_sampler(const lily_sampler_t* s) {
    return s != nullptr ? LILY_OK : api_fail(LILY_ERR_INVALID_ARG, "sampler is null");
}

}  // namespace

extern "C" {

int lily_rms_norm(lily_sampler_t* s, const lily_norm* norm) {
    if (int rc = check_norm(norm)) {
        return rc;
    }
    if (int rc = need_sampler(s)) {
        return rc;
    }
    ON_DEVICE(sampler_device(s));
    HIP_TRY(launch_rms_norm(sampler_stream(s), *norm));
    return LILY_OK;
}

int lily_project(lily_sampler_t* s, const lily_projection* p) {
    if (int rc = check_projection(p)) {
        return rc;
    }
    if (int rc = need_sampler(s)) {
        return rc;
    }
    ON_DEVICE(sampler_device(s));
    ProjectWorkspace ws;
    sampler_project_workspace(s, &ws);
    HIP_TRY(launch_project(sampler_stream(s), *p, ws));
    return LILY_OK;
}

}  // extern "C"
