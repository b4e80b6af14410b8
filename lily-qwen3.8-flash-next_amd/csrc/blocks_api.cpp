// blocks_api.cpp - the C ABI of 8-bit floats with a scale for each block: checks of arguments and the launches.
//
// A descriptor is looked at before the sampler is: what is wrong with a call is said the same way
// with or without a device.
#include <cstdint>

#include "../../include/lily_sampler.h"
#include "operators.h"
#include "operators_check.h"

using namespace lily;

namespace {

constexpr uint64_t blocks_of(uint64_t n) { return (n + LILY_BLOCK - 1u) / LILY_BLOCK; }

int check_blocks(const lily_blocks* q) {
    if (q == nullptr || q->x_dev == nullptr || q->out_dev == nullptr || q->scales_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "blocks, x, out and scales are required");
    }
    if (q->rows == 0u || q->d == 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows and d must be positive");
    }
    if (q->x_dtype > LILY_BF16) {
        return api_fail(LILY_ERR_INVALID_ARG, "x is LILY_F32 or LILY_BF16");
    }
    if (q->block_rows != 1u && q->block_rows != LILY_BLOCK) {
        return api_fail(LILY_ERR_INVALID_ARG, "block_rows is 1 or LILY_BLOCK");
    }
    // (what the kernels add to an element's place stays below 2^32)
    if (q->d > 0xffffff80u) {
        return api_fail(LILY_ERR_RANGE, "a call takes rows of up to 2^32 - 128 elements");
    }
    const uint64_t down = q->block_rows == 1u ? q->rows : blocks_of(q->rows), across = blocks_of(q->d);
    // (16 threads a block of a row, 256 a block of rows)
    if (down * across > MAX_THREADS / (q->block_rows == 1u ? 16u : 256u)) {
        return api_fail(LILY_ERR_RANGE, "a call takes up to 2^28 - 1 blocks of a row, 2^24 - 1 of rows");
    }
    if ((q->rows > 1u && (q->x_stride < q->d || q->out_stride < q->d)) || (down > 1u && q->scales_stride < across)) {
        return api_fail(LILY_ERR_INVALID_ARG, "a stride is shorter than its row");
    }
    const Span x = span(q->x_dev, q->rows, q->d, q->x_stride, q->x_dtype);
    const Span out = span(q->out_dev, q->rows, q->d, q->out_stride, LILY_E4M3);
    const Span scales = span(q->scales_dev, down, across, q->scales_stride, LILY_F32);
    if (int rc = check_places({&x, &out, &scales})) {
        return rc;
    }
    if (overlap(out, x) || overlap(scales, x) || overlap(out, scales)) {
        return api_fail(LILY_ERR_INVALID_ARG, "x, out and scales overlap");
    }
    return LILY_OK;
}

int check_block_projection(const lily_block_projection* p) {
    if (p == nullptr || p->x_dev == nullptr || p->weight_dev == nullptr || p->out_dev == nullptr || p->x_scales_dev == nullptr ||
        p->weight_scales_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "projection, x, weight, their scales and out are required");
    }
    if (p->rows == 0u || p->n == 0u || p->d == 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows, n and d must be positive");
    }
    if (p->bias_dtype > LILY_BF16 || p->residual_dtype > LILY_BF16 || p->out_dtype > LILY_BF16) {
        return api_fail(LILY_ERR_INVALID_ARG, "bias, residual and out are LILY_F32 or LILY_BF16");
    }
    if (p->activation > LILY_ACT_RELU) {
        return api_fail(LILY_ERR_INVALID_ARG, "unknown activation %u", p->activation);
    }
    if (p->reserved != 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "reserved must be 0");
    }
    if (p->d % 16u != 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "d must be a multiple of 16 bytes: of 16 elements");
    }
    if (p->d > 0xffffff80u || p->rows > (1u << 24) || p->n > (1u << 26)) {
        return api_fail(LILY_ERR_RANGE, "a product takes up to 2^24 rows, 2^26 outputs and rows of 2^32 - 128 bytes");
    }
    // (the smallest tile that many rows may get: 256 threads for 64 x 64)
    if (((p->rows + 63ull) / 64u) * ((p->n + 63ull) / 64u) > MAX_THREADS / 256u) {
        return api_fail(LILY_ERR_RANGE, "a product has up to 2^24 - 1 tiles of 64 x 64 outputs");
    }
    const uint64_t down = blocks_of(p->n), across = blocks_of(p->d);
    if ((p->rows > 1u && (p->x_stride < p->d || p->out_stride < p->n || (p->residual_dev != nullptr && p->residual_stride < p->n) ||
                          p->x_scales_stride < across)) ||
        (p->n > 1u && p->weight_stride < p->d) || (down > 1u && p->weight_scales_stride < across)) {
        return api_fail(LILY_ERR_INVALID_ARG, "a stride is shorter than its row");
    }
    const Span x = span(p->x_dev, p->rows, p->d, p->x_stride, LILY_E4M3);
    const Span w = span(p->weight_dev, p->n, p->d, p->weight_stride, LILY_E4M3);
    const Span out = span(p->out_dev, p->rows, p->n, p->out_stride, p->out_dtype);
    const Span res = span(p->residual_dev, p->rows, p->n, p->residual_stride, p->residual_dtype);
    const Span bias = span(p->bias_dev, 1, p->n, p->n, p->bias_dtype);
    const Span xs = span(p->x_scales_dev, p->rows, across, p->x_scales_stride, LILY_F32);
    const Span ws = span(p->weight_scales_dev, down, across, p->weight_scales_stride, LILY_F32);
    if (!aligned(x) || !aligned(w)) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows of x and weight must start at multiples of 16 bytes");
    }
    if ((p->rows > 1u && x.stride > (1u << 23)) || (p->n > 1u && w.stride > (1u << 23))) {
        return api_fail(LILY_ERR_RANGE, "rows of x and weight lie at most 2^23 bytes apart");
    }
    if ((p->rows > 1u && xs.stride > (1u << 23)) || (down > 1u && ws.stride > (1u << 23))) {
        return api_fail(LILY_ERR_RANGE, "rows of scales lie at most 2^23 bytes apart");
    }
    if (int rc = check_places({&x, &w, &out, &res, &bias, &xs, &ws})) {
        return rc;
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

}  // namespace

extern "C" {

int lily_quantize_blocks(lily_sampler_t* s, const lily_blocks* blocks) {
    if (int rc = check_blocks(blocks)) {
        return rc;
    }
    if (int rc = need_sampler(s)) {
        return rc;
    }
    ON_DEVICE(sampler_device(s));
    HIP_TRY(launch_quantize_blocks(sampler_stream(s), *blocks));
    return LILY_OK;
}

int lily_project_blocks(lily_sampler_t* s, const lily_block_projection* p) {
    if (int rc = check_block_projection(p)) {
        return rc;
    }
    if (int rc = need_sampler(s)) {
        return rc;
    }
    ON_DEVICE(sampler_device(s));
    ProjectWorkspace ws;
    sampler_project_workspace(s, &ws);
    HIP_TRY(launch_project_blocks(sampler_stream(s), *p, ws));
    return LILY_OK;
}

}  // extern "C"
