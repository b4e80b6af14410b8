// operators_api.cpp - the C ABI of the operators around the head: checks of arguments and one launch.
//
// A descriptor is looked at before the sampler is: what is wrong with a call is said the same way
// with or without a device.
#include <cmath>
#include <cstdint>

#include "../../include/lily_sampler.h"
#include "api_internal.h"
#include "device_scope.h"
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

// An operand as memory: `rows` rows of `width` bytes, `stride` bytes apart.
struct Span {
    uint64_t at = 0, rows = 0, width = 0, stride = 0;
    uint32_t dtype = 0;
};

uint64_t size_of(uint32_t dtype) { return dtype == LILY_F32 ? 4u : dtype == LILY_BF16 ? 2u : 1u; }

Span span(const void* p, uint64_t rows, uint64_t columns, uint64_t stride, uint32_t dtype) {
    const uint64_t e = size_of(dtype);
    Span s;
    s.at = reinterpret_cast<uintptr_t>(p);
    s.rows = p != nullptr ? rows : 0u;
    s.width = columns * e;
    s.stride = rows > 1u ? stride * e : columns * e;   // (one row: its stride says nothing)
    s.dtype = dtype;
    return s;
}

bool aligned(const Span& s) { return s.rows == 0u || (s.at % 16u == 0u && s.stride % 16u == 0u); }

// The last byte behind a span must be an address.
bool fits(const Span& s) {
    if (s.rows == 0u) {
        return true;
    }
    const unsigned __int128 end = (unsigned __int128)s.at + (unsigned __int128)(s.rows - 1u) * s.stride + s.width;
    return end <= (unsigned __int128)1 << 63;
}

// Whether two operands share a byte.  Rows of one stride are compared within it, so that columns of a
// wider buffer side by side are apart; otherwise the whole ranges are.
bool overlap(const Span& a, const Span& b) {
    if (a.rows == 0u || b.rows == 0u) {
        return false;
    }
    const uint64_t end_a = a.at + (a.rows - 1u) * a.stride + a.width, end_b = b.at + (b.rows - 1u) * b.stride + b.width;
    if (end_a <= b.at || end_b <= a.at) {
        return false;
    }
    if (a.stride == b.stride && a.rows > 1u && b.rows > 1u) {
        const uint64_t s = a.stride, off = b.at >= a.at ? (b.at - a.at) % s : (s - (a.at - b.at) % s) % s;
        return !(off >= a.width && off + b.width <= s);
    }
    return true;
}

// An output may be an input itself: then every element is read by the thread that writes it, or a
// row is read whole before any of it is written.
bool same(const Span& a, const Span& b) {
    return a.at == b.at && a.dtype == b.dtype && a.stride == b.stride && a.width == b.width;
}

int check_norm(const lily_norm* n, bool* pieces) {
    if (n == nullptr || n->x_dev == nullptr || n->out_dev == nullptr) {
        return api_fail(LILY_ERR_INVALID_ARG, "norm, x and out are required");
    }
    if (n->rows == 0u || n->d == 0u) {
        return api_fail(LILY_ERR_INVALID_ARG, "rows and d must be positive");
    }
    if (n->d > LILY_NORM_MAX_D || n->rows > 0x7fffffffu) {
        return api_fail(LILY_ERR_RANGE, "a norm takes rows of up to %u elements, 2^31 - 1 of them", LILY_NORM_MAX_D);
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
    *pieces = n->d % 8u == 0u && aligned(x) && aligned(res) && aligned(sum) && w.at % 16u == 0u &&
              out.at % (n->out_dtype == LILY_E4M3 ? 8u : 16u) == 0u &&
              out.stride % (n->out_dtype == LILY_E4M3 ? 8u : 16u) == 0u;
    return LILY_OK;
}

int need_sampler(const lily_sampler_t* s) {
    return s != nullptr ? LILY_OK : api_fail(LILY_ERR_INVALID_ARG, "sampler is null");
}

}  // namespace

extern "C" {

int lily_rms_norm(lily_sampler_t* s, const lily_norm* norm) {
    bool pieces = false;
    if (int rc = check_norm(norm, &pieces)) {
        return rc;
    }
    if (int rc = need_sampler(s)) {
        return rc;
    }
    ON_DEVICE(sampler_device(s));
    HIP_TRY(launch_rms_norm(sampler_stream(s), *norm, pieces));
    return LILY_OK;
}

}  // extern "C"
