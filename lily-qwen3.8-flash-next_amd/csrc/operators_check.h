// operators_check.h - what the entry points of the operators share: runtime calls that may fail, a call's device, its
// operands as memory.
#pragma once

#include <hip/hip_runtime_api.h>

#include <initializer_list>

#include "api_internal.h"
#include "device_scope.h"
#include "operand_span.h"

namespace lily {

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

inline int need_sampler(const lily_sampler_t* s) {
    return s != nullptr ? LILY_OK : api_fail(LILY_ERR_INVALID_ARG, "sampler is null");
}

// Every operand lies within the address space and starts at one of its elements.
inline int check_places(std::initializer_list<const Span*> spans) {
    for (const Span* s : spans) {
        if (!fits(*s)) {
            return api_fail(LILY_ERR_RANGE, "rows and strides reach beyond the address space");
        }
        if (s->rows != 0u && (s->at % size_of(s->dtype) != 0u)) {
            return api_fail(LILY_ERR_INVALID_ARG, "an array does not start at a multiple of its element's size");
        }
    }
    return LILY_OK;
}

}  // namespace lily
