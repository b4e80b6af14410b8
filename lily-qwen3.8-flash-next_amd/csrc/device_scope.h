// device_scope.h - a library call works on its object's device and leaves the calling thread on the
// one it came with.
#pragma once

#include <hip/hip_runtime_api.h>

namespace lily {

// Makes `device` the calling thread's current device for the rest of the enclosing scope and
// puts the caller's own choice back on the way out: a library call must not leave the host
// thread on another GPU than it came with.
struct DeviceScope {
    int before = -1;
    bool switched = false;
    hipError_t err = hipSuccess;
    explicit DeviceScope(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) {
            err = hipSetDevice(device);
            switched = err == hipSuccess;
        }
    }
    ~DeviceScope() {
        if (switched) {
            (void)hipSetDevice(before);
        }
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

}  // namespace lily
