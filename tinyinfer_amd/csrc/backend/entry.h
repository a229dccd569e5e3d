// What the C entries without a context share: refusals, the stream's device
// and errors.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <new>
#include <string>

#include "../../../include/mp_hip.h"

namespace mphip {

void set_free_error(const std::string& message);

inline int refuse_call(const char* message) {
    set_free_error(message);
    return MP_INVALID_ARGUMENT;
}

// Makes the device of a caller's stream current for a call's launches.
class StreamDevice {
public:
    explicit StreamDevice(hipStream_t s) {
        // The null, legacy and per-thread streams belong to the current device.
        if (reinterpret_cast<uintptr_t>(s) <= 2) return;
        hipDevice_t wanted = 0;
        int current = 0;
        status = hipStreamGetDevice(s, &wanted);
        if (status == hipSuccess) status = hipGetDevice(&current);
        if (status != hipSuccess || wanted == current) return;
        status = hipSetDevice(wanted);
        if (status == hipSuccess) previous_ = current;
    }
    ~StreamDevice() {
        if (previous_ >= 0) (void)hipSetDevice(previous_);
    }
    StreamDevice(const StreamDevice&) = delete;
    StreamDevice& operator=(const StreamDevice&) = delete;
    hipError_t status = hipSuccess;

private:
    int previous_ = -1;
};

inline int call_done(hipError_t e, const char* what) {
    if (e == hipSuccess) return MP_OK;
    set_free_error(std::string(what) + ": " + hipGetErrorString(e));
    return MP_DEVICE_ERROR;
}

// No exception leaves a C entry.
template <typename Body>
int c_entry(Body body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return MP_OUT_OF_MEMORY;
    } catch (...) {
        return MP_DEVICE_ERROR;
    }
}

}  // namespace mphip
