/*
 * mzs_error.h — the library's error channel (mzs_last_error) and current-device handling for the kernel units
 * outside mzsearch.hip.
 */
#ifndef MZS_ERROR_H
#define MZS_ERROR_H

#include <hip/hip_runtime.h>

#include <cstdio>

#include "../../include/mzsearch.h"

namespace mzs {

/* stores the text mzs_last_error() returns on this thread; returns `code` (defined in mzsearch.hip, never throws) */
int set_error(int code, const char* text) noexcept;

inline int hip_error(const char* what, hipError_t e) noexcept {
    char text[256];
    std::snprintf(text, sizeof text, "%s: %s", what, hipGetErrorString(e));
    return set_error(MZS_E_HIP, text);
}

/* makes `device` current for a call and puts the caller's device back afterwards */
struct DeviceScope {
    int before = -1;
    hipError_t status;
    explicit DeviceScope(int device) noexcept {
        status = hipGetDevice(&before);
        if (status == hipSuccess && before != device) status = hipSetDevice(device);
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

}  // namespace mzs
#endif
