// What the operator registrations share: element types, the device and stream
// of a call, and the C ABI's return codes as exceptions.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <hip/hip_runtime_api.h>

#include "../../include/ple_hip.h"

namespace {

int ple_dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return PLE_DTYPE_F32;
        case at::kHalf: return PLE_DTYPE_F16;
        case at::kBFloat16: return PLE_DTYPE_BF16;
        default: return -1;
    }
}

// Makes `index` the current HIP device for the scope (the launch enqueues on
// that device's current stream).
class DeviceScope {
   public:
    explicit DeviceScope(c10::DeviceIndex index) {
        TORCH_CHECK(hipGetDevice(&prev_) == hipSuccess, "hipGetDevice failed");
        if (prev_ != index) {
            TORCH_CHECK(hipSetDevice(index) == hipSuccess, "hipSetDevice failed");
            changed_ = true;
        }
    }
    ~DeviceScope() {
        if (changed_) (void)hipSetDevice(prev_);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;

   private:
    int prev_ = 0;
    bool changed_ = false;
};

void check_rc(int rc, const char *what) {
    TORCH_CHECK(rc == PLE_OK, what, " failed: ", ple_error_string(rc), " (code ", rc, ")");
}

void *current_stream(const at::Tensor &t) {
    return static_cast<void *>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

}  // namespace
