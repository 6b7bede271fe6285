// capi_check.hpp — argument checks of the C-ABI entry points (files that say
// `using namespace axf`).
#pragma once

#include "capi_internal.hpp"

#define AXF_CHECK_CTX(ctx) \
    if (!(ctx)) return fail(AXF_ERR_INVALID_ARG, std::string(__func__) + ": null context")
#define AXF_REQUIRE(cond, msg) \
    if (!(cond)) return fail(AXF_ERR_INVALID_ARG, std::string(__func__) + ": " + (msg))
#define AXF_HIP(call)                                          \
    do {                                                       \
        hipError_t e_ = (call);                                \
        if (e_ != hipSuccess) return hip_fail(e_, __func__);   \
    } while (0)

static inline bool aligned(const void* p, size_t a) {
    return (reinterpret_cast<uintptr_t>(p) % a) == 0;
}

namespace axf {

// Makes the context's device current for one call and puts the caller's back.
class DeviceScope {
  public:
    explicit DeviceScope(const axf_ctx* ctx) {
        if (hipGetDevice(&before_) == hipSuccess && before_ != ctx->device)
            set_ = hipSetDevice(ctx->device) == hipSuccess;
    }
    ~DeviceScope() {
        if (set_) (void)hipSetDevice(before_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;

  private:
    int before_ = -1;
    bool set_ = false;
};

}  // namespace axf
