// What every operator dispatcher does around its checks: element types, stream, launch errors.
#pragma once

#include "ops.hpp"

#include "../core/core.hpp"
#include "../device/runtime_api.hpp"
#include "../kernels/launch.hpp"
#include "../utils/check.hpp"
#include "../utils/types.hpp"

namespace llaisys::ops {

inline bool isFloat(llaisysDataType_t dt) {
    return dt == LLAISYS_DTYPE_F32 || dt == LLAISYS_DTYPE_BF16 || dt == LLAISYS_DTYPE_F16;
}

inline void requireFloat(llaisysDataType_t dt) {
    if (!isFloat(dt)) EXCEPTION_UNSUPPORTED_DATATYPE(dt);
}

// Makes the device of `t` current and returns its stream; only the AMD device computes.
inline hipStream_t streamFor(const tensor_t &t) {
    if (t->deviceType() != LLAISYS_DEVICE_AMD) EXCEPTION_UNSUPPORTED_DEVICE;
    auto &ctx = core::context();
    ctx.setDevice(t->deviceType(), t->deviceId());
    return static_cast<hipStream_t>(ctx.runtime().stream());
}

// Reports a failed launch (bad configuration, no code object for this GPU) at the call.
inline void launched(const char *op) { device::amd::check(hipGetLastError(), op); }

// Byte ranges of two contiguous tensors intersect.
inline bool overlaps(const tensor_t &a, const tensor_t &b) {
    const std::byte *a0 = a->data(), *b0 = b->data();
    return a0 < b0 + b->numel() * b->elementSize() && b0 < a0 + a->numel() * a->elementSize();
}

} // namespace llaisys::ops
