// The context behind the C ABI's opaque handle, shared by the files that
// implement its entry points.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "gemm_internal.h"

struct sn_context {
    int device = 0;
    hipStream_t stream = nullptr;
    uint32_t kernel = SN_KERNEL_MFMA_F32;
    sn::Env env;
};
