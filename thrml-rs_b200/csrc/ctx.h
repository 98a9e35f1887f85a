// Device context shared by the translation units of the library, and the CUDA error-check macro.
#pragma once
#include <cuda_runtime.h>

#include <string>

#include "tables.h"

struct thrml_ctx {
    int device = 0;
    cudaStream_t stream = nullptr;
    int sm_count = 148;
    // Raised by a kernel on a caller's stream whose bounded wait ran out (0 = none), and up until the caller takes it down: every
    // stream and thread of the context learns of it.  Kernels only ever raise it, so that one's loss ends no other's waits.  Pinned host memory
    // that the device sees: the host reads it without waiting for any stream.
    int* wait_flag = nullptr;
    int* wait_flag_dev = nullptr;

    int32_t check_waits() const {
        if (!wait_flag) return THRML_OK;
        const int code = *static_cast<volatile int*>(wait_flag);
        if (code == 0) return THRML_OK;
        return thrml::fail(THRML_ERR_TIMEOUT, "a tensor-core kernel of an earlier call gave up waiting on a pipeline barrier (role " + std::to_string(code) +
                                                  ") and left its output unwritten; thrml_ctx_reset_waits takes this report down");
    }
};

#define CU_TRY(expr)                                                                                                      \
    do {                                                                                                                  \
        cudaError_t e__ = (expr);                                                                                         \
        if (e__ != cudaSuccess) return thrml::fail(THRML_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e__)); \
    } while (0)
