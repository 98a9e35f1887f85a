// Device context shared by the translation units of the library, and the CUDA error-check macro.
#pragma once
#include <cuda_runtime.h>

#include <string>

#include "tables.h"

struct thrml_ctx {
    int device = 0;
    cudaStream_t stream = nullptr;
    int sm_count = 148;
    // Raised by a kernel on a caller's stream whose bounded wait ran out (0 = none).  Pinned host memory that the device sees:
    // the host reads it without waiting for any stream.
    int* wait_flag = nullptr;
    int* wait_flag_dev = nullptr;

    // The report of such a wait, once, by the first call that finds it.
    int32_t check_waits() {
        if (!wait_flag) return THRML_OK;
        const int code = *static_cast<volatile int*>(wait_flag);
        if (code == 0) return THRML_OK;
        *static_cast<volatile int*>(wait_flag) = 0;
        return thrml::fail(THRML_ERR_TIMEOUT, "a tensor-core kernel of an earlier call gave up waiting on a pipeline barrier (role " + std::to_string(code) + ")");
    }
};

#define CU_TRY(expr)                                                                                                      \
    do {                                                                                                                  \
        cudaError_t e__ = (expr);                                                                                         \
        if (e__ != cudaSuccess) return thrml::fail(THRML_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(e__)); \
    } while (0)
