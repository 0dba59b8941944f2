// Host-side error reporting shared by the library's translation units.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/aie_conv.h"

namespace aie {

// This thread's last failure (aie_last_error).
inline thread_local char t_err[512];

inline int fail(int status, const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(t_err, sizeof t_err, fmt, ap);
    va_end(ap);
    return status;
}

inline int cuda_fail(cudaError_t e, const char *what)
{
    return fail(AIE_E_CUDA, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

// Read and clear the sequence kernels' device error word (aie_seq.cu).
cudaError_t seq_take_device_error(uint32_t *code);

}  // namespace aie

#define CUDA_TRY(call)                                  \
    do {                                                \
        cudaError_t e_ = (call);                        \
        if (e_ != cudaSuccess) return aie::cuda_fail(e_, #call); \
    } while (0)
