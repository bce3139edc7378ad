// What the host sources of the C ABI share: the engine and its error reports.
#pragma once

#include <cuda_runtime.h>

#include "../../include/splsage.h"

struct spl_sage {
    cudaStream_t stream;
    int head_dim;
    spl_sage_config config;
    int device;
    int sm_count;
    int reserved_sms;  // SMs the persistent kernels leave free (spl_sage_reserve_sms)
    int gemm_pairs;    // GEMMs on SM pairs (spl_sage_gemm_pairs)
    uint32_t* err;     // device error word of the calls that run without a workspace
};

namespace sp {

// Records the message that spl_sage_last_error returns on this thread, and
// returns the code.
int fail(int code, const char* fmt, ...);
int cuda_fail(cudaError_t e, const char* what);

}  // namespace sp
