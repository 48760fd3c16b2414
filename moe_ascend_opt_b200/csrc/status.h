// Error reporting shared by the C ABI's translation units (include/moe_b200.h).
#pragma once
#include <cuda_runtime.h>

#include <string>

#include "../../include/moe_b200.h"

namespace moe {
// Sets moe_last_error() of the calling thread and returns `code`.
int fail(int code, const std::string& msg);
}  // namespace moe

#define CUDA_TRY(expr)                                                                              \
    do {                                                                                            \
        cudaError_t _e = (expr);                                                                    \
        if (_e != cudaSuccess)                                                                      \
            return moe::fail(MOE_ERR_CUDA, std::string(#expr) + ": " + cudaGetErrorString(_e)); \
    } while (0)
