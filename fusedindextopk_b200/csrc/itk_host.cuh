// Host-side helpers that the C-ABI translation units share: error reporting, argument checks and the
// driver's tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <mutex>
#include <string>

#include "../../include/itk_b200.h"

namespace itk {

// Message of the calling thread's last failure.
inline std::string& last_error() {
    static thread_local std::string message;
    return message;
}

inline int fail(int code, const char* format, ...) {
    char buffer[512];
    va_list args;
    va_start(args, format);
    vsnprintf(buffer, sizeof(buffer), format, args);
    va_end(args);
    last_error() = buffer;
    return code;
}

#define ITK_REQUIRE(condition, ...)                             \
    do {                                                        \
        if (!(condition)) return fail(ITK_ERR_ARGUMENT, __VA_ARGS__); \
    } while (0)

#define ITK_CUDA(call)                                                                        \
    do {                                                                                      \
        const cudaError_t status_ = (call);                                                   \
        if (status_ != cudaSuccess)                                                           \
            return fail(ITK_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(status_));   \
    } while (0)

inline bool aligned16(const void* pointer) { return (reinterpret_cast<uintptr_t>(pointer) & 15u) == 0; }

// ---------------------------------------------------------------- driver entry point

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled_entry() {
    static EncodeTiled entry = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* symbol = nullptr;
        cudaDriverEntryPointQueryResult query;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &symbol, cudaEnableDefault, &query) == cudaSuccess &&
            query == cudaDriverEntryPointSuccess) {
            entry = reinterpret_cast<EncodeTiled>(symbol);
        }
    });
    return entry;
}

}  // namespace itk
