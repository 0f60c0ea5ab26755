// fields.hpp - what the label-field kernels (rows.hip, blocks.hip, linear.hip, distill.hip) share: element types, vectors of them,
// and the host's checks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/gsx_hip.h"

namespace gsx_amd {

void set_last_error(const char* what);

inline gsx_hip_status fields_fail(gsx_hip_status code, const char* what) {
    set_last_error(what);
    return code;
}

inline gsx_hip_status fields_launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GSX_HIP_SUCCESS : fields_fail((gsx_hip_status)e, what);
}

// Element types: float, __bf16 and _Float16. Arithmetic is in float; one rounding to nearest even on the way out.
template <typename T>
__device__ inline float to_float(T x) {
    return (float)x;
}
template <typename T>
__device__ inline T from_float(float x) {
    return (T)x;
}

// V elements loaded or stored together (V * sizeof(T) bytes, at that alignment up to 16).
template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Vec {
    T v[V];
};

inline bool known_type(int32_t type) {
    return type == GSX_HIP_DTYPE_F32 || type == GSX_HIP_DTYPE_BF16 || type == GSX_HIP_DTYPE_F16;
}
inline int64_t type_bytes(int32_t type) { return type == GSX_HIP_DTYPE_F32 ? 4 : 2; }

// f(T()) for the element type of a (known) type code.
template <typename F>
gsx_hip_status with_type(int32_t type, F f) {
    switch (type) {
        case GSX_HIP_DTYPE_F32: return f(float());
        case GSX_HIP_DTYPE_BF16: return f(__bf16());
        default: return f(_Float16());
    }
}

inline bool aligned_to(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }

// rows * stride elements (the last row only `width` long) stay within 2^63 bytes
inline bool rows_fit(int64_t rows, int64_t stride, int64_t width) {
    return rows >= 0 && width >= 0 && stride >= width && (rows == 0 || stride == 0 || rows <= (INT64_MAX >> 4) / stride);
}

__host__ __device__ inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace gsx_amd
