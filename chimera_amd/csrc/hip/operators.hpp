// Operators beside the index (include/chimera_operators.h): what their
// translation units share, and the launch functions that operators.hip calls.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "chimera_operators.h"
#include "common.hpp"

namespace chimera {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

inline size_t type_bytes(int type) { return type == CHIMERA_F32 ? 4 : 2; }

// Rounds to nearest even, as every narrowing here does.
template <typename T>
__device__ __forceinline__ T from_float(float v) {
    return static_cast<T>(v);
}
template <typename T>
__device__ __forceinline__ float to_float(T v) {
    return static_cast<float>(v);
}

// ---- dense layer (kernels_linear.hip) ----

struct LinearForward {
    chimera_linear_shape s;
    chimera_linear_forward a;
};
struct LinearBackward {
    chimera_linear_shape s;
    chimera_linear_backward a;
};

size_t linear_forward_workspace(const chimera_linear_shape& s);
size_t linear_backward_workspace(const chimera_linear_shape& s);
hipError_t launch_linear_forward(hipStream_t st, const LinearForward& f);
hipError_t launch_linear_backward(hipStream_t st, const LinearBackward& b);

// ---- quantised cache (kernels_cache.hip) ----

inline int cache_row_bytes(const chimera_cache& c) {
    return (c.dim + 31) / 32 * (c.format == CHIMERA_CACHE_INT4 ? 16 : 32);
}
inline int cache_row_scales(const chimera_cache& c) { return (c.dim + c.group - 1) / c.group; }

hipError_t launch_cache_write(hipStream_t st, const chimera_cache& c, const void* rows, int type, int64_t stride,
                              const int64_t* slots, int64_t n);
hipError_t launch_cache_read(hipStream_t st, const chimera_cache& c, const int64_t* slots, int64_t n, void* out,
                             int type, int64_t stride);
size_t cache_maxsim_workspace(const chimera_cache_maxsim& m);
hipError_t launch_cache_maxsim(hipStream_t st, const chimera_cache& c, const chimera_cache_maxsim& m);

}  // namespace chimera
