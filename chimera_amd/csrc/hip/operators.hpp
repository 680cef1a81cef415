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
typedef float f32x2_t __attribute__((ext_vector_type(2)));
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

// Eight neighbouring values of a row, of which the first `count` (8 or more:
// all) exist. Addresses need the alignment of T only: global memory takes
// 16-byte accesses at any, a little slower where they cross lines.
// kOnce: past the caches, for data that are not needed again soon.
template <typename T, bool kOnce = false>
__device__ __forceinline__ void load8(const T* p, int count, float (&v)[8]) {
    if (count >= 8) {
        typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int kPer = 16 / static_cast<int>(sizeof(T));
#pragma unroll
        for (int h = 0; h < 8 / kPer; ++h) {
            typedef vec_t any_t __attribute__((aligned(sizeof(T))));
            const any_t* from = reinterpret_cast<const any_t*>(p + h * kPer);
            const vec_t t = kOnce ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[h * kPer + j] = to_float(static_cast<T>(t[j]));
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < count ? to_float(p[j]) : 0.0f;
}

template <typename T, bool kOnce = false>
__device__ __forceinline__ void store8(T* p, int count, const float (&v)[8]) {
    if (count >= 8) {
        typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int kPer = 16 / static_cast<int>(sizeof(T));
#pragma unroll
        for (int h = 0; h < 8 / kPer; ++h) {
            vec_t t;
#pragma unroll
            for (int j = 0; j < kPer; ++j) t[j] = from_float<T>(v[h * kPer + j]);
            typedef vec_t any_t __attribute__((aligned(sizeof(T))));
            any_t* to = reinterpret_cast<any_t*>(p + h * kPer);
            if constexpr (kOnce)
                __builtin_nontemporal_store(t, to);
            else
                *to = t;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j < count) p[j] = from_float<T>(v[j]);
}

// A value from another lane by a DPP control.
template <int kCtrl>
__device__ __forceinline__ float lane_move(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kCtrl, 0xF, 0xF, false));
}
constexpr int kRotate8 = 0x128, kMirror8 = 0x141, kSwap2 = 0x4E, kSwap1 = 0xB1;  // of a row of 16 lanes

// Sum over the wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
    v += lane_move<kSwap1>(v);
    v += lane_move<kSwap2>(v);
    v += lane_move<kMirror8>(v);
    v += lane_move<kRotate8>(v);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
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

size_t linear_forward_workspace(const chimera_linear_shape& s);  // of any call of the shape
size_t linear_forward_workspace(const LinearForward& f);         // of this one
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
