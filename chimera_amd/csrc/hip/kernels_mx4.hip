// Rows in microscaled 4-bit floating point, and the dense layer on a weight
// that is held so (include/chimera_operators.h):
//   e = max(exponent of max |x| - 2, -127) for each block of 32 values,
//   code = e2m1(x / 2^e), to nearest, ties to even, 6 at the most
//   Y = act(Q(X) W^T + b) + R, or its rows divided by their lengths
// Products of codes are exact, their sums are held in 32 bits.
#include "dense_tile.hpp"

namespace chimera {

namespace {

constexpr int kBlock = 32;        // values of a scale
constexpr int kStepBlocks = 8;    // blocks of a step of the product; rows of scales are whole steps
constexpr int kNotFinite = 0xFF;  // the scale of a block with a value that is not finite

// ---- a block's scale and codes -------------------------------------------------

// The scale (exponent + 127) of a block whose largest magnitude has these bits:
// its exponent less 2, that of the largest code.
__device__ __forceinline__ uint32_t scale_of(uint32_t most) {
    const int e = static_cast<int>(most >> 23);
    return e == 255 ? kNotFinite : static_cast<uint32_t>(max(e - 2, 0));
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Eight values over the scale as codes, the first in the lowest bits. The
// conversion instruction rounds to nearest even, keeps 6 for what is larger
// and divides by a power of two; small scales are taken away from the end of
// the 32-bit range first (exactly).
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], uint32_t scale) {
    if (scale == kNotFinite) return 0u;
    const bool low = scale < 64;
    const float by = __uint_as_float((low ? scale + 64 : scale) << 23);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = low ? x[j] * 0x1p64f : x[j];
    uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], by, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], by, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], by, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], by, 3);
}

// 2^(scale - 127), NaN for a block that was not finite.
__device__ __forceinline__ float power_of(uint32_t scale) {
    return __uint_as_float(scale == kNotFinite ? 0x7FC00000u : scale == 0 ? 0x00400000u : scale << 23);
}

// ---- rows ----------------------------------------------------------------------

struct RowsArgs {
    const void* x;
    void* out;
    uint8_t* codes;
    uint8_t* scales;
    int64_t stride;  // elements between rows of x or out
    int64_t rows;
    int cols;
    int units, groups;  // of eight values a row: up to whole blocks, and to whole rows of scales
};

// Four neighbouring lanes take a block, eight values each. One pass, bound by
// memory.
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantise_kernel(RowsArgs a) {
    const int64_t total = a.rows * a.groups;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int64_t r = i / a.groups;
        const int u = static_cast<int>(i - r * a.groups);
        float x[8] = {};
        const int count = a.cols - 8 * u;
        if (count > 0) load8(static_cast<const T*>(a.x) + r * a.stride + 8 * u, count, x);
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, magnitude(x[j]));
        most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), kSwap1, 0xF, 0xF, false)));
        most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), kSwap2, 0xF, 0xF, false)));
        const uint32_t scale = scale_of(most);
        if (u < a.units) reinterpret_cast<uint32_t*>(a.codes)[r * a.units + u] = codes8(x, scale);
        if (u % 4 == 0) a.scales[r * (a.groups / 4) + u / 4] = static_cast<uint8_t>(scale);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_read_kernel(RowsArgs a) {
    const int64_t total = a.rows * a.units;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int64_t r = i / a.units;
        const int u = static_cast<int>(i - r * a.units);
        const int count = a.cols - 8 * u;
        if (count <= 0) continue;
        const uint32_t c = reinterpret_cast<const uint32_t*>(a.codes)[i];
        const float power = power_of(a.scales[r * (a.groups / 4) + u / 4]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // exponent and mantissa at their places in 32 bits, 126 too low
            const uint32_t code = c >> (4 * j);
            v[j] = __uint_as_float((code & 7u) << 22 | (code & 8u) << 28) * 0x1p126f * power;
        }
        store8(static_cast<T*>(a.out) + r * a.stride + 8 * u, count, v);
    }
}

// ---- the layer -----------------------------------------------------------------

template <typename T, int BM, int BN, int WM, int WN, int kSlotsA, int kSlotsB, End kEnd>
__global__ __launch_bounds__(WM* WN* kWave) void mx4_tile_kernel(Product p, Epilogue e) {
    __shared__ __align__(1024) unsigned char lds[tile_lds<BM, BN, WM, WN, kSlotsA, kSlotsB>()];
    tile_product<Mx4, T, BM, BN, WM, WN, kSlotsA, kSlotsB, false, false, kEnd>(lds, p, e, static_cast<int>(blockIdx.x), 0);
}

template <typename T>
void quantise(hipStream_t st, const RowsArgs& a) {
    const int64_t blocks = ceil_div(a.rows * a.groups, 256);
    hipLaunchKernelGGL((mx4_quantise_kernel<T>), dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 65536))), dim3(256), 0,
                       st, a);
}

RowsArgs rows_args(int64_t rows, int cols, int64_t stride, uint8_t* codes, uint8_t* scales) {
    RowsArgs a = {};
    a.codes = codes;
    a.scales = scales;
    a.stride = stride;
    a.rows = rows;
    a.cols = cols;
    a.units = mx4_row_bytes(cols) / 4;
    a.groups = mx4_row_scales(cols) * 4;
    return a;
}

struct Mx4Plan {
    uint8_t *codes, *scales;
};
size_t carve(const chimera_linear_shape& s, void* base, Mx4Plan* plan) {
    Carve c{static_cast<char*>(base)};
    plan->codes = static_cast<uint8_t*>(c.take(static_cast<size_t>(s.rows) * mx4_row_bytes(s.in_features)));
    plan->scales = static_cast<uint8_t*>(c.take(static_cast<size_t>(s.rows) * mx4_row_scales(s.in_features)));
    return c.off;
}

template <typename T>
hipError_t layer(hipStream_t st, const chimera_linear_shape& s, const chimera_mx4_linear& a) {
    Mx4Plan plan;
    (void)carve(s, a.workspace, &plan);
    RowsArgs rows = rows_args(s.rows, s.in_features, a.x_stride, plan.codes, plan.scales);
    rows.x = a.x;
    quantise<T>(st, rows);
    Epilogue e = {};
    e.bias = a.bias;
    e.residual = a.residual;
    e.y = a.y;
    e.residual_stride = a.residual_stride;
    e.y_stride = a.y_stride;
    e.m = s.rows;
    e.n = s.out_features;
    const bool narrow = type_bytes(s.out_type) == 2;
    e.act = s.activation == CHIMERA_ACT_GELU && narrow ? kRoundedGelu : s.activation;
    e.out_f32 = !narrow;
    e.normalize = s.normalize != 0;
    Product p = {};
    p.a = plan.codes;
    p.b = a.codes;
    p.a_stride = p.b_stride = mx4_row_bytes(s.in_features);
    p.a_scales = plan.scales;
    p.b_scales = a.scales;
    p.a_scales_stride = p.b_scales_stride = mx4_row_scales(s.in_features);
    p.m = s.rows;
    p.n = s.out_features;
    p.sum = mx4_row_bytes(s.in_features);
    p.steps = p.steps_per_split = static_cast<int>(ceil_div(p.sum, kStepBytes));
    auto launch = [&](auto kernel, int bm, int bn, int threads) {
        p.tiles_m = static_cast<int>(ceil_div(p.m, bm));
        p.tiles_n = static_cast<int>(ceil_div(p.n, bn));
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.tiles_m * p.tiles_n)), dim3(static_cast<unsigned>(threads)), 0,
                           st, p, e);
    };
    if (s.normalize) {
        if (p.n > 64)
            launch(mx4_tile_kernel<T, 32, 128, 1, 4, 3, 3, kNormalizedLayer>, 32, 128, 256);
        else
            launch(mx4_tile_kernel<T, 64, 64, 2, 2, 3, 2, kNormalizedLayer>, 64, 64, 256);
    } else if (ceil_div(p.m, 128) * ceil_div(p.n, 128) >= kCus) {
        launch(mx4_tile_kernel<T, 128, 128, 2, 2, 3, 2, kPlainLayer>, 128, 128, 256);
    } else {
        launch(mx4_tile_kernel<T, 64, 64, 2, 2, 3, 2, kPlainLayer>, 64, 64, 256);
    }
    return hipGetLastError();
}

template <typename Call>
auto by_type(int type, Call&& call) {
    switch (type) {
        case CHIMERA_F32: return call(float{});
        case CHIMERA_F16: return call(_Float16{});
        default: return call(__bf16{});
    }
}

}  // namespace

size_t mx4_linear_workspace(const chimera_linear_shape& s) {
    Mx4Plan plan;
    return carve(s, nullptr, &plan);
}

hipError_t launch_mx4_quantise(hipStream_t st, const void* x, int type, int64_t stride, int64_t rows, int cols,
                               uint8_t* codes, uint8_t* scales) {
    RowsArgs a = rows_args(rows, cols, stride, codes, scales);
    a.x = x;
    by_type(type, [&](auto t) { quantise<decltype(t)>(st, a); });
    return hipGetLastError();
}

hipError_t launch_mx4_read(hipStream_t st, const uint8_t* codes, const uint8_t* scales, int64_t rows, int cols, void* out,
                           int type, int64_t stride) {
    RowsArgs a = rows_args(rows, cols, stride, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(scales));
    a.out = out;
    const int64_t blocks = ceil_div(rows * a.units, 256);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, 65536)));
    by_type(type, [&](auto t) { hipLaunchKernelGGL((mx4_read_kernel<decltype(t)>), grid, dim3(256), 0, st, a); });
    return hipGetLastError();
}

hipError_t launch_mx4_linear(hipStream_t st, const chimera_linear_shape& s, const chimera_mx4_linear& a) {
    return by_type(s.type, [&](auto t) { return layer<decltype(t)>(st, s, a); });
}

}  // namespace chimera
