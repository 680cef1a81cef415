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

// The largest of a block's magnitudes, of which this lane and its three
// neighbours have eight each.
__device__ __forceinline__ uint32_t block_most(const float (&x)[8]) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, magnitude(x[j]));
    most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), kSwap1, 0xF, 0xF, false)));
    return max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), kSwap2, 0xF, 0xF, false)));
}

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

// Of eight scales of a row of a weight, those of the blocks that there are, in
// the order of scale_place. Past the end codes are zeros, but scales may be
// anything; NaN would reach the sums.
__device__ __forceinline__ uint2 step_scales(const uint8_t* from, int blocks) {
    uint2 v = *reinterpret_cast<const uint2*>(from);
    if (blocks < 4) v.x &= (1u << (8 * blocks)) - 1u;
    if (blocks < 8) v.y = blocks <= 4 ? 0u : v.y & ((1u << (8 * (blocks - 4))) - 1u);
    return make_uint2(__builtin_amdgcn_perm(v.y, v.x, 0x06040200u), __builtin_amdgcn_perm(v.y, v.x, 0x07050301u));
}

// 2^(scale - 127), NaN for a block that was not finite.
__device__ __forceinline__ float power_of(uint32_t scale) {
    return __uint_as_float(scale == kNotFinite ? 0x7FC00000u : scale == 0 ? 0x00400000u : scale << 23);
}

// Place of a block's scale among the eight of its step for a layer: those that
// a half of a wave takes together.
__device__ __forceinline__ int scale_place(int block) { return block % 8 / 2 + block % 2 * 4; }

// ---- rows ----------------------------------------------------------------------

// Scales [row][block], or as a layer reads them: [step of the sum][row][8] or
// [32 rows][step][row][8], the eight in the order of scale_place.
enum ScaleLayout { kByRows, kBySteps, kWalked };

struct RowsArgs {
    const void* x;
    void* out;
    uint8_t* codes;
    uint8_t* scales;
    int64_t stride;  // elements between rows of x or out
    int64_t rows;
    int cols;
    int units;   // eights of a row of codes
    int steps;   // 256 values each
    int layout;  // of the scales
    unsigned row_blocks;
    // kBySteps: the weight's are laid out so too, by blocks after the rows'
    const uint8_t* weight_scales;
    uint8_t* weight_by_steps;
    int out_features;
};

// A block takes 256 values of 32 rows, four eights a thread; four neighbouring
// lanes are a block of values. Its scales go out together: a byte at a time
// they took as long as the codes. One pass, bound by memory.
template <typename T>
__global__ __launch_bounds__(256) void mx4_quantise_kernel(RowsArgs a) {
    const int t = static_cast<int>(threadIdx.x);
    if (blockIdx.x >= a.row_blocks) {  // a row's scales of a step, a thread
        const int steps = a.steps;
        const int64_t i = (blockIdx.x - a.row_blocks) * 256ll + t;
        if (i >= static_cast<int64_t>(a.out_features) * steps) return;
        const int64_t n = i / steps;
        const int s = static_cast<int>(i - n * steps);
        const uint2 v = step_scales(a.weight_scales + 8 * i, a.units / 4 - s * kStepBlocks);
        reinterpret_cast<uint2*>(a.weight_by_steps)[s * static_cast<int64_t>(a.out_features) + n] = v;
        return;
    }
    __shared__ unsigned char scales[32 * kStepBlocks];
    const int64_t unit = blockIdx.x / a.steps;
    const int step = static_cast<int>(blockIdx.x - unit * a.steps);
    float x[4][8] = {};
    const int u = step * 32 + t % 32, count = a.cols - 8 * u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = unit * 32 + i * 8 + t / 32;
        if (r < a.rows && count > 0) load8(static_cast<const T*>(a.x) + r * a.stride + 8 * u, count, x[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + t / 32;
        const int64_t r = unit * 32 + row;
        const uint32_t scale = scale_of(block_most(x[i]));
        if (r < a.rows && u < a.units) reinterpret_cast<uint32_t*>(a.codes)[r * a.units + u] = codes8(x[i], scale);
        if (t % 4 == 0) {
            const int block = t % 32 / 4;
            scales[row * kStepBlocks + (a.layout == kByRows ? block : scale_place(block))] = static_cast<unsigned char>(scale);
        }
    }
    __syncthreads();
    const int64_t r = unit * 32 + t;
    if (t >= 32 || r >= a.rows) return;
    const int64_t at = a.layout == kByRows  ? r * a.steps + step
                       : a.layout == kBySteps ? step * a.rows + r
                                            : (unit * a.steps + step) * 32 + t;
    reinterpret_cast<uint2*>(a.scales)[at] = reinterpret_cast<const uint2*>(scales)[t];
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_read_kernel(RowsArgs a) {
    const int64_t unit = blockIdx.x / a.steps;
    const int step = static_cast<int>(blockIdx.x - unit * a.steps);
    const int t = static_cast<int>(threadIdx.x), u = step * 32 + t % 32, count = a.cols - 8 * u;
    if (count <= 0) return;
    uint32_t c[4];
    float power[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = min(unit * 32 + i * 8 + t / 32, a.rows - 1);
        c[i] = reinterpret_cast<const uint32_t*>(a.codes)[r * a.units + u];
        power[i] = power_of(a.scales[r * a.steps * kStepBlocks + u / 4]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = unit * 32 + i * 8 + t / 32;
        if (r >= a.rows) break;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // exponent and mantissa at their places in 32 bits, 126 too low
            const uint32_t code = c[i] >> (4 * j);
            v[j] = __uint_as_float((code & 7u) << 22 | (code & 8u) << 28) * 0x1p126f * power[i];
        }
        store8(static_cast<T*>(a.out) + r * a.stride + 8 * u, count, v);
    }
}

// ---- the layer -----------------------------------------------------------------

// A wave keeps 32 rows of W, all of their sum, in registers and walks tiles of
// kUnits x 32 rows of X, whose codes go to LDS once for the block's 32 kWaves
// columns; a tile is one meeting of the block. kSteps: 256 values of the sum
// each. X comes quantised from memory, two tiles by turns, the next one under
// way while this one is multiplied and stored.
//
// LDS of 32 rows: their codes, chunk c of row r at place c ^ swizzle(r), so
// that the 16 rows of a 256-byte read lie in different banks; then the scales
// [kSteps][32 rows][8], a half wave's four together.
template <int kSteps>
struct Mx4Unit {
    static constexpr int kRowBytes = kSteps * 128;
    static constexpr int kCodes = 32 * kRowBytes, kScales = kSteps * 256;
    static constexpr int kBytes = kCodes + kScales;
    __device__ static __forceinline__ int swizzle(int row) {
        return kSteps % 2 ? (row >> 1) & 7 : row & 15;  // rows are odd or even multiples of 128 bytes
    }
};

struct Mx4Args {
    const void* x;  // few rows
    int64_t x_stride;
    int cols;
    const uint8_t* tiles;  // X's codes [rows][kRowBytes], up to whole tiles
    const uint8_t* tile_scales;  // [tiles][kSteps][32][8]
    const uint8_t* codes;  // W's
    const uint8_t* scales;
    int row_bytes, row_scales;  // W's
    int m_tiles, groups, ranges;  // tiles of rows, groups of columns, ranges of tiles
};

template <int kStores>
__device__ __forceinline__ void wait_before_stores() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((kStores & 15) | (kStores >> 4 << 14) | (7 << 4));
    asm volatile("" ::: "memory");
}

// GELU as max(z, 0) - |z| 2^P(|z|) with a polynomial P fitted to log2 of the
// normal distribution's tail, where the result is rounded to 16 bits. fp16 ends
// near -6: degree 7 is within 2^-17 of the size down to there, which makes about
// one result in a hundred another neighbour. bf16 goes on: degree 9 is within
// 2^-16.8 down to -6 and 2^-12 from there to -12.9, where the tail is no normal
// number any more (degree 7 is 16 % off at -10). The tail is 0 past 16. 65,536 x
// 1024 -> 4096 of bf16 takes 297 us in all, with degree 7 286, with 10 302, and
// without an activation 241; a comparison and a selection instead of the two
// limits take 8 more.
constexpr int kShortGelu = -2;
template <typename T, int kCount, typename Values>
__device__ __forceinline__ void gelu_short(Values& v) {
    constexpr bool kLong = __is_same(T, __bf16);
    constexpr int kTerms = kLong ? 10 : 8;
    constexpr float kP[2][10] = {
        {-1.8348062e-6f, 6.1598182e-5f, -9.3052391e-4f, 8.5078869e-3f, -5.3960058e-2f, -4.5846441e-1f, -1.1512511f, -0.99999529f},
        {-2.1041304e-9f, 1.5312204e-7f, -4.8620313e-6f, 8.9347304e-5f, -1.067303e-3f, 8.883602e-3f, -5.4517057e-2f, -4.5806479e-1f,
         -1.1513578f, -0.99999088f}};
#pragma unroll
    for (int j = 0; j < kCount; ++j) {
        const float a = __builtin_elementwise_minimum(fabsf(v[j]), 16.0f);  // NaN stays
        float p = kP[kLong][0];
#pragma unroll
        for (int i = 1; i < kTerms; ++i) p = fmaf(p, a, kP[kLong][i]);
        v[j] = fmaf(-a, __builtin_amdgcn_exp2f(p), __builtin_elementwise_maximum(v[j], 0.0f));
    }
}

// act(v) in place, one branch for all.
template <typename T, typename Values>
__device__ __forceinline__ void activate_few(Values& v, int act) {
    auto all = [&](auto a) {
#pragma unroll
        for (int j = 0; j < static_cast<int>(sizeof(Values) / sizeof(float)); ++j) v[j] = activation(v[j], decltype(a)::value);
    };
    switch (act) {
        case CHIMERA_ACT_RELU: all(std::integral_constant<int, CHIMERA_ACT_RELU>{}); break;
        case CHIMERA_ACT_GELU: all(std::integral_constant<int, CHIMERA_ACT_GELU>{}); break;
        case kShortGelu:
            if constexpr (sizeof(T) == 2) gelu_short<T, static_cast<int>(sizeof(Values) / sizeof(float))>(v);
            break;
        case CHIMERA_ACT_GELU_TANH: all(std::integral_constant<int, CHIMERA_ACT_GELU_TANH>{}); break;
        case CHIMERA_ACT_SILU: all(std::integral_constant<int, CHIMERA_ACT_SILU>{}); break;
        default: break;
    }
}

// What is added to a tile's 32 x 32 values, where its columns are whole: loaded
// before the products, as they take less time than a trip to memory.
template <typename T>
struct Residual {
    typedef T four_t __attribute__((ext_vector_type(4)));
    four_t r[4];

    __device__ __forceinline__ void load(const Epilogue& e, int64_t m, int n0, int half) {
        typedef four_t any_t __attribute__((aligned(sizeof(T))));
        const T* from = static_cast<const T*>(e.residual) + min(m, e.m - 1) * e.residual_stride + n0 + 4 * half;
#pragma unroll
        for (int g = 0; g < 4; ++g) r[g] = *reinterpret_cast<const any_t*>(from + 8 * g);
    }
};

// Activation, residual and the stores of a tile's 32 x 32 values: lane l holds
// row l % 32 and the columns 8 g + 4 (l / 32) + i, i < 4.
template <typename T>
__device__ __forceinline__ void finish_tile(f32x16_t& v, const Epilogue& e, const Residual<T>& added, int64_t m, int n0,
                                            bool full, int half) {
    activate_few<T>(v, e.act);
    if (m >= e.m) return;
    if (e.residual) {
        if (full) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] += to_float(static_cast<T>(added.r[j / 4][j % 4]));
        } else {
            const T* from = static_cast<const T*>(e.residual) + m * e.residual_stride + n0 + 4 * half;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (n0 + 8 * (j / 4) + 4 * half + j % 4 < e.n) v[j] += to_float(from[8 * (j / 4) + j % 4]);
        }
    }
    const int64_t at = m * e.y_stride + n0;
    if (full && e.out_f32) {
        typedef f32x4_t any_t __attribute__((aligned(4)));
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<any_t*>(static_cast<float*>(e.y) + at + 8 * g + 4 * half) =
                f32x4_t{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
        return;
    }
    if constexpr (sizeof(T) == 2) {
        if (full) {
            // the halves' fours of columns next to each other: 16 bytes a lane
            uint32_t u[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const T pair[2] = {from_float<T>(v[2 * j]), from_float<T>(v[2 * j + 1])};
                __builtin_memcpy(&u[j], pair, 4);
            }
            typedef u32x4_t any_t __attribute__((aligned(2)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const auto x = __builtin_amdgcn_permlane32_swap(u[4 * h], u[4 * h + 2], false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(u[4 * h + 1], u[4 * h + 3], false, false);
                *reinterpret_cast<any_t*>(static_cast<T*>(e.y) + at + 16 * h + 8 * half) = u32x4_t{x[0], y[0], x[1], y[1]};
            }
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int n = 8 * (j / 4) + 4 * half + j % 4;
        if (n0 + n >= e.n) continue;
        if (e.out_f32)
            static_cast<float*>(e.y)[at + n] = v[j];
        else
            static_cast<T*>(e.y)[at + n] = from_float<T>(v[j]);
    }
}

template <typename T, int kSteps, int kWaves, int kUnits>
__global__ __launch_bounds__(kWaves* kWave) void mx4_walk_kernel(Mx4Args a, Epilogue e) {
    using Unit = Mx4Unit<kSteps>;
    constexpr int kTileBytes = kUnits * Unit::kBytes;
    __shared__ __align__(1024) unsigned char lds[2 * kTileBytes];
    const int l = lane_id(), half = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(wave_id());
    // blocks go round the 8 XCDs; each takes a run of a range's groups of columns
    // after the other, so that those that walk the same rows share an L2
    const int id = static_cast<int>(blockIdx.x), xcd = id % 8, blocks = static_cast<int>(gridDim.x);
    const int at = xcd * (blocks / 8) + min(xcd, blocks % 8) + id / 8;
    const int group = at % a.groups, range = at / a.groups;
    const int first = static_cast<int>(static_cast<int64_t>(a.m_tiles) * range / a.ranges);
    const int last = static_cast<int>(static_cast<int64_t>(a.m_tiles) * (range + 1) / a.ranges);
    const int n0 = (group * kWaves + w) * 32;
    const bool works = n0 < e.n, full = n0 + 32 <= e.n;

    // pieces of a tile that this wave loads: 1 KB of codes, 256 bytes of scales
    constexpr int kPieces = Unit::kCodes / 1024, kLoads = (kUnits * kPieces + kWaves - 1) / kWaves;
    constexpr int kScaleLoads = (kUnits * kSteps + kWaves - 1) / kWaves;
    uint32_t off[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int piece = (i * kWaves + w) % (kUnits * kPieces);
        const int byte = piece % kPieces * 1024 + 16 * l;
        const int row = byte / Unit::kRowBytes, place = byte % Unit::kRowBytes / 16;
        off[i] = static_cast<uint32_t>(piece / kPieces * Unit::kCodes + row * Unit::kRowBytes + (place ^ Unit::swizzle(row)) * 16);
    }
    auto fetch = [&](int tile) {
        unsigned char* to = lds + (tile - first) % 2 * kTileBytes;
        const uint8_t* from = a.tiles + static_cast<int64_t>(tile) * kUnits * Unit::kCodes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int piece = (i * kWaves + w) % (kUnits * kPieces);
            load_to_lds(from + off[i], to + piece / kPieces * Unit::kBytes + piece % kPieces * 1024);
        }
        const uint8_t* scales = a.tile_scales + static_cast<int64_t>(tile) * kUnits * Unit::kScales;
#pragma unroll
        for (int i = 0; i < kScaleLoads; ++i) {
            const int s = (i * kWaves + w) % (kUnits * kSteps);
            __builtin_amdgcn_global_load_lds(
                scales + s * 256 + 4 * l, lds_at(to + s / kSteps * Unit::kBytes + Unit::kCodes + s % kSteps * 256), 4, 0, 0);
        }
    };
    if (first < last) fetch(first);

    // W's rows (past the end the last one again) and their scales
    u32x4_t wc[4 * kSteps];
    uint32_t ws[kSteps];
    f32x16_t bias;
    {
        const int64_t row = min(n0 + (l & 31), e.n - 1);
        const uint8_t* from = a.codes + row * a.row_bytes;
        const int blocks = a.row_bytes / 16;
#pragma unroll
        for (int q = 0; q < 4 * kSteps; ++q) {
            const int c = 2 * q + half;
            wc[q] = c < blocks ? *reinterpret_cast<const u32x4_t*>(from + 16 * c) : u32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            uint2 v = make_uint2(0u, 0u);
            if (8 * s < a.row_scales) v = step_scales(a.scales + row * a.row_scales + 8 * s, blocks - 8 * s);
            ws[s] = half ? v.y : v.x;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int n = n0 + 8 * (j / 4) + 4 * half + j % 4;
            bias[j] = e.bias && n < e.n ? to_float(static_cast<const T*>(e.bias)[n]) : 0.0f;
        }
        // all have come: the loop would wait for them, and for its own loads, at every turn
#pragma unroll
        for (int q = 0; q < 4 * kSteps; ++q) asm volatile("" : "+v"(wc[q]));
#pragma unroll
        for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(ws[s]));
        asm volatile("" : "+v"(bias));
    }

    f32x16_t acc[kUnits];
    const int x0 = ((half ^ Unit::swizzle(l & 31)) << 4), row_at = (l & 31) * Unit::kRowBytes;
    // X's operands two quarters ahead of the products
    auto multiply = [&](const unsigned char* from) {
        constexpr int kAll = 4 * kSteps, kAhead = 2;
        u32x4_t x[kAhead + 1][kUnits];
        uint32_t xs[kSteps][kUnits];
        auto read = [&](int q) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u)
                x[q % (kAhead + 1)][u] =
                    *reinterpret_cast<const u32x4_t*>(from + u * Unit::kBytes + row_at + (x0 ^ (q << 5)));
        };
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int u = 0; u < kUnits; ++u)
                xs[s][u] = *reinterpret_cast<const uint32_t*>(from + u * Unit::kBytes + Unit::kCodes + s * 256 + (l & 31) * 8 + 4 * half);
#pragma unroll
        for (int q = 0; q < kAhead; ++q) read(q);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            auto quarter = [&](auto kq) {
                constexpr int kQuarter = decltype(kq)::value;
                const int q = 4 * s + kQuarter;
                if (q + kAhead < kAll) read(q + kAhead);
#pragma unroll
                for (int u = 0; u < kUnits; ++u)
                    acc[u] = mma32_mx4<kQuarter>(wc[q], ws[s], x[q % (kAhead + 1)][u], xs[s][u], q == 0 ? bias : acc[u]);
#pragma unroll
                for (int u = 0; u < kUnits; ++u) {
                    __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
                    if (q + kAhead < kAll) __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
                }
            };
            quarter(std::integral_constant<int, 0>{});
            quarter(std::integral_constant<int, 1>{});
            quarter(std::integral_constant<int, 2>{});
            quarter(std::integral_constant<int, 3>{});
        }
    };
    const bool narrow = sizeof(T) == 2 && !e.out_f32;
    for (int tile = first; tile < last; ++tile) {
        // the stores of a whole tile come after the loads that are waited for
        const bool whole = tile > first && works && full;
        if (whole && narrow)
            wait_before_stores<2 * kUnits>();
        else if (whole && e.out_f32)
            wait_before_stores<4 * kUnits>();
        else
            wait_before_stores<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (tile + 1 < last) fetch(tile + 1);
        if (!works) continue;
        Residual<T> added[kUnits];
        const int64_t row = tile * int64_t{kUnits} * 32 + (l & 31);
        if (e.residual && full) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) added[u].load(e, row + 32 * u, n0, half);
        }
        multiply(lds + (tile - first) % 2 * kTileBytes);
#pragma unroll
        for (int u = 0; u < kUnits; ++u) finish_tile<T>(acc[u], e, added[u], row + 32 * u, n0, full, half);
    }
}

// ---- few rows, and rows of length one ------------------------------------------

// A block takes kRows rows of X and 32 kCols columns. 1,024 values of the sum at a
// time it quantises its rows to LDS, while W's codes are on their way to the
// registers of kSplit waves for each 32 columns, which divide the sum; the
// parts are joined in LDS, and each wave finishes a share of the columns.
// Bound by the latency of a trip to memory and of the meetings (one row, 1024
// -> 4096) or, with many rows of length one, by reading X.
template <typename T, int kCols, int kSplit, bool kNormalize, int kRows = 32>
__global__ __launch_bounds__(kCols* kSplit* kWave) void mx4_few_kernel(Mx4Args a, Epilogue e) {
    using Unit = Mx4Unit<4>;
    constexpr int kWaves = kCols * kSplit, kThreads = kWaves * kWave;
    constexpr int kChunk = 1024, kEights = kChunk / 8;  // of the sum
    constexpr int kRound = kRows * kEights / kThreads;  // eights of a thread
    constexpr int kShare = 16 / kSplit;                 // values of a lane that it finishes
    constexpr int kQuarters = 16 / kSplit;              // of a chunk, of a wave
    constexpr int kParts = kSplit > 1 ? kWaves * 16 * kWave * 4 : 0;
    typedef T eight_t __attribute__((ext_vector_type(8)));
    typedef eight_t any_eight_t __attribute__((aligned(sizeof(T))));
    __shared__ __align__(1024) unsigned char lds[kParts > Unit::kBytes ? kParts : Unit::kBytes];
    __shared__ f32x2_t lengths[kNormalize ? kWaves * 32 : 1];
    float* parts = reinterpret_cast<float*>(lds);
    const int t = static_cast<int>(threadIdx.x), l = lane_id(), half = l >> 5;
    const int w = __builtin_amdgcn_readfirstlane(wave_id()), part = w % kSplit;
    const int n0 = (static_cast<int>(blockIdx.x) * kCols + w / kSplit) * 32;
    const int64_t n = min(n0 + (l & 31), e.n - 1);  // rows past the end take the last one's
    const uint8_t* codes = a.codes + n * a.row_bytes;
    const uint8_t* scales = a.scales + n * a.row_scales;
    const int blocks = a.row_bytes / 16;
    const int x0 = ((half ^ Unit::swizzle(l & 31)) << 4), row_at = (l & 31) * Unit::kRowBytes;
    const int row0 = t / kEights, col0 = t % kEights * 8;
    constexpr int kRowsARound = kThreads / kEights;
    const int64_t m0 = (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * kRows, m = m0 + (l & 31);
    if (m0 >= e.m) return;
    const int rows = static_cast<int>(min(e.m - m0, int64_t{kRows}));
    f32x16_t acc = {};
    for (int chunk = 0; chunk < a.cols; chunk += kChunk) {
        eight_t x[kRound];
        {
            const int count = a.cols - chunk - col0;
            const T* from = static_cast<const T*>(a.x) + (m0 + row0) * a.x_stride + chunk + col0;
#pragma unroll
            for (int i = 0; i < kRound; ++i) {
                x[i] = eight_t{};
                if (row0 + i * kRowsARound < rows) {
                    if (count >= 8) {
                        x[i] = *reinterpret_cast<const any_eight_t*>(from);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (j < count) x[i][j] = from[j];
                    }
                }
                from += kRowsARound * a.x_stride;
            }
        }
        u32x4_t wc[kQuarters];
        uint32_t ws[kQuarters];
        const int c = chunk / kBlock + 2 * part * kQuarters + half;
#pragma unroll
        for (int i = 0; i < kQuarters; ++i) {
            wc[i] = u32x4_t{0, 0, 0, 0};
            ws[i] = 0;
            if (c + 2 * i < blocks) {
                wc[i] = reinterpret_cast<const u32x4_t*>(codes)[c + 2 * i];
                ws[i] = scales[c + 2 * i];
            }
        }
        if (chunk > 0) __syncthreads();  // the chunk before has been read
#pragma unroll
        for (int i = 0; i < kRound; ++i) {
            const int row = row0 + i * kRowsARound, u = t % kEights;
            if (row < rows) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = to_float(static_cast<T>(x[i][j]));
                const uint32_t scale = scale_of(block_most(f));
                unsigned char* to = lds + row * Unit::kRowBytes + ((u / 4 ^ Unit::swizzle(row)) << 4) + u % 4 * 4;
                *reinterpret_cast<uint32_t*>(to) = codes8(f, scale);
                if (u % 4 == 0) lds[Unit::kCodes + row * 32 + u / 4] = static_cast<unsigned char>(scale);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kQuarters; ++i) {
            const int q = part * kQuarters + i;
            const u32x4_t xc = *reinterpret_cast<const u32x4_t*>(lds + row_at + (x0 ^ (q << 5)));
            const uint32_t xs = lds[Unit::kCodes + (l & 31) * 32 + 2 * q + half];
            acc = mma32_mx4<0>(wc[i], ws[i], xc, xs, acc);
        }
    }
    // the sums of values `part` kShare on: neighbouring columns of this lane's row
    float v[kShare];
    const int j0 = part * kShare;
    auto column = [&](int i) { return n0 + 8 * ((j0 + i) / 4) + 4 * half + (j0 + i) % 4; };
    const bool in = (l & 31) < rows;
    if constexpr (kSplit > 1) {
        __syncthreads();  // the parts take the codes' place
#pragma unroll
        for (int j = 0; j < 16; ++j) parts[(w * 16 + j) * kWave + l] = acc[j];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
        float sum = 0.0f;
        if constexpr (kSplit > 1) {
#pragma unroll
            for (int o = 0; o < kSplit; ++o) sum += parts[((w - part + o) * 16 + j0 + i) * kWave + l];
        } else {
            sum = acc[i];
        }
        if (e.bias && column(i) < e.n) sum += to_float(static_cast<const T*>(e.bias)[column(i)]);
        v[i] = sum;
    }
    activate_few<T>(v, e.act);
    if (e.residual && in) {
#pragma unroll
        for (int i = 0; i < kShare; ++i)
            if (column(i) < e.n) v[i] += to_float(static_cast<const T*>(e.residual)[m * e.residual_stride + column(i)]);
    }
    if constexpr (kNormalize) {
        // the squares' sum, and that of the values times 2^-72 for rows whose squares overflow
        float sum = 0.0f, low_sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kShare; ++i) {
            const float low = v[i] * 0x1p-72f;
            sum = column(i) < e.n ? fmaf(v[i], v[i], sum) : sum;
            low_sum = column(i) < e.n ? fmaf(low, low, low_sum) : low_sum;
        }
        sum += __shfl_xor(sum, 32, kWave);
        low_sum += __shfl_xor(low_sum, 32, kWave);
        if (half == 0) lengths[w * 32 + l] = f32x2_t{sum, low_sum};
        __syncthreads();
        sum = low_sum = 0.0f;
#pragma unroll
        for (int o = 0; o < kWaves; ++o) {
            const f32x2_t u = lengths[o * 32 + (l & 31)];
            sum += u[0];
            low_sum += u[1];
        }
        const bool large = sum == INFINITY;
        const float norm = sqrtf(large ? low_sum : sum);  // times 2^-72 where large
        const float inv = 1.0f / (norm < kLeastNorm && !large ? kLeastNorm : norm), before = large ? 0x1p-72f : 1.0f;
#pragma unroll
        for (int i = 0; i < kShare; ++i) v[i] = v[i] * before * inv;
    }
    if (!in) return;
    // up to four neighbours at a time
    constexpr int kRun = kShare < 4 ? kShare : 4;
#pragma unroll
    for (int i = 0; i < kShare; i += kRun) {
        const int64_t at = m * e.y_stride + column(i);
        auto put = [&](auto type) {
            using S = decltype(type);
            S* to = static_cast<S*>(e.y) + at;
            typedef S vec_t __attribute__((ext_vector_type(kRun)));
            typedef vec_t any_t __attribute__((aligned(sizeof(S))));
            vec_t u;
#pragma unroll
            for (int j = 0; j < kRun; ++j) u[j] = from_float<S>(v[i + j]);
            if (column(i) + kRun <= e.n) {
                *reinterpret_cast<any_t*>(to) = u;
            } else {
#pragma unroll
                for (int j = 0; j < kRun; ++j)
                    if (column(i) + j < e.n) to[j] = u[j];
            }
        };
        if (e.out_f32)
            put(float{});
        else
            put(T{});
    }
}

// Sums too long for registers: the dense layers' tiles.
template <typename T, int BM, int BN, int WM, int WN, int kSlotsA, int kSlotsB>
__global__ __launch_bounds__(WM* WN* kWave) void mx4_tile_kernel(Product p, Epilogue e) {
    __shared__ __align__(1024) unsigned char lds[tile_lds<BM, BN, WM, WN, kSlotsA, kSlotsB>()];
    tile_product<Mx4, T, BM, BN, WM, WN, kSlotsA, kSlotsB, false, false, kPlainLayer>(lds, p, e, static_cast<int>(blockIdx.x), 0);
}

unsigned row_blocks(const RowsArgs& a) { return static_cast<unsigned>(ceil_div(a.rows, 32) * a.steps); }

template <typename T>
void quantise(hipStream_t st, RowsArgs a) {
    a.row_blocks = row_blocks(a);
    const int64_t weight_blocks = ceil_div(static_cast<int64_t>(a.out_features) * a.steps, 256);
    hipLaunchKernelGGL((mx4_quantise_kernel<T>), dim3(a.row_blocks + static_cast<unsigned>(weight_blocks)), dim3(256), 0, st, a);
}

// What rows_args describes, in launches of at most 2^20 blocks, which take most of
// a millisecond each: the most rows that a call may have are up to 2^31 blocks of
// 256 threads, and a launch has less than 2^32 threads. (A layer's rows, at most
// 2^23 blocks, are one launch.)
template <typename Call>
void by_parts(const RowsArgs& all, const void* x, void* out, int type, Call&& call) {
    constexpr int64_t kMostBlocks = 1 << 20;
    const int64_t most = std::max<int64_t>(1, kMostBlocks / all.steps) * 32, row = all.stride * static_cast<int64_t>(type_bytes(type));
    for (int64_t at = 0; at < all.rows; at += most) {
        RowsArgs a = all;
        a.rows = std::min(most, all.rows - at);
        a.x = x ? static_cast<const char*>(x) + at * row : nullptr;
        a.out = out ? static_cast<char*>(out) + at * row : nullptr;
        a.codes += at * all.units * 4;
        a.scales += at * all.steps * kStepBlocks;
        call(a);
    }
}

RowsArgs rows_args(int64_t rows, int cols, int64_t stride, uint8_t* codes, uint8_t* scales) {
    RowsArgs a = {};
    a.codes = codes;
    a.scales = scales;
    a.stride = stride;
    a.rows = rows;
    a.cols = cols;
    a.units = mx4_row_bytes(cols) / 4;
    a.steps = mx4_row_scales(cols) / kStepBlocks;
    return a;
}

// ---- plans ---------------------------------------------------------------------

constexpr int kMostSteps = 8;  // of a sum in registers

// Whether each 32 rows and columns quantise their rows for themselves: with
// normalize, where a block has all columns, and where there are few. us of that
// and of quantising first: 1024 -> 512 with 512 rows 7.3 and 10.3, with 1,024 10.6
// and 10.4, with 2,048 18.4 and 10.8; 1024 -> 4096 with 64 rows 7.0 and 10.2, with
// 128 8.9 and 10.3, with 192 12.9 and 10.5. So with sums of 1024 the line could
// lie at 550; longer ones, which take tiles that walk the whole sum, have not been
// compared.
bool few_rows(const chimera_linear_shape& s) {
    return s.normalize || ceil_div(s.rows, 32) * ceil_div(s.out_features, 32) * ceil_div(s.in_features, 1024) <= 768;
}

// Steps of the sum that the walk is compiled for.
int walk_steps(int in_features) {
    const int steps = static_cast<int>(ceil_div(in_features, 256));
    return steps <= 4 ? steps : kMostSteps;
}

struct Mx4Plan {
    uint8_t *codes, *scales, *weight_scales;
};
size_t carve(const chimera_linear_shape& s, void* base, Mx4Plan* plan) {
    Carve c{static_cast<char*>(base)};
    const int64_t steps = ceil_div(s.in_features, 256);
    *plan = {};
    if (few_rows(s)) return 0;
    if (steps > kMostSteps) {
        plan->weight_scales = static_cast<uint8_t*>(c.take(static_cast<size_t>(s.out_features) * mx4_row_scales(s.in_features)));
        plan->codes = static_cast<uint8_t*>(c.take(static_cast<size_t>(s.rows) * mx4_row_bytes(s.in_features)));
        plan->scales = static_cast<uint8_t*>(c.take(static_cast<size_t>(s.rows) * mx4_row_scales(s.in_features)));
    } else {
        const size_t rows = static_cast<size_t>(round_up(s.rows, 64)), wide = static_cast<size_t>(walk_steps(s.in_features));
        plan->codes = static_cast<uint8_t*>(c.take(rows * wide * 128));
        plan->scales = static_cast<uint8_t*>(c.take(rows * wide * 8));
    }
    return c.off;
}

template <typename T, int kSteps>
hipError_t walk(hipStream_t st, const chimera_linear_shape& s, const chimera_mx4_linear& a, Mx4Args g, const Epilogue& e) {
    Mx4Plan plan;
    (void)carve(s, a.workspace, &plan);
    g.tiles = plan.codes;
    g.tile_scales = plan.scales;
    RowsArgs rows = rows_args(s.rows, s.in_features, a.x_stride, plan.codes, plan.scales);
    rows.x = a.x;
    rows.layout = kWalked;
    rows.units = kSteps * 32;
    rows.steps = kSteps;
    quantise<T>(st, rows);
    auto launch = [&](auto waves, auto units, int blocks_a_cu) {
        constexpr int kWaves = decltype(waves)::value, kUnits = decltype(units)::value;
        g.m_tiles = static_cast<int>(ceil_div(s.rows, 32 * kUnits));
        g.groups = static_cast<int>(ceil_div(s.out_features, 32 * kWaves));
        g.ranges = static_cast<int>(std::min<int64_t>(g.m_tiles, std::max(1, blocks_a_cu * kCus / g.groups)));
        const unsigned blocks = static_cast<unsigned>(g.ranges * g.groups);
        hipLaunchKernelGGL((mx4_walk_kernel<T, kSteps, kWaves, kUnits>), dim3(blocks), dim3(kWaves * kWave), 0, st, g, e);
    };
    constexpr std::integral_constant<int, 1> k1;
    constexpr std::integral_constant<int, 4> k4;
    constexpr std::integral_constant<int, 8> k8;
    constexpr std::integral_constant<int, (kSteps > 4 ? 1 : 2)> k2;  // the weight takes half of the registers
    // Blocks of 256 columns that walk many tiles of 64 rows, or of 128 and 32:
    // 65,536 x 1024 -> 4096 with GELU 288 and 312 us, -> 2560 195 and 205, -> 1088
    // 97 and 94 (1,280 columns and 1,152), 16,384 x 1024 -> 1024 31.8 and 30.2,
    // 32,768 of these 51 and 51, 2,048 x 1024 -> 512 13.9 and 10.7.
    const int64_t n = s.out_features;
    if (ceil_div(s.rows, 64) * ceil_div(n, 256) >= 8 * kCus && round_up(n, 256) * 16 <= round_up(n, 128) * 17)
        launch(k8, k2, 1);
    else
        launch(k4, k1, 2);
    return hipGetLastError();
}

template <typename T>
hipError_t few(hipStream_t st, const chimera_linear_shape& s, const Mx4Args& g, const Epilogue& e) {
    auto launch = [&](auto kernel, int cols, int split, int rows = 32) {
        // the rows' tiles in two dimensions of at most 2^16 blocks
        const int64_t tiles = ceil_div(s.rows, rows), high = ceil_div(tiles, 65535);
        const dim3 grid(static_cast<unsigned>(ceil_div(s.out_features, 32 * cols)), static_cast<unsigned>(ceil_div(tiles, high)),
                        static_cast<unsigned>(high));
        hipLaunchKernelGGL(kernel, grid, dim3(static_cast<unsigned>(cols * split * kWave)), 0, st, g, e);
    };
    // Blocks of eight rows, a quarter of the products' 32, while each CU has at most
    // one (of 512 threads, two): a block's time is that of quantising its rows. us
    // with 8 and with 32: 32 x 768 -> 128 of length one 6.8 and 8.2, 2,048 of them
    // 7.2 and 8.5, 4,000 11.5 and 8.4; 32 x 1024 -> 4096 6.2 and 7.4, 128 x 1024 ->
    // 1024 6.0 and 7.4, 512 x 1024 -> 512 8.3 and 7.6.
    const int64_t columns = s.normalize ? 1 : ceil_div(s.out_features, 32);
    const bool eight = ceil_div(s.rows, 8) * columns <= (s.normalize ? 1 : 2) * kCus;
    if (!s.normalize && eight)
        launch(mx4_few_kernel<T, 1, 8, false, 8>, 1, 8, 8);
    else if (!s.normalize)
        launch(mx4_few_kernel<T, 1, 8, false>, 1, 8);
    else if (s.out_features > 64 && eight)
        launch(mx4_few_kernel<T, 4, 4, true, 8>, 4, 4, 8);
    else if (eight)
        launch(mx4_few_kernel<T, 2, 8, true, 8>, 2, 8, 8);
    else if (s.out_features > 64 && s.rows > 32 * kCus)
        launch(mx4_few_kernel<T, 4, 1, true>, 4, 1);
    else if (s.out_features > 64)
        launch(mx4_few_kernel<T, 4, 4, true>, 4, 4);
    else
        launch(mx4_few_kernel<T, 2, 8, true>, 2, 8);
    return hipGetLastError();
}

template <typename T>
hipError_t layer(hipStream_t st, const chimera_linear_shape& s, const chimera_mx4_linear& a) {
    Epilogue e = {};
    e.bias = a.bias;
    e.residual = a.residual;
    e.y = a.y;
    e.residual_stride = a.residual_stride;
    e.y_stride = a.y_stride;
    e.m = s.rows;
    e.n = s.out_features;
    const bool narrow = type_bytes(s.out_type) == 2;
    e.act = s.activation == CHIMERA_ACT_GELU && narrow ? kShortGelu : s.activation;
    e.out_f32 = !narrow;
    e.normalize = s.normalize != 0;
    Mx4Args g = {};
    g.x = a.x;
    g.x_stride = a.x_stride;
    g.cols = s.in_features;
    g.codes = a.codes;
    g.scales = a.scales;
    g.row_bytes = mx4_row_bytes(s.in_features);
    g.row_scales = mx4_row_scales(s.in_features);
    if (few_rows(s)) return few<T>(st, s, g, e);
    switch (ceil_div(s.in_features, 256)) {
        case 1: return walk<T, 1>(st, s, a, g, e);
        case 2: return walk<T, 2>(st, s, a, g, e);
        case 3: return walk<T, 3>(st, s, a, g, e);
        case 4: return walk<T, 4>(st, s, a, g, e);
        case 5:
        case 6:
        case 7:
        case 8: return walk<T, 8>(st, s, a, g, e);
        default: break;
    }
    // what the dense layers' tiles have; that for 16 bits ends at -6, too
    if (e.act == kShortGelu) e.act = s.type == CHIMERA_BF16 ? CHIMERA_ACT_GELU : kRoundedGelu;
    Mx4Plan plan;
    (void)carve(s, a.workspace, &plan);
    RowsArgs rows = rows_args(s.rows, s.in_features, a.x_stride, plan.codes, plan.scales);
    rows.x = a.x;
    rows.layout = kBySteps;
    rows.weight_scales = a.scales;
    rows.weight_by_steps = plan.weight_scales;
    rows.out_features = s.out_features;
    quantise<T>(st, rows);
    Product p = {};
    p.a = plan.codes;
    p.b = a.codes;
    p.a_stride = p.b_stride = mx4_row_bytes(s.in_features);
    p.a_scales = plan.scales;
    p.b_scales = plan.weight_scales;
    p.m = s.rows;
    p.n = s.out_features;
    p.sum = mx4_row_bytes(s.in_features);
    p.steps = p.steps_per_split = rows.steps;
    auto launch = [&](auto kernel, int bm, int bn, int threads) {
        p.tiles_m = static_cast<int>(ceil_div(p.m, bm));
        p.tiles_n = static_cast<int>(ceil_div(p.n, bn));
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.tiles_m * p.tiles_n)), dim3(static_cast<unsigned>(threads)), 0,
                           st, p, e);
    };
    if (ceil_div(p.m, 128) * ceil_div(p.n, 128) >= kCus) {
        launch(mx4_tile_kernel<T, 128, 128, 2, 2, 2, 2>, 128, 128, 256);
    } else {
        launch(mx4_tile_kernel<T, 64, 64, 2, 2, 3, 2>, 64, 64, 256);
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
    by_parts(rows_args(rows, cols, stride, codes, scales), x, nullptr, type,
             [&](const RowsArgs& a) { by_type(type, [&](auto t) { quantise<decltype(t)>(st, a); }); });
    return hipGetLastError();
}

hipError_t launch_mx4_read(hipStream_t st, const uint8_t* codes, const uint8_t* scales, int64_t rows, int cols, void* out,
                           int type, int64_t stride) {
    by_parts(rows_args(rows, cols, stride, const_cast<uint8_t*>(codes), const_cast<uint8_t*>(scales)), nullptr, out, type,
             [&](const RowsArgs& a) {
                 by_type(type, [&](auto t) {
                     hipLaunchKernelGGL((mx4_read_kernel<decltype(t)>), dim3(row_blocks(a)), dim3(256), 0, st, a);
                 });
             });
    return hipGetLastError();
}

hipError_t launch_mx4_linear(hipStream_t st, const chimera_linear_shape& s, const chimera_mx4_linear& a) {
    return by_type(s.type, [&](auto t) { return layer<decltype(t)>(st, s, a); });
}

}  // namespace chimera
