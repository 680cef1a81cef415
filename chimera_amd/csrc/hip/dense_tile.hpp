// The tiled product of the dense layers and what happens to its sums (bias,
// activation, residual, the rows' lengths), shared by the translation units
// whose operands differ.
#pragma once

#include "operators.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace chimera {

namespace {

// ---- host arithmetic of the plans ----------------------------------------------

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

// Arrays one after the other at multiples of 256 bytes.
struct Carve {
    char* base;
    size_t off = 0;
    void* take(size_t bytes) {
        off = (off + 255) / 256 * 256;
        void* p = base ? base + off : nullptr;
        off += bytes;
        return p;
    }
};

constexpr int kCus = 256;

// Whether rows of `stride` elements from p all start at multiples of 16 bytes.
bool rows_aligned(const void* p, int64_t stride, size_t elem) {
    return (reinterpret_cast<uintptr_t>(p) | (static_cast<uint64_t>(stride) * elem)) % 16 == 0;
}

constexpr float kLeastNorm = 1e-12f;

// ---- activations ---------------------------------------------------------------

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHalfLog2e = 0.72134751f, kHalfLog2eRest = 9.6298152e-9f;  // 1 / (2 ln 2)
constexpr float kGeluTanhC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluTanhA = 0.044715f;

__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
}

// Phi(z) = (1 + erf(z / sqrt 2)) / 2 and exp(-z^2 / 2). For a = |z|, Phi(-a) =
// exp(-a^2 / 2) t Q(t) with t = 1 / (1 + 0.35 a) and Q a minimax fit on
// [0, 14.5], within 3.2e-8 of its size. The rounding of a^2 / (2 ln 2), up to
// 2^-18, is put back into the exponential. Below zero Phi is that product
// itself, so small values keep their digits: within 2^-20 of their size down
// to -13, beyond which the result is below 32 bits' normal numbers.
__device__ __forceinline__ float normal_cdf(float z, float* gauss) {
    const float a = fminf(fabsf(z), 16.0f);  // infinity squared less itself is NaN
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, a, 1.0f));
    float q = fmaf(-2.9157868e-2f, t, 1.44030839e-1f);
    q = fmaf(q, t, -2.5583884e-1f);
    q = fmaf(q, t, 1.5931952e-1f);
    q = fmaf(q, t, -2.3212234e-2f);
    q = fmaf(q, t, 1.05552457e-1f);
    q = fmaf(q, t, 1.1982130e-1f);
    q = fmaf(q, t, 1.3986352e-1f);
    q = fmaf(q, t, 1.3962130e-1f);
    const float square = a * a, exponent = square * kHalfLog2e;
    float rest = fmaf(square, kHalfLog2e, -exponent);
    rest = fmaf(square, kHalfLog2eRest, rest);
    rest = fmaf(fmaf(a, a, -square), kHalfLog2e, rest);
    const float g = __builtin_amdgcn_exp2f(-exponent);
    *gauss = fmaf(g * -0.69314718f, rest, g);
    const float tail = *gauss * (q * t);
    return z < 0.0f ? tail : 1.0f - tail;
}

// z Phi(z) for results that are rounded to 16 bits: Phi(-a) = 2^P(a) for
// a >= 0 with P a minimax fit on [0, 6] (2.5e-7 of the size), so that results
// are within 3e-6 of their size there, most of which is P's own rounding, and
// within 6e-9 below -6, where P falls to -infinity. 14 full-rate instructions
// and one quarter-rate one. (Five coefficients less give 1.9e-4, which is seen
// in the rounding: 8 % of fp16 results were not the nearest value. They took
// 65,536 x 4096 outputs 630 us instead of 657.)
__device__ __forceinline__ float gelu_16(float z) {
    const float a = fabsf(z);
    float p = fmaf(-1.2316869e-8f, a, 4.1466188e-7f);
    p = fmaf(p, a, -5.9383565e-6f);
    p = fmaf(p, a, 4.5272715e-5f);
    p = fmaf(p, a, -1.6424450e-4f);
    p = fmaf(p, a, -2.6072026e-4f);
    p = fmaf(p, a, 7.2999932e-3f);
    p = fmaf(p, a, -5.2711684e-2f);
    p = fmaf(p, a, -4.5911723e-1f);
    p = fmaf(p, a, -1.1511194f);
    p = fmaf(p, a, -0.99999964f);
    const float tail = __builtin_amdgcn_exp2f(p);
    return z * (z > 0.0f ? 1.0f - tail : tail);
}

constexpr int kRoundedGelu = -1;  // gelu_16 for CHIMERA_ACT_GELU

__device__ __forceinline__ float activation(float z, int act) {
    switch (act) {
        case CHIMERA_ACT_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case CHIMERA_ACT_GELU: {
            float gauss;
            return z * normal_cdf(z, &gauss);
        }
        case kRoundedGelu: return gelu_16(z);
        case CHIMERA_ACT_GELU_TANH:  // (1 + tanh u) / 2 is the sigmoid of 2 u
            return z * sigmoid(2.0f * kGeluTanhC * fmaf(kGeluTanhA * z * z, z, z));
        case CHIMERA_ACT_SILU: return z * sigmoid(z);
        default: return z;
    }
}

__device__ __forceinline__ float activation_slope(float z, int act) {
    switch (act) {
        case CHIMERA_ACT_RELU: return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
        case CHIMERA_ACT_GELU: {
            float gauss;
            const float cdf = normal_cdf(z, &gauss);
            return fmaf(z * 0.3989422804014327f, gauss, cdf);
        }
        case CHIMERA_ACT_GELU_TANH: {
            const float g = sigmoid(2.0f * kGeluTanhC * fmaf(kGeluTanhA * z * z, z, z));
            // g (1 - g) is zero long before z or its square overflow in this
            const float near = fminf(fmaxf(z, -1e6f), 1e6f);
            return fmaf(2.0f * kGeluTanhC * near * g * (1.0f - g), fmaf(3.0f * kGeluTanhA * near, near, 1.0f), g);
        }
        case CHIMERA_ACT_SILU: {
            const float g = sigmoid(z);
            return g * fmaf(z, 1.0f - g, 1.0f);
        }
        default: return 1.0f;
    }
}

// ---- what happens to a product's sums ------------------------------------------

struct Epilogue {
    const void* bias;
    const void* residual;
    void* y;
    void* saved;
    float* norms;
    float* partial;  // [split][m][n] sums of a split product instead of all that follows
    int64_t residual_stride, y_stride, saved_stride;
    int64_t m;
    int n;
    int act;
    bool out_f32, normalize;
};

// act(v) for many values, one branch for all.
template <typename T, int kRuns>
__device__ __forceinline__ void activate(float (&v)[kRuns][16], int act) {
    auto all = [&](auto a) {
#pragma unroll
        for (int j = 0; j < kRuns; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) v[j][r] = activation(v[j][r], decltype(a)::value);
    };
    switch (act) {
        case CHIMERA_ACT_RELU: all(std::integral_constant<int, CHIMERA_ACT_RELU>{}); break;
        case CHIMERA_ACT_GELU: all(std::integral_constant<int, CHIMERA_ACT_GELU>{}); break;
        case kRoundedGelu:
            if constexpr (sizeof(T) == 2) all(std::integral_constant<int, kRoundedGelu>{});
            break;
        case CHIMERA_ACT_GELU_TANH: all(std::integral_constant<int, CHIMERA_ACT_GELU_TANH>{}); break;
        case CHIMERA_ACT_SILU: all(std::integral_constant<int, CHIMERA_ACT_SILU>{}); break;
        default: break;
    }
}
// act'(z) for eight values.
__device__ __forceinline__ void slope8(const float (&z)[8], float (&v)[8], int act) {
    switch (act) {
#define CHIMERA_SLOPE(A)                                          \
    case A:                                                       \
        _Pragma("unroll") for (int j = 0; j < 8; ++j) v[j] = activation_slope(z[j], A); \
        break;
        CHIMERA_SLOPE(CHIMERA_ACT_RELU)
        CHIMERA_SLOPE(CHIMERA_ACT_GELU)
        CHIMERA_SLOPE(CHIMERA_ACT_GELU_TANH)
        CHIMERA_SLOPE(CHIMERA_ACT_SILU)
#undef CHIMERA_SLOPE
        default: break;
    }
}

// ---- matrix-core steps ---------------------------------------------------------

// The operands in microscaled 4-bit floating point: a byte holds two values,
// so sums are counted in bytes, 16 of which are a block with one scale.
struct Mx4 {
    unsigned char pair;
};

// One 16-byte chunk of a row of A and of B per lane: a 32 x 32 tile's product
// over 32 bytes of the summed axis (lanes 0..31 hold the rows' first chunk,
// lanes 32..63 the second). For 32-bit operands the four values of a chunk go
// into four instructions; which index of the axis a lane's value has does not
// matter as long as A and B agree.
template <typename T>
__device__ __forceinline__ f32x16_t mma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, _Float16)) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
}
// The same of two blocks of 4-bit values: byte kQuarter of scale_a and scale_b
// is the exponent of the lane's chunk of A and of B.
template <int kQuarter>
__device__ __forceinline__ f32x16_t mma32_mx4(u32x4_t a, uint32_t scale_a, u32x4_t b, uint32_t scale_b, f32x16_t c) {
    typedef int i32x8_t __attribute__((ext_vector_type(8)));
    const auto wide = [](u32x4_t v) {
        return i32x8_t{static_cast<int>(v[0]), static_cast<int>(v[1]), static_cast<int>(v[2]), static_cast<int>(v[3]), 0, 0, 0, 0};
    };
    constexpr int kFp4 = 4;
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a), wide(b), c, kFp4, kFp4, kQuarter,
                                                           static_cast<int>(scale_a), kQuarter, static_cast<int>(scale_b));
}
__device__ __forceinline__ __attribute__((address_space(3))) void* lds_at(void* p) {
    return (__attribute__((address_space(3))) void*)(p);
}

// 16 bytes a lane from memory straight to LDS, lane after lane from `to` on.
__device__ __forceinline__ void load_to_lds(const void* from, void* to) {
    __builtin_amdgcn_global_load_lds(from, lds_at(to), 16, 0, 0);
}
// Of each 16 lanes, lane s gives the address of four 16-bit values, columns
// 4 (s % 4) on of row s / 4 of a block of 4 x 16; lane i gets column i.
__device__ __forceinline__ u32x2_t read_transposed(const void* from) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                           (__attribute__((address_space(3))) s16x4*)(from)));
}

// What lanes past the end of the summed axis load.
__device__ __align__(256) unsigned char g_zero_chunk[256];

// C [m, n] = the sum over k < sum of A[., k] B[., k]. A matrix lies with its
// rows along the sum ("[m, sum]"), or across it ("[sum, m]", as X and dZ lie
// for dW).
struct Product {
    const void* a;
    const void* b;
    int64_t a_stride, b_stride;  // bytes between rows, multiples of 16 as is the first row's address
    int64_t m;
    int n;
    int64_t sum;  // with rows along it, whole 16-byte chunks; so are m and n with rows across it
    int tiles_m, tiles_n;
    int steps, steps_per_split;  // of kStepBytes along the sum
    // of 4-bit operands [steps][m or n][8]: those of a step's chunks 0, 2, 4, 6
    // and 1, 3, 5, 7, as the halves of a wave take them; zeros past the sum
    const uint8_t *a_scales, *b_scales;
};

// ---- tiled product -------------------------------------------------------------

constexpr int kStepBytes = 128;  // of the summed axis per step: 64 or 32 values

constexpr int kSchedMfma = 0x008, kSchedLdsRead = 0x100;  // instruction groups of the scheduler
constexpr int kWaitLds = 0xC07F;  // s_waitcnt lgkmcnt(0), the others not waited on

// Waits until at most kLoads of the wave's loads (and no LDS access) are under
// way, then for the block.
template <int kLoads>
__device__ __forceinline__ void wait_and_meet() {
    __builtin_amdgcn_s_waitcnt((kLoads & 15) | (kLoads >> 4 << 14) | (7 << 4));
    asm volatile("" ::: "memory");  // LDS accesses stay on their side
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// One operand of a tile: 128 bytes of the summed axis of its B rows (or
// columns, kAcross) a step, loaded by W waves.
//
// Rows along the sum: a step is 128 bytes of each row, whole lines (with 64
// bytes a CU loads 60 GB/s into LDS, with 128 it loads 125; the largest tile
// needs 75 at the matrix cores' rate); chunk c of row r lies at place
// c ^ (r / 2 % 8), so that 16 lanes that follow each other in an LDS read of 16
// bytes, two rows of which fill the banks, hit different ones (with r % 8 half
// of the reads' cycles were conflicts).
// Rows across the sum: a step is 64 (or 32, of 32 bits) rows of B values. For
// 16-bit values the LDS's transposing read gives 16 lanes four values of a
// column each from four rows of 32 bytes; chunk c of row r lies at place
// c ^ 2 (r % 4), which puts those four rows in different banks. 32-bit values
// are read one by one, neighbouring columns in neighbouring lanes.
template <typename T, int B, int W, bool kAcross>
struct Side {
    static constexpr int kBytes = B * kStepBytes;
    static constexpr int kRowBytes = kAcross ? B * static_cast<int>(sizeof(T)) : kStepBytes;
    static constexpr int kPieces = kBytes / 1024;                   // one load instruction of a wave each
    static constexpr int kLoads = (kPieces + W - 1) / W;            // of each wave; some load the same piece
    static constexpr int kStepRows = kStepBytes / sizeof(T);        // values of the sum a step
    static constexpr int kPer = 16 / sizeof(T);
    const char* base;
    int64_t step_bytes;  // between steps
    uint32_t off[kLoads];
    uint32_t piece[kLoads];

    __device__ __forceinline__ void init(const void* p, int64_t stride, int64_t first, int64_t count, int step0, int w, int l) {
        const int last = static_cast<int>(min(count - first, static_cast<int64_t>(B))) - 1;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            piece[i] = static_cast<uint32_t>((i * W + w) % kPieces) * 1024u;
            const int byte = static_cast<int>(piece[i]) + 16 * l;
            const int row = byte / kRowBytes, place = byte % kRowBytes / 16;
            if constexpr (kAcross) {
                const int chunk = sizeof(T) == 2 ? place ^ ((row & 3) << 1) : place;
                // columns past the end load the last ones
                off[i] = static_cast<uint32_t>(row) * static_cast<uint32_t>(stride) +
                         16u * static_cast<uint32_t>(min(chunk, last / kPer));
            } else {
                const int chunk = place ^ ((row >> 1) & 7);
                off[i] = static_cast<uint32_t>(min(row, last)) * static_cast<uint32_t>(stride) + 16u * chunk;
            }
        }
        if constexpr (kAcross) {
            base = static_cast<const char*>(p) + first * static_cast<int64_t>(sizeof(T));
            step_bytes = kStepRows * stride;
        } else {
            base = static_cast<const char*>(p) + first * stride;
            step_bytes = kStepBytes;
        }
        base += step0 * step_bytes;
    }
    // `left` values of the sum are left in a step that it ends within; lanes
    // past them load zeros (an offset is chosen, not a load: every lane takes
    // part in each).
    __device__ __forceinline__ void fetch(int s, unsigned char* to, bool whole, int left, int l) const {
        const char* from = base + s * step_bytes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            int64_t o = off[i];
            if (!whole) {
                const int row = (static_cast<int>(piece[i]) + 16 * l) / kRowBytes;
                // the first value of the sum in this lane's chunk (or its row), within the step
                const int first = kAcross ? row : ((l & 7) ^ ((row >> 1) & 7)) * kPer;
                const int64_t zero = reinterpret_cast<const char*>(g_zero_chunk) - from;
                o = first >= left ? zero : o;
            }
            load_to_lds(from + o, to + piece[i]);
        }
    }
};

// The operands of one wave: kCount tiles of 32 rows (or columns) from `first`
// on, a quarter of a step at a time (two 16-byte chunks of the sum, one for
// each half of the wave).
template <typename T, int kCount, bool kAcross, int kRowBytes>
struct Reader {
    static constexpr int kReads = !kAcross ? 1 : sizeof(T) == 4 ? 4 : 2;  // of a tile's quarter step
    uint32_t off[kAcross && sizeof(T) == 2 ? kCount : 1];

    __device__ __forceinline__ void init(int first, int l) {
        if constexpr (!kAcross) {
            off[0] = static_cast<uint32_t>(first + (l & 31)) * kStepBytes + (((l >> 5) ^ ((l >> 1) & 7)) << 4);
        } else if constexpr (sizeof(T) == 4) {
            off[0] = static_cast<uint32_t>(4 * (l >> 5)) * kRowBytes + 4u * static_cast<uint32_t>(first + (l & 31));
        } else {
            const int row = 8 * (l >> 5) + ((l & 15) >> 2);
#pragma unroll
            for (int i = 0; i < kCount; ++i) {
                const int col = first + 32 * i + 16 * ((l >> 4) & 1) + 4 * (l & 3);
                off[i] = static_cast<uint32_t>(row) * kRowBytes + (((col >> 3) ^ ((row & 3) << 1)) << 4) + (col & 7) * 2u;
            }
        }
    }
    __device__ __forceinline__ void read(const unsigned char* from, int quarter, u32x4_t (&o)[kCount]) const {
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            if constexpr (!kAcross) {
                o[i] = *reinterpret_cast<const u32x4_t*>(from + i * 32 * kStepBytes + (off[0] ^ (quarter << 5)));
            } else if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[i][j] = *reinterpret_cast<const uint32_t*>(from + (8 * quarter + j) * kRowBytes + 128 * i + off[0]);
            } else {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const u32x2_t u = read_transposed(from + (16 * quarter + 4 * t) * kRowBytes + off[i]);
                    o[i][2 * t] = u[0];
                    o[i][2 * t + 1] = u[1];
                }
            }
        }
    }
};

// The scales of kCount tiles of 32 rows of 4-bit values: of each step, the
// four of this lane's row and half of the wave in one word. 32 rows' are two
// lines (where they lay with their rows, each in a line of its own, a step's
// loads of scales took the caches longer than those of its codes).
template <int kCount>
struct RowScales {
    const uint8_t* base;
    int64_t step_bytes;
    uint32_t off[kCount];
    __device__ __forceinline__ void init(const uint8_t* p, int64_t first, int64_t count, int step0, int l) {
        const int64_t from = min(first, count - 1);  // rows past the end take the last one's
        step_bytes = 8 * count;
        base = p + step0 * step_bytes + 8 * from + 4 * (l >> 5);
#pragma unroll
        for (int i = 0; i < kCount; ++i) off[i] = static_cast<uint32_t>(min(first + 32 * i + (l & 31), count - 1) - from) * 8u;
    }
    __device__ __forceinline__ void load(int s, uint32_t (&v)[kCount]) const {
        const uint8_t* from = base + s * step_bytes;
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] = *reinterpret_cast<const uint32_t*>(from + off[i]);
    }
};

// C tile of BM x BN by WM x WN waves. The operands go straight from memory to
// rings of LDS slots, one step each: kSlotsA of A, kSlotsB of B. Three and two
// fill the LDS with one tile of 256 (two of 128, four of 64) a CU, and leave
// half of a step's loads two steps to arrive and half of them one. A wave
// reads the operands of a quarter step while the matrix cores work on the
// quarter before it; once all waves have read a step's last quarter, its slots
// take new loads, before that quarter is multiplied. One meeting a step.
// Bound by the matrix cores and the LDS and loads that feed them: 8192 x 8192 x
// 8192 bf16 takes 880 us (1.25 PFLOP/s), 65,536 x 1024 -> 4096 with bias and
// GELU 657 (0.84; the same sums without the epilogue 530). Four waves of
// 128 x 128, two blocks a CU on 128 x 256, deeper rings and a whole step in
// registers were all slower.
// kEnd: the sums are stored, or go through the layer's epilogue, without or
// with the division by the rows' length (a tile then has all their columns).
enum End { kSums, kPlainLayer, kNormalizedLayer };

// LDS of a tile: the rings, or the rows on their way out.
template <int BM, int BN, int WM, int WN, int kSlotsA, int kSlotsB>
constexpr int tile_lds() {
    const int rings = (kSlotsA * BM + kSlotsB * BN) * kStepBytes, rows = WM * WN * 32 * (BN / WN + 4) * 4;
    return rings > rows ? rings : rows;
}

// Op: what A and B hold; T: the layer's type.
template <typename Op, typename T, int BM, int BN, int WM, int WN, int kSlotsA, int kSlotsB, bool kAcrossA, bool kAcrossB, End kEnd>
__device__ __forceinline__ void tile_product(unsigned char* lds, const Product& p, const Epilogue& e, int id, int split) {
    constexpr bool kLayer = kEnd != kSums;
    constexpr bool kNormalize = kEnd == kNormalizedLayer;
    constexpr int W = WM * WN;
    constexpr int TM = BM / WM, TN = BN / WN;
    constexpr int IM = TM / 32, IN = TN / 32;
    using SideA = Side<Op, BM, W, kAcrossA>;
    using SideB = Side<Op, BN, W, kAcrossB>;
    constexpr bool kScaled = sizeof(Op) == 1;
    constexpr int kPitch = TN + 4;

    const int l = lane_id();
    const int w = __builtin_amdgcn_readfirstlane(wave_id());
    const int wm = w / WN, wn = w % WN;

    // blocks go round the 8 XCDs; each XCD takes a run of tiles, in bands of
    // 8 tiles of rows, so that its L2 serves a band's rows and columns
    const int tiles = p.tiles_m * p.tiles_n;
    const int per = tiles / 8, rest = tiles % 8, xcd = id % 8;
    const int t = xcd * per + (xcd < rest ? xcd : rest) + id / 8;
    constexpr int kBand = 8;
    const int band = t / (kBand * p.tiles_n);
    const int height = min(kBand, p.tiles_m - band * kBand);
    const int in_band = t - band * kBand * p.tiles_n;
    const int64_t m0 = static_cast<int64_t>(band * kBand + in_band % height) * BM;
    const int n0 = in_band / height * BN;
    const int step0 = split * p.steps_per_split;
    const int steps = min(p.steps_per_split, p.steps - step0);

    SideA side_a;
    SideB side_b;
    side_a.init(p.a, p.a_stride, m0, p.m, step0, w, l);
    side_b.init(p.b, p.b_stride, n0, p.n, step0, w, l);
    Reader<Op, IM, kAcrossA, SideA::kRowBytes> reader_a;
    Reader<Op, IN, kAcrossB, SideB::kRowBytes> reader_b;
    reader_a.init(wm * TM, l);
    reader_b.init(wn * TN, l);
    // steps before the one that the sum ends within, if there is one
    const int left = static_cast<int>(p.sum % SideA::kStepRows);
    const int whole = steps - (left != 0 && step0 + steps == p.steps ? 1 : 0);
    unsigned char* const ring_b = lds + kSlotsA * SideA::kBytes;
    // the operands' parts of step s, if there is one
    auto fetch_a = [&](int s) {
        unsigned char* to = lds + s % kSlotsA * SideA::kBytes;
        if (s < whole)
            side_a.fetch(s, to, true, left, l);
        else if (s < steps)
            side_a.fetch(s, to, false, left, l);
    };
    auto fetch_b = [&](int s) {
        unsigned char* to = ring_b + s % kSlotsB * SideB::kBytes;
        if (s < whole)
            side_b.fetch(s, to, true, left, l);
        else if (s < steps)
            side_b.fetch(s, to, false, left, l);
    };

    f32x16_t acc[IM][IN];
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) acc[i][j] = f32x16_t{};
    struct Operands {
        u32x4_t a[IM], b[IN];
    };
    auto read = [&](int s, int quarter, Operands& o) {
        reader_a.read(lds + s % kSlotsA * SideA::kBytes, quarter, o.a);
        reader_b.read(ring_b + s % kSlotsB * SideB::kBytes, quarter, o.b);
    };
    // The products of a quarter, with the LDS reads before it spread between
    // them (issued all at once they held up the first products: 8192 x 8192 x
    // 8192 took 950 us, 880 so).
    constexpr int kMfmas = IM * IN * (sizeof(Op) == 4 ? 4 : 1);
    constexpr int kReads = IM * decltype(reader_a)::kReads + IN * decltype(reader_b)::kReads;
    constexpr int kBetween = (kReads + kMfmas - 1) / kMfmas;
    // Scales of the step that is multiplied, of the next one and, on their way,
    // of the one after it: these loads are issued before that step's parts, so
    // they are there when the parts are waited for and no wait grows by them.
    // Past the last step they are loaded again: a branch here would divide the
    // loop, and its products would be moved behind the meeting.
    struct Scales {
        uint32_t a[IM], b[IN];
    };
    Scales scales, next_scales, far_scales;
    RowScales<IM> scales_a;
    RowScales<IN> scales_b;
    auto load_scales = [&](int s, Scales& to) {
        scales_a.load(min(s, steps - 1), to.a);
        scales_b.load(min(s, steps - 1), to.b);
        asm volatile("" ::: "memory");
    };
    // Said to be read here: a copy that the loop carries would be made before
    // they have come, and wait.
    auto take_scales = [&](const Scales& from, Scales& to) {
        auto take = [&](uint32_t v) {
            uint32_t t;
            asm volatile("v_mov_b32 %0, %1" : "=v"(t) : "v"(v) : "memory");
            return t;
        };
#pragma unroll
        for (int i = 0; i < IM; ++i) to.a[i] = take(from.a[i]);
#pragma unroll
        for (int j = 0; j < IN; ++j) to.b[j] = take(from.b[j]);
    };
    if constexpr (kScaled) {
        scales_a.init(p.a_scales, m0 + wm * TM, p.m, step0, l);
        scales_b.init(p.b_scales, n0 + wn * TN, p.n, step0, l);
        load_scales(0, next_scales);
        load_scales(1, far_scales);
    }
    auto multiply = [&](const Operands& o, auto quarter) {
#pragma unroll
        for (int i = 0; i < IM; ++i)
#pragma unroll
            for (int j = 0; j < IN; ++j) {
                if constexpr (kScaled)
                    acc[i][j] = mma32_mx4<decltype(quarter)::value>(o.b[j], scales.b[j], o.a[i], scales.a[i], acc[i][j]);
                else
                    acc[i][j] = mma32<Op>(o.b[j], o.a[i], acc[i][j]);
            }
#pragma unroll
        for (int g = 0; g < kReads / kBetween; ++g) {
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, kBetween, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    constexpr std::integral_constant<int, 0> q0;
    constexpr std::integral_constant<int, 1> q1;
    constexpr std::integral_constant<int, 2> q2;
    constexpr std::integral_constant<int, 3> q3;
    Operands even, odd;
    // the first three quarters of step s, whose first one is in `even`
    auto quarters = [&](int s) {
        read(s, 1, odd);
        multiply(even, q0);
        __builtin_amdgcn_s_waitcnt(kWaitLds);  // said before the next reads, it does not wait for them
        read(s, 2, even);
        multiply(odd, q1);
        __builtin_amdgcn_s_waitcnt(kWaitLds);
        read(s, 3, odd);
        multiply(even, q2);
    };
    // in the order that the loop goes on with: B and then A of a step, with A
    // kSlotsA - kSlotsB steps ahead
    static_assert(kSlotsA >= kSlotsB && kSlotsB >= 2, "");
    constexpr int kLead = kSlotsA - kSlotsB;
#pragma unroll
    for (int s = 0; s < kLead; ++s) fetch_a(s);
#pragma unroll
    for (int s = 0; s < kSlotsB; ++s) {
        fetch_b(s);
        fetch_a(s + kLead);
    }
    // at a step's meeting the next step's parts have to be there: of what is
    // under way, all up to B's part of it, or A's where that comes after
    constexpr int kPair = SideA::kLoads + SideB::kLoads;
    constexpr int kUnderWay = (kLead > 0 ? SideA::kLoads : 0) + (kSlotsB - 2) * kPair;
    if (steps >= kSlotsA)
        wait_and_meet<kUnderWay + kPair>();
    else
        wait_and_meet<0>();
    if constexpr (kScaled) take_scales(next_scales, scales);
    read(0, 0, even);
    int s = 0;
    for (; s + kSlotsA < whole; ++s) {
        quarters(s);
        wait_and_meet<kUnderWay>();
        if constexpr (kScaled) {
            take_scales(far_scales, next_scales);
            load_scales(s + 2, far_scales);
        }
        side_b.fetch(s + kSlotsB, ring_b + s % kSlotsB * SideB::kBytes, true, left, l);
        side_a.fetch(s + kSlotsA, lds + s % kSlotsA * SideA::kBytes, true, left, l);
        read(s + 1, 0, even);
        multiply(odd, q3);
        __builtin_amdgcn_s_waitcnt(kWaitLds);
        if constexpr (kScaled) scales = next_scales;
    }
    for (; s < steps; ++s) {
        quarters(s);
        wait_and_meet<0>();
        if constexpr (kScaled) {
            take_scales(far_scales, next_scales);
            load_scales(s + 2, far_scales);
        }
        fetch_b(s + kSlotsB);
        fetch_a(s + kSlotsA);
        if (s + 1 < steps) read(s + 1, 0, even);
        multiply(odd, q3);
        if constexpr (kScaled) scales = next_scales;
    }

    // With W as the first operand, D lane l holds row l % 32 of X and of each
    // tile the columns 8 (r / 4) + 4 (l / 32) + r % 4: four neighbours at a
    // time. Bias, activation and length are dealt with there; then the values
    // go through LDS, in 16 bits where that is all that is left to do, so that
    // a wave's stores are whole 128-byte lines.
    constexpr int kLanes = TN / 8, kRows = kWave / kLanes;
    const bool inside = m0 + BM <= p.m && n0 + BN <= p.n;
    const int half = l >> 5;
    const int col0 = n0 + wn * TN;
    unsigned char* stage = lds + w * 32 * kPitch * 4;
    auto put = [&](const float(&v)[IN][16], auto type) {
        using S = decltype(type);
        S* to = reinterpret_cast<S*>(stage + (l & 31) * (TN * sizeof(S) + 16)) + 4 * half;
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                S t[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) t[r] = from_float<S>(v[j][4 * q + r]);
                if constexpr (sizeof(S) == 4)
                    *reinterpret_cast<u32x4_t*>(to + 32 * j + 8 * q) = *reinterpret_cast<const u32x4_t*>(t);
                else
                    *reinterpret_cast<u32x2_t*>(to + 32 * j + 8 * q) = *reinterpret_cast<const u32x2_t*>(t);
            }
        wave_lds_sync();
    };
    // each(visit, row of the 32, first of eight columns, its place in LDS) for the rows put
    auto each_row = [&](auto type, auto&& each) {
        using S = decltype(type);
#pragma unroll
        for (int q = 0; q < 32 / kRows; ++q) {
            const int row = q * kRows + l / kLanes, col = l % kLanes * 8;
            each(q, row, col, reinterpret_cast<const S*>(stage + row * (TN * sizeof(S) + 16)) + col);
        }
        wave_lds_sync();
    };
    // the rows put in T, as they are, to a matrix of T
    auto copy_out = [&](void* to, int64_t stride, int64_t m_first) {
        each_row(T{}, [&](int, int row, int col, const T* from) {
            const int64_t m = m_first + row;
            const int n = col0 + col;
            const int count = inside ? 8 : m < e.m ? e.n - n : 0;
            T* dst = static_cast<T*>(to) + m * stride + n;
            if (count >= 8) {
#pragma unroll
                for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h) {
                    const u32x4_t t = reinterpret_cast<const u32x4_t*>(from)[h];
                    __builtin_memcpy(dst + h * (16 / sizeof(T)), &t, 16);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < count) dst[j] = from[j];
            }
        });
    };
    float bias[IN][16];
    if constexpr (kLayer) {
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int n = col0 + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3);
                bias[j][r] = e.bias && n < e.n ? to_float(static_cast<const T*>(e.bias)[n]) : 0.0f;
            }
    }
    // The residual's values for the rows that each_row gives a lane, a tile
    // ahead: read between the stores, each waited for memory (10,007 x 520
    // outputs of a short sum took 14.3 us instead of 8.5 without a residual).
    typedef T row8_t __attribute__((ext_vector_type(8)));
    row8_t added[2][32 / kRows];
    const bool adds = kLayer && !kNormalize && e.residual;
    auto load_added = [&](int64_t m_first, row8_t(&to)[32 / kRows]) {
        typedef row8_t any_t __attribute__((aligned(sizeof(T))));
#pragma unroll
        for (int q = 0; q < 32 / kRows; ++q) {
            const int64_t m = m_first + q * kRows + l / kLanes;
            const int n = col0 + l % kLanes * 8;
            const int count = inside ? 8 : m < e.m ? e.n - n : 0;
            const T* from = static_cast<const T*>(e.residual) + m * e.residual_stride + n;
            if (count >= 8) {
                to[q] = *reinterpret_cast<const any_t*>(from);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) to[q][j] = j < count ? from[j] : from_float<T>(0.0f);
            }
        }
    };
    if (adds) load_added(m0 + wm * TM, added[0]);
    // what is left to do after LDS: nothing, or something in 32 bits
    const bool narrow = sizeof(T) == 2 && !e.out_f32 && !e.partial && (!kLayer || kNormalize || !e.residual);
#pragma unroll
    for (int i = 0; i < IM; ++i) {
        const int64_t m_first = m0 + wm * TM + 32 * i;
        float v[IN][16];
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) v[j][r] = kLayer ? acc[i][j][r] + bias[j][r] : acc[i][j][r];
        if constexpr (kLayer) {
            if (e.saved) {
                put(v, T{});
                copy_out(e.saved, e.saved_stride, m_first);
            }
            activate<T>(v, e.act);
            if constexpr (kNormalize) {
                const int64_t m = m_first + (l & 31);
                // the squares' sum, and that of the values times 2^-72 for rows
                // whose squares overflow (a length from 1.8e19 on)
                float sum = 0.0f, low_sum = 0.0f;
#pragma unroll
                for (int j = 0; j < IN; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int n = col0 + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3);
                        if (e.residual && m < e.m && n < e.n)
                            v[j][r] += to_float(static_cast<const T*>(e.residual)[m * e.residual_stride + n]);
                        const float low = v[j][r] * 0x1p-72f;
                        sum = n < e.n ? fmaf(v[j][r], v[j][r], sum) : sum;
                        low_sum = n < e.n ? fmaf(low, low, low_sum) : low_sum;
                    }
                sum += __shfl_xor(sum, 32, kWave);
                low_sum += __shfl_xor(low_sum, 32, kWave);
                if constexpr (WN > 1) {
                    static_assert(IM == 1, "one exchange of the waves' sums");
                    f32x2_t* sums = reinterpret_cast<f32x2_t*>(lds);
                    __syncthreads();
                    if (half == 0) sums[w * 32 + l] = f32x2_t{sum, low_sum};
                    __syncthreads();
                    sum = low_sum = 0.0f;
#pragma unroll
                    for (int o = 0; o < WN; ++o) {
                        const f32x2_t t = sums[(wm * WN + o) * 32 + (l & 31)];
                        sum += t[0];
                        low_sum += t[1];
                    }
                    __syncthreads();  // the rows go through the same LDS next
                }
                const bool large = sum == INFINITY;
                const float norm = sqrtf(large ? low_sum : sum);  // times 2^-72 where large
                const float held = norm < kLeastNorm && !large ? kLeastNorm : norm;  // NaN stays
                const float inv = 1.0f / held, before = large ? 0x1p-72f : 1.0f;
#pragma unroll
                for (int j = 0; j < IN; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) v[j][r] = v[j][r] * before * inv;
                if (e.norms && wn == 0 && half == 0 && m < e.m) e.norms[m] = large ? held * 0x1p72f : held;
            }
        }
        if (narrow) {
            put(v, T{});
            copy_out(e.y, e.y_stride, m_first);
            continue;
        }
        put(v, 0.0f);
        if (adds && i + 1 < IM) load_added(m_first + 32, added[(i + 1) & 1]);
        each_row(0.0f, [&](int q, int row, int col, const float* from) {
            const int64_t m = m_first + row;
            const int n = col0 + col;
            const int count = inside ? 8 : m < e.m ? e.n - n : 0;
            if (count <= 0) return;
            float u[8];
            load8(static_cast<const float*>(__builtin_assume_aligned(from, 16)), 8, u);
            if (e.partial) {
                store8(e.partial + (split * e.m + m) * e.n + n, count, u);
                return;
            }
            if (adds) {
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] += to_float(static_cast<T>(added[i & 1][q][j]));
            }
            const int64_t at = m * e.y_stride + n;
            if (e.out_f32)
                store8(static_cast<float*>(e.y) + at, count, u);
            else
                store8(static_cast<T*>(e.y) + at, count, u);
        });
    }
}

}  // namespace

}  // namespace chimera
