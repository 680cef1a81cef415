// Dense layers that turn hidden states into token embeddings, forward and
// backward (include/chimera_operators.h):
//   Z = X W^T + b,  H = act(Z) + R,  Y = H or H / max(|H|, 1e-12)
//   dH = dY or (dY - Y <Y, dY>) / norm,  dZ = dH act'(Z),
//   dX = dZ W,  dW = dZ^T X,  db = sum of dZ's rows,  dR = dH
// All three products are C = A B^T with both operands' rows along the summed
// axis; the backward pass lays W, X and dZ out that way (transposed) first.
#include "operators.hpp"

#include <algorithm>
#include <type_traits>

namespace chimera {

namespace {

constexpr float kLeastNorm = 1e-12f;

// ---- activations ---------------------------------------------------------------

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGeluTanhC = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kGeluTanhA = 0.044715f;

__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * z));
}

// Phi(z) = (1 + erf(z / sqrt 2)) / 2 and exp(-z^2 / 2). The error function is
// Abramowitz and Stegun's rational approximation 7.1.26, within 1.5e-7; below
// zero its complement is Phi itself, so small values keep their digits. A
// tenth of the instructions of the library's erff: the epilogue of a layer of
// 65,536 x 4096 outputs is not hidden by its products.
__device__ __forceinline__ float normal_cdf(float z, float* gauss) {
    const float x = fabsf(z) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    *gauss = __builtin_amdgcn_exp2f(-kLog2e * x * x);
    const float tail = 0.5f * p * t * *gauss;
    return z < 0.0f ? tail : 1.0f - tail;
}

// Phi(z) for values that are rounded to 16 bits: 1/2 + z P(z^2), a minimax
// fit on [-4, 4] held to 0 and 1 at its ends (and, clamped, beyond), within
// 3.4e-5 of Phi, so that gelu is within 1.4e-4: a thirtieth of a bf16 step at
// 1, half an fp16 rounding. 11 full-rate instructions where the exact form
// takes 20 and two quarter-rate ones: 65,536 x 4096 outputs took 200 us with
// that form, a third of the layer's products.
__device__ __forceinline__ float normal_cdf_16(float z) {
    const float c = __builtin_amdgcn_fmed3f(z, -4.0f, 4.0f);
    const float t = c * c;
    float p = fmaf(-1.2773050395153973e-09f, t, 1.0440346898121788e-07f);
    p = fmaf(p, t, -3.708714984895778e-06f);
    p = fmaf(p, t, 7.617972005391493e-05f);
    p = fmaf(p, t, -1.020980766043067e-03f);
    p = fmaf(p, t, 9.581183083355427e-03f);
    p = fmaf(p, t, -6.606381386518478e-02f);
    p = fmaf(p, t, 0.3988054394721985f);
    return __builtin_amdgcn_fmed3f(fmaf(p, c, 0.5f), 0.0f, 1.0f);
}

// T: the type that the result is rounded to or that the layer works in.
template <typename T>
__device__ __forceinline__ float activation(float z, int act) {
    switch (act) {
        case CHIMERA_ACT_RELU: return z > 0.0f ? z : (z != z ? z : 0.0f);
        case CHIMERA_ACT_GELU: {
            if constexpr (sizeof(T) == 2) return z * normal_cdf_16(z);
            float gauss;
            return z * normal_cdf(z, &gauss);
        }
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
            return fmaf(2.0f * kGeluTanhC * z * g * (1.0f - g), fmaf(3.0f * kGeluTanhA * z, z, 1.0f), g);
        }
        case CHIMERA_ACT_SILU: {
            const float g = sigmoid(z);
            return g * fmaf(z, 1.0f - g, 1.0f);
        }
        default: return 1.0f;
    }
}

// Whether rows of `stride` elements from p all start at multiples of 16 bytes.
bool rows_aligned(const void* p, int64_t stride, size_t elem) {
    return (reinterpret_cast<uintptr_t>(p) | (static_cast<uint64_t>(stride) * elem)) % 16 == 0;
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
    bool bias_vec, residual_vec, y_vec, saved_vec;
    bool vec;  // all of them
};

// act(v) for many values, one branch for all.
template <typename T, int kRuns>
__device__ __forceinline__ void activate(float (&v)[kRuns][16], int act) {
    auto all = [&](auto a) {
#pragma unroll
        for (int j = 0; j < kRuns; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) v[j][r] = activation<T>(v[j][r], decltype(a)::value);
    };
    switch (act) {
        case CHIMERA_ACT_RELU: all(std::integral_constant<int, CHIMERA_ACT_RELU>{}); break;
        case CHIMERA_ACT_GELU: all(std::integral_constant<int, CHIMERA_ACT_GELU>{}); break;
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

// The layer's epilogue on eight neighbouring sums of one row; with
// normalize the row lies in kLanes neighbouring lanes, which all call it.
template <typename T, int kLanes>
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t m, int n0, float (&v)[8]) {
    const int count = m < e.m ? e.n - n0 : 0;  // may be <= 0
    const bool whole = count >= 8;
    if (count > 0) {
        if (e.bias) {
            float b[8];
            load8(static_cast<const T*>(e.bias) + n0, whole && e.bias_vec, count, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += b[j];
        }
        if (e.saved) store8(static_cast<T*>(e.saved) + m * e.saved_stride + n0, whole && e.saved_vec, count, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = activation<T>(v[j], e.act);
        if (e.residual) {
            float r[8];
            load8(static_cast<const T*>(e.residual) + m * e.residual_stride + n0, whole && e.residual_vec, count, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += r[j];
        }
    }
    if (e.normalize) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s = j < count ? fmaf(v[j], v[j], s) : s;
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) s += __shfl_xor(s, o, kWave);
        const float norm = sqrtf(s);
        const float held = norm < kLeastNorm ? kLeastNorm : norm;  // NaN stays
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] / held;
        if (e.norms && n0 == 0 && count > 0) e.norms[m] = held;
    }
    if (count <= 0) return;
    const int64_t at = m * e.y_stride + n0;
    if (e.out_f32)
        store8(static_cast<float*>(e.y) + at, whole && e.y_vec, count, v);
    else
        store8(static_cast<T*>(e.y) + at, whole && e.y_vec, count, v);
}

// ---- matrix-core steps ---------------------------------------------------------

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
// The same for a 16 x 16 tile over 64 bytes (lane / 16 is the chunk).
template <typename T>
__device__ __forceinline__ f32x4_t mma16(u32x4_t a, u32x4_t b, f32x4_t c) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, _Float16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
}

__device__ __forceinline__ __attribute__((address_space(3))) void* lds_at(void* p) {
    return (__attribute__((address_space(3))) void*)(p);
}

// What lanes past the end of the summed axis load.
__device__ __align__(256) unsigned char g_zero_chunk[256];

struct Product {
    const void* a;  // [m, k]
    const void* b;  // [n, k]
    int64_t a_stride, b_stride;  // bytes; rows at multiples of 16 bytes
    int64_t m;
    int n;
    int64_t k_bytes;  // of a row, a multiple of 16
    int tiles_m, tiles_n;
    int steps, steps_per_split;  // of kStepBytes
};

// ---- tiled product -------------------------------------------------------------

constexpr int kStepBytes = 64;  // of the summed axis per step: 32 or 16 values

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

// C tile of BM x BN by WM x WN waves. The rows of A and B, 64 bytes of the
// summed axis a step, go straight from memory to a ring of four LDS slots:
// with three steps on their way the loads' latency is covered at full rate
// (256 x 256 tiles read 16 KB of LDS-bound data in the 512 cycles that a
// step's products take a wave). Chunk c of row r lies at place c ^ (r / 4 % 4),
// so that the 16 lanes that follow each other in an LDS read hit different
// banks. A wave reads the operands of one half of a step while the matrix
// cores work on the other half.
template <typename T, int BM, int BN, int WM, int WN, int kSlots>
__global__ __launch_bounds__(WM* WN* kWave) void linear_tile_kernel(Product p, Epilogue e) {
    constexpr int W = WM * WN;
    constexpr int TM = BM / WM, TN = BN / WN;
    constexpr int IM = TM / 32, IN = TN / 32;
    constexpr int LA = BM / 16 / W, LB = BN / 16 / W;  // loads of 16 rows per wave and step
    static_assert(LA * 16 * W == BM && LB * 16 * W == BN, "every wave loads the same number of rows");
    constexpr int kSlot = (BM + BN) * kStepBytes;
    constexpr int kPitch = TN + 4;
    constexpr int kStage = W * 32 * kPitch * 4;
    __shared__ __align__(1024) unsigned char lds[kSlots * kSlot > kStage ? kSlots * kSlot : kStage];

    const int l = lane_id();
    const int w = __builtin_amdgcn_readfirstlane(wave_id());
    const int wm = w / WN, wn = w % WN;

    // blocks go round the 8 XCDs; each XCD takes a run of tiles, in bands of
    // 8 tiles of rows, so that its L2 serves a band's rows and columns
    const int tiles = p.tiles_m * p.tiles_n;
    const int id = static_cast<int>(blockIdx.x);
    const int per = tiles / 8, rest = tiles % 8, xcd = id % 8;
    const int t = xcd * per + (xcd < rest ? xcd : rest) + id / 8;
    constexpr int kBand = 8;
    const int band = t / (kBand * p.tiles_n);
    const int height = min(kBand, p.tiles_m - band * kBand);
    const int in_band = t - band * kBand * p.tiles_n;
    const int64_t m0 = static_cast<int64_t>(band * kBand + in_band % height) * BM;
    const int n0 = in_band / height * BN;
    const int split = static_cast<int>(blockIdx.y);
    const int step0 = split * p.steps_per_split;
    const int steps = min(p.steps_per_split, p.steps - step0);

    // lane l loads chunk (l % 4) ^ (l / 16) of row l / 4 of its sixteen rows;
    // rows past the end load the last row
    const int chunk = (l & 3) ^ (l >> 4);
    const char* base_a = static_cast<const char*>(p.a) + m0 * p.a_stride + static_cast<int64_t>(step0) * kStepBytes;
    const char* base_b = static_cast<const char*>(p.b) + n0 * p.b_stride + static_cast<int64_t>(step0) * kStepBytes;
    uint32_t off_a[LA], off_b[LB];
    const int last_a = static_cast<int>(min(p.m - m0, static_cast<int64_t>(BM))) - 1, last_b = min(p.n - n0, BN) - 1;
#pragma unroll
    for (int i = 0; i < LA; ++i)
        off_a[i] = static_cast<uint32_t>(min((i * W + w) * 16 + (l >> 2), last_a)) * static_cast<uint32_t>(p.a_stride) +
                   16u * chunk;
#pragma unroll
    for (int i = 0; i < LB; ++i)
        off_b[i] = static_cast<uint32_t>(min((i * W + w) * 16 + (l >> 2), last_b)) * static_cast<uint32_t>(p.b_stride) +
                   16u * chunk;
    auto fetch = [&](int s, auto whole) {
        unsigned char* to = lds + s % kSlots * kSlot;
        const char* a = base_a + static_cast<int64_t>(s) * kStepBytes;
        const char* b = base_b + static_cast<int64_t>(s) * kStepBytes;
        // in its last step, lanes past the end of the summed axis load zeros
        // (an offset is chosen, not a load: every lane takes part in each)
        const bool zero = !whole && 16 * chunk >= p.k_bytes % kStepBytes;
        const int64_t zero_a = reinterpret_cast<const char*>(g_zero_chunk) - a;
        const int64_t zero_b = reinterpret_cast<const char*>(g_zero_chunk) - b;
#pragma unroll
        for (int i = 0; i < LA; ++i)
            __builtin_amdgcn_global_load_lds(a + (zero ? zero_a : static_cast<int64_t>(off_a[i])),
                                             lds_at(to + (i * W + w) * 1024), 16, 0, 0);
#pragma unroll
        for (int i = 0; i < LB; ++i)
            __builtin_amdgcn_global_load_lds(b + (zero ? zero_b : static_cast<int64_t>(off_b[i])),
                                             lds_at(to + BM * kStepBytes + (i * W + w) * 1024), 16, 0, 0);
    };
    // steps before the one that the axis ends within, if there is one
    const bool partial = p.k_bytes % kStepBytes != 0 && step0 + steps == p.steps;
    const int whole = steps - (partial ? 1 : 0);
    constexpr auto kWhole = std::true_type{};
    constexpr auto kPartial = std::false_type{};

    f32x16_t acc[IM][IN];
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) acc[i][j] = f32x16_t{};

    // halves of a step: chunks 0, 1 and 2, 3
    const uint32_t place = (((l >> 5) ^ ((l >> 2) & 3)) << 4);
    const uint32_t row_a = (wm * TM + (l & 31)) * kStepBytes + place;
    const uint32_t row_b = BM * kStepBytes + (wn * TN + (l & 31)) * kStepBytes + place;
    struct Operands {
        u32x4_t a[IM], b[IN];
    };
    auto read = [&](int s, int half, Operands& o) {
        const unsigned char* from = lds + s % kSlots * kSlot;
#pragma unroll
        for (int i = 0; i < IM; ++i)
            o.a[i] = *reinterpret_cast<const u32x4_t*>(from + i * 32 * kStepBytes + (row_a ^ (half << 5)));
#pragma unroll
        for (int j = 0; j < IN; ++j)
            o.b[j] = *reinterpret_cast<const u32x4_t*>(from + j * 32 * kStepBytes + (row_b ^ (half << 5)));
    };
    auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int i = 0; i < IM; ++i)
#pragma unroll
            for (int j = 0; j < IN; ++j) acc[i][j] = mma32<T>(o.b[j], o.a[i], acc[i][j]);
    };

    constexpr int kLoads = LA + LB;
    Operands first, second;
#pragma unroll
    for (int i = 0; i < IM; ++i) second.a[i] = u32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < IN; ++j) second.b[j] = u32x4_t{0, 0, 0, 0};
    auto step = [&](int s, auto&& more) {
        more();
        read(s, 0, first);
        __builtin_amdgcn_sched_barrier(0);
        multiply(second);  // the step before's; zeros at first
        __builtin_amdgcn_sched_barrier(0);
        // the first half is in registers by now; said here, it needs no wait
        // for the second half's reads below
        __builtin_amdgcn_s_waitcnt(kWaitLds);
        read(s, 1, second);
        __builtin_amdgcn_sched_barrier(0);
        multiply(first);
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr int kAhead = kSlots - 1;
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
        if (s < whole)
            fetch(s, kWhole);
        else if (s < steps)
            fetch(s, kPartial);
    }
    if (steps >= kAhead)
        wait_and_meet<(kAhead - 1) * kLoads>();
    else
        wait_and_meet<0>();
    int s = 0;
    for (; s + kAhead < whole; ++s) {
        step(s, [&] { fetch(s + kAhead, kWhole); });
        wait_and_meet<(kAhead - 1) * kLoads>();
        __builtin_amdgcn_sched_barrier(0);
    }
    for (; s < steps; ++s) {
        step(s, [&] {
            if (s + kAhead < steps) fetch(s + kAhead, kPartial);
        });
        wait_and_meet<0>();
        __builtin_amdgcn_sched_barrier(0);
    }
    multiply(second);

    // With W as the first operand, D lane l holds row l % 32 of X and of each
    // tile the columns 8 (r / 4) + 4 (l / 32) + r % 4: four neighbours at a
    // time. Bias, activation and length are dealt with there; then the values
    // go through LDS, in 16 bits where that is all that is left to do, so that
    // a wave's stores are whole 128-byte lines.
    constexpr int kLanes = TN / 8, kRows = kWave / kLanes;
    const bool inside = m0 + BM <= p.m && n0 + BN <= p.n && e.vec;
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
    // each(row of the 32, first of eight columns, its place in LDS) for the rows put
    auto each_row = [&](auto type, auto&& each) {
        using S = decltype(type);
#pragma unroll
        for (int q = 0; q < 32 / kRows; ++q) {
            const int row = q * kRows + l / kLanes, col = l % kLanes * 8;
            each(row, col, reinterpret_cast<const S*>(stage + row * (TN * sizeof(S) + 16)) + col);
        }
        wave_lds_sync();
    };
    // the rows put in T, as they are, to a matrix of T
    auto copy_out = [&](void* to, int64_t stride, bool vec, int64_t m_first) {
        each_row(T{}, [&](int row, int col, const T* from) {
            const int64_t m = m_first + row;
            const int n = col0 + col;
            const int count = inside ? 8 : m < e.m ? e.n - n : 0;
            T* dst = static_cast<T*>(to) + m * stride + n;
            if (inside || (vec && count >= 8)) {
#pragma unroll
                for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h)
                    reinterpret_cast<u32x4_t*>(dst)[h] = reinterpret_cast<const u32x4_t*>(from)[h];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < count) dst[j] = from[j];
            }
        });
    };
    float bias[IN][16];
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int n = col0 + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3);
            bias[j][r] = e.bias && n < e.n ? to_float(static_cast<const T*>(e.bias)[n]) : 0.0f;
        }
    // what is left to do after LDS: nothing, or something in 32 bits
    const bool narrow = sizeof(T) == 2 && !e.out_f32 && !e.partial && (!e.residual || e.normalize);
#pragma unroll
    for (int i = 0; i < IM; ++i) {
        const int64_t m_first = m0 + wm * TM + 32 * i;
        float v[IN][16];
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) v[j][r] = acc[i][j][r] + bias[j][r];
        if (e.saved) {
            put(v, T{});
            copy_out(e.saved, e.saved_stride, e.saved_vec, m_first);
        }
        activate<T>(v, e.act);
        if (e.normalize) {
            const int64_t m = m_first + (l & 31);
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < IN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int n = col0 + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3);
                    if (e.residual && m < e.m && n < e.n)
                        v[j][r] += to_float(static_cast<const T*>(e.residual)[m * e.residual_stride + n]);
                    s = n < e.n ? fmaf(v[j][r], v[j][r], s) : s;
                }
            s += __shfl_xor(s, 32, kWave);
            const float norm = sqrtf(s);
            const float held = norm < kLeastNorm ? kLeastNorm : norm;  // NaN stays
            const float inv = 1.0f / held;
#pragma unroll
            for (int j = 0; j < IN; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) v[j][r] *= inv;
            if (e.norms && half == 0 && m < e.m) e.norms[m] = held;
        }
        if (narrow) {
            put(v, T{});
            copy_out(e.y, e.y_stride, e.y_vec, m_first);
            continue;
        }
        put(v, 0.0f);
        each_row(0.0f, [&](int row, int col, const float* from) {
            const int64_t m = m_first + row;
            const int n = col0 + col;
            const int count = inside ? 8 : m < e.m ? e.n - n : 0;
            if (count <= 0) return;
            const bool whole = count >= 8;
            float u[8];
            load8(from, true, 8, u);
            if (e.partial) {
                store8(e.partial + (split * e.m + m) * e.n + n, inside || (whole && e.y_vec), count, u);
                return;
            }
            if (e.residual && !e.normalize) {
                float r[8];
                load8(static_cast<const T*>(e.residual) + m * e.residual_stride + n, inside || (whole && e.residual_vec),
                      count, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j] += r[j];
            }
            const int64_t at = m * e.y_stride + n;
            if (e.out_f32)
                store8(static_cast<float*>(e.y) + at, inside || (whole && e.y_vec), count, u);
            else
                store8(static_cast<T*>(e.y) + at, inside || (whole && e.y_vec), count, u);
        });
    }
}

// ---- few rows ------------------------------------------------------------------

// 16 rows of X against NT tiles of 16 rows of W; KW waves share the summed
// axis of each tile and join in LDS. Every row of W is read by one wave
// straight into registers, with no barrier before the join.
template <typename T, int NT, int KW>
__global__ __launch_bounds__(NT* KW* kWave) void linear_rows_kernel(Product p, Epilogue e, int k, bool aligned) {
    constexpr int kCols = NT * 16;
    constexpr int kPitch = kCols + 4;
    __shared__ __align__(16) float part[KW][16][kPitch];
    const int l = lane_id();
    const int w = __builtin_amdgcn_readfirstlane(wave_id());
    const int nt = w % NT, kw = w / NT;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 16;
    const int n0 = static_cast<int>(blockIdx.x) * kCols;
    const int64_t row_x = min(m0 + (l & 15), p.m - 1);
    const int row_w = min(n0 + nt * 16 + (l & 15), p.n - 1);
    const char* x = static_cast<const char*>(p.a) + row_x * p.a_stride;
    const char* wt = static_cast<const char*>(p.b) + row_w * p.b_stride;
    constexpr int kPer = 16 / sizeof(T);  // values of a chunk
    const int steps = (k + 4 * kPer - 1) / (4 * kPer);
    const int share = (steps + KW - 1) / KW;
    const int s_end = min(steps, (kw + 1) * share);
    auto chunk = [&](const char* row, int s) {
        const int at = (4 * s + (l >> 4)) * kPer;  // first value
        u32x4_t v = {0, 0, 0, 0};
        if (aligned) {
            if (at < k) v = *reinterpret_cast<const u32x4_t*>(row + static_cast<int64_t>(at) * sizeof(T));
        } else {
            T t[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                t[j] = at + j < k ? reinterpret_cast<const T*>(row)[at + j] : from_float<T>(0.0f);
            v = *reinterpret_cast<const u32x4_t*>(t);
        }
        return v;
    };
    f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = kw * share; s < s_end; s += 4) {
        u32x4_t a[4], b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool in = s + u < s_end;
            a[u] = in ? chunk(wt, s + u) : u32x4_t{0, 0, 0, 0};
            b[u] = in ? chunk(x, s + u) : u32x4_t{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) acc = mma16<T>(a[u], b[u], acc);
    }
    // D lane l holds row l % 16 of X, columns 4 (l / 16) .. + 3 of the tile
    *reinterpret_cast<f32x4_t*>(&part[kw][l & 15][nt * 16 + 4 * (l >> 4)]) = acc;
    __syncthreads();
    constexpr int kLanes = kCols / 8;
    const int tid = static_cast<int>(threadIdx.x);
    if (tid >= 16 * kLanes) return;
    const int row = tid / kLanes, col = tid % kLanes * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = part[0][row][col + j];
#pragma unroll
    for (int o = 1; o < KW; ++o)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += part[o][row][col + j];
    finish8<T, kLanes>(e, m0 + row, n0 + col, v);
}

// ---- layouts -------------------------------------------------------------------

// dst [rows][dst_stride] = src, zeros from column `cols` on: rows of any
// alignment laid out at multiples of 16 bytes.
template <typename T>
__global__ __launch_bounds__(256) void linear_align_kernel(const T* __restrict__ src, int64_t src_stride, int64_t rows,
                                                           int cols, T* __restrict__ dst, int dst_cols) {
    constexpr int kPer = 16 / sizeof(T);
    const int chunks = dst_cols / kPer;
    const int64_t total = rows * chunks;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const int64_t r = i / chunks;
        const int c = static_cast<int>(i - r * chunks) * kPer;
        T t[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) t[j] = c + j < cols ? src[r * src_stride + c + j] : from_float<T>(0.0f);
        *reinterpret_cast<u32x4_t*>(dst + r * dst_cols + c) = *reinterpret_cast<const u32x4_t*>(t);
    }
}

// dst [cols][dst_cols] = src^T, zeros from column `rows` on; dst_cols a
// multiple of 64. A block takes 64 x 64 values.
template <typename T>
__global__ __launch_bounds__(256) void linear_transpose_kernel(const T* __restrict__ src, int64_t src_stride,
                                                               int64_t rows, int cols, T* __restrict__ dst,
                                                               int64_t dst_cols) {
    __shared__ T tile[64][65];
    const int64_t r0 = static_cast<int64_t>(blockIdx.x) * 64;
    const int c0 = static_cast<int>(blockIdx.y) * 64;
    const int x = static_cast<int>(threadIdx.x) & 63, y = static_cast<int>(threadIdx.x) >> 6;
#pragma unroll 4
    for (int i = y; i < 64; i += 4)
        tile[i][x] = r0 + i < rows && c0 + x < cols ? src[(r0 + i) * src_stride + c0 + x] : from_float<T>(0.0f);
    __syncthreads();
#pragma unroll 4
    for (int i = y; i < 64; i += 4)
        if (c0 + i < cols) dst[static_cast<int64_t>(c0 + i) * dst_cols + r0 + x] = tile[x][i];
}

// ---- the gradient before the products ------------------------------------------

struct GradArgs {
    const void* dy;
    const void* y;
    const void* saved;
    const float* norms;
    void* dresidual;
    void* g;    // dZ [m][g_cols], zeros from column n on, or NULL
    void* gt;   // dZ^T [n][gt_cols], zeros from column m on, or NULL
    float* sums;  // column sums of dZ by blocks of 64 rows [blocks][n], or NULL
    int64_t dy_stride, y_stride, saved_stride, dresidual_stride, gt_cols;
    int64_t m;
    int n, g_cols, act;
    bool out_f32, normalize, dy_vec, y_vec, saved_vec, dresidual_vec;
};

// 64 rows x 128 columns a block, eight neighbouring columns of four rows a
// thread: with normalize (n <= 128) a row is 16 neighbouring lanes.
template <typename T>
__global__ __launch_bounds__(256) void linear_grad_kernel(GradArgs a) {
    __shared__ T tile[64][129];
    __shared__ float sums[16][129];
    const int tid = static_cast<int>(threadIdx.x);
    const int col = tid % 16 * 8, n0 = static_cast<int>(blockIdx.y) * 128 + col;
    const int64_t m0 = static_cast<int64_t>(blockIdx.x) * 64;
    float sum[8] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = tid / 16 + 16 * i;
        const int64_t m = m0 + row;
        const int count = m < a.m ? a.n - n0 : 0;
        const bool whole = count >= 8;
        float g[8] = {};
        auto load = [&](const void* p, int64_t stride, bool vec, float(&v)[8]) {
            if (a.out_f32)
                load8(static_cast<const float*>(p) + m * stride + n0, whole && vec, count, v);
            else
                load8(static_cast<const T*>(p) + m * stride + n0, whole && vec, count, v);
        };
        if (count > 0) load(a.dy, a.dy_stride, a.dy_vec, g);
        if (a.normalize) {
            float y[8] = {};
            if (count > 0) load(a.y, a.y_stride, a.y_vec, y);
            float dot = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) dot = fmaf(y[j], g[j], dot);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) dot += __shfl_xor(dot, o, kWave);
            const float norm = count > 0 ? a.norms[m] : 1.0f;
            // at its least value the norm is a constant
            dot = norm > kLeastNorm ? dot : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = fmaf(-y[j], dot, g[j]) / norm;
        }
        if (a.dresidual && count > 0)
            store8(static_cast<T*>(a.dresidual) + m * a.dresidual_stride + n0, whole && a.dresidual_vec, count, g);
        if (a.act != CHIMERA_ACT_NONE && count > 0) {
            float z[8];
            load8(static_cast<const T*>(a.saved) + m * a.saved_stride + n0, whole && a.saved_vec, count, z);
            float slope[8];
            slope8(z, slope, a.act);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = j < count ? g[j] * slope[j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += g[j];
        if (a.g && m < a.m && n0 < a.g_cols) store8(static_cast<T*>(a.g) + m * a.g_cols + n0, true, 8, g);
        if (a.gt) {
#pragma unroll
            for (int j = 0; j < 8; ++j) tile[row][col + j] = from_float<T>(g[j]);
        }
    }
    if (a.sums) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[tid / 16][col + j] = sum[j];
    }
    __syncthreads();
    const int nb = static_cast<int>(blockIdx.y) * 128;
    if (a.sums && tid < 128 && nb + tid < a.n) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += sums[i][tid];
        a.sums[static_cast<int64_t>(blockIdx.x) * a.n + nb + tid] = s;
    }
    if (a.gt) {
        for (int i = tid; i < 128 * 64; i += 256) {
            const int c = i / 64, r = i % 64;
            if (nb + c < a.n) static_cast<T*>(a.gt)[static_cast<int64_t>(nb + c) * a.gt_cols + m0 + r] = tile[r][c];
        }
    }
}

// dst[i] = sum over s of src[s][i], in order, for i < count: the parts of a
// split product (rows of `cols` values to rows of dst_stride) or the blocks'
// column sums. Four waves share the parts of 64 values.
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(const float* __restrict__ src, int64_t parts, int64_t count,
                                                          int cols, T* __restrict__ dst, int64_t dst_stride) {
    __shared__ float sums[4][kWave];
    const int l = lane_id(), w = wave_id();
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kWave + l;
    const int64_t share = (parts + 3) / 4;
    float s = 0.0f;
    if (i < count) {
        const int64_t end = min(parts, (w + 1) * share);
        for (int64_t k = w * share; k < end; ++k) s += src[k * count + i];
    }
    sums[w][l] = s;
    __syncthreads();
    if (w != 0 || i >= count) return;
    s = ((sums[0][l] + sums[1][l]) + sums[2][l]) + sums[3][l];
    dst[i / cols * dst_stride + i % cols] = from_float<T>(s);
}

template <typename T>
__global__ __launch_bounds__(256) void linear_zero_kernel(T* dst, int64_t rows, int cols, int64_t stride) {
    const int64_t i = blockIdx.x * 256ll + threadIdx.x;
    if (i < rows * cols) dst[i / cols * stride + i % cols] = from_float<T>(0.0f);
}

// ---- plans ---------------------------------------------------------------------

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

constexpr int kNormalizeCols = 128;
// Rows up to which a product without a split goes by 16 rows a block.
constexpr int64_t kFewRows = 64;

template <typename T>
void launch_tiles(hipStream_t st, Product p, Epilogue e, int splits) {
    p.steps = static_cast<int>(ceil_div(p.k_bytes, kStepBytes));
    p.steps_per_split = static_cast<int>(ceil_div(p.steps, splits));
    splits = static_cast<int>(ceil_div(p.steps, p.steps_per_split));
    auto plan = [&](int bm, int bn) {
        p.tiles_m = static_cast<int>(ceil_div(p.m, bm));
        p.tiles_n = static_cast<int>(ceil_div(p.n, bn));
        return dim3(static_cast<unsigned>(p.tiles_m * p.tiles_n), static_cast<unsigned>(splits));
    };
    if (e.normalize) {
        const dim3 grid = plan(128, 128);
        hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 4, 1, 4>), grid, dim3(256), 0, st, p, e);
        return;
    }
    if (ceil_div(p.m, 256) * ceil_div(p.n, 256) * splits >= 256) {
        const dim3 grid = plan(256, 256);
        hipLaunchKernelGGL((linear_tile_kernel<T, 256, 256, 2, 4, 4>), grid, dim3(512), 0, st, p, e);
        return;
    }
    const dim3 grid = plan(128, 128);
    hipLaunchKernelGGL((linear_tile_kernel<T, 128, 128, 2, 2, 4>), grid, dim3(256), 0, st, p, e);
}

// A matrix as a product reads it: as it lies where its rows start at
// multiples of 16 bytes and end at one, else laid out again in `copy`
// (rows x round_up(cols, 64)).
template <typename T>
void aligned_rows(hipStream_t st, const void* src, int64_t stride, int64_t rows, int cols, void* copy, const void** p,
                  int64_t* stride_bytes, int64_t* k_bytes) {
    constexpr int64_t kMostStride = int64_t{1} << 22;  // a tile's rows within 32-bit offsets
    if (rows_aligned(src, stride, sizeof(T)) && cols * sizeof(T) % 16 == 0 && stride * static_cast<int64_t>(sizeof(T)) <= kMostStride) {
        *p = src;
        *stride_bytes = stride * static_cast<int64_t>(sizeof(T));
        *k_bytes = cols * static_cast<int64_t>(sizeof(T));
        return;
    }
    const int wide = static_cast<int>(round_up(cols, 64));
    const int64_t chunks = rows * (wide * static_cast<int64_t>(sizeof(T)) / 16);
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(ceil_div(chunks, 256), 65536));
    hipLaunchKernelGGL((linear_align_kernel<T>), dim3(blocks), dim3(256), 0, st, static_cast<const T*>(src), stride, rows,
                       cols, static_cast<T*>(copy), wide);
    *p = copy;
    *stride_bytes = wide * static_cast<int64_t>(sizeof(T));
    *k_bytes = *stride_bytes;
}

struct ForwardPlan {
    void* x;
    void* weight;
};
size_t carve_forward(const chimera_linear_shape& s, void* base, ForwardPlan* plan) {
    Carve c{static_cast<char*>(base)};
    const size_t wide = round_up(s.in_features, 64) * type_bytes(s.type);
    plan->x = c.take(static_cast<size_t>(s.rows) * wide);
    plan->weight = c.take(static_cast<size_t>(s.out_features) * wide);
    return c.off;
}

template <typename T>
hipError_t forward(hipStream_t st, const LinearForward& f) {
    const auto& s = f.s;
    const auto& a = f.a;
    const size_t out = s.out_type == CHIMERA_F32 ? 4 : sizeof(T);
    Epilogue e = {};
    e.bias = a.bias;
    e.residual = a.residual;
    e.y = a.y;
    e.saved = a.saved;
    e.norms = a.norms;
    e.residual_stride = a.residual_stride;
    e.y_stride = a.y_stride;
    e.saved_stride = a.saved_stride;
    e.m = s.rows;
    e.n = s.out_features;
    e.act = s.activation;
    e.out_f32 = out == 4;
    e.normalize = s.normalize != 0;
    e.residual_vec = rows_aligned(a.residual, a.residual_stride, sizeof(T));
    e.y_vec = rows_aligned(a.y, a.y_stride, out);
    e.saved_vec = rows_aligned(a.saved, a.saved_stride, sizeof(T));
    e.bias_vec = rows_aligned(a.bias, 0, sizeof(T));
    e.vec = e.y_vec && e.bias_vec && (!a.residual || e.residual_vec) && (!a.saved || e.saved_vec);
    Product p = {};
    p.m = s.rows;
    p.n = s.out_features;
    if (s.rows <= kFewRows) {
        p.a = a.x;
        p.b = a.weight;
        p.a_stride = a.x_stride * static_cast<int64_t>(sizeof(T));
        p.b_stride = a.weight_stride * static_cast<int64_t>(sizeof(T));
        const bool aligned = rows_aligned(a.x, a.x_stride, sizeof(T)) && rows_aligned(a.weight, a.weight_stride, sizeof(T)) &&
                             s.in_features * sizeof(T) % 16 == 0;
        const unsigned by = static_cast<unsigned>(ceil_div(s.rows, 16));
        if (e.normalize)
            hipLaunchKernelGGL((linear_rows_kernel<T, 8, 2>), dim3(1, by), dim3(1024), 0, st, p, e, s.in_features, aligned);
        else
            hipLaunchKernelGGL((linear_rows_kernel<T, 1, 8>), dim3(static_cast<unsigned>(ceil_div(s.out_features, 16)), by),
                               dim3(512), 0, st, p, e, s.in_features, aligned);
        return hipGetLastError();
    }
    ForwardPlan plan;
    (void)carve_forward(s, a.workspace, &plan);
    int64_t k_x = 0, k_w = 0;
    aligned_rows<T>(st, a.x, a.x_stride, s.rows, s.in_features, plan.x, &p.a, &p.a_stride, &k_x);
    aligned_rows<T>(st, a.weight, a.weight_stride, s.out_features, s.in_features, plan.weight, &p.b, &p.b_stride, &k_w);
    p.k_bytes = std::min(k_x, k_w);
    launch_tiles<T>(st, p, e, 1);
    return hipGetLastError();
}

struct BackwardPlan {
    int64_t m_pad;
    int n_pad;
    int splits;
    void *g, *gt, *xt, *wt;
    float *sums, *parts;
};

// Parts of dW's sum over the rows: enough blocks of 128 x 128 for the GPU,
// sixteen steps of 64 bytes a part at least.
int dweight_splits(const chimera_linear_shape& s) {
    const int64_t tiles = ceil_div(s.out_features, 128) * ceil_div(s.in_features, 128);
    const int64_t steps = ceil_div(round_up(s.rows, 64) * type_bytes(s.type), kStepBytes);
    return static_cast<int>(std::max<int64_t>(1, std::min(ceil_div(512, tiles), steps / 16)));
}

size_t carve_backward(const chimera_linear_shape& s, void* base, BackwardPlan* plan) {
    Carve c{static_cast<char*>(base)};
    const size_t e = type_bytes(s.type);
    plan->m_pad = round_up(s.rows, 64);
    plan->n_pad = static_cast<int>(round_up(s.out_features, 64));
    plan->splits = dweight_splits(s);
    const size_t k = static_cast<size_t>(s.in_features), n = static_cast<size_t>(s.out_features);
    plan->g = c.take(static_cast<size_t>(s.rows) * plan->n_pad * e);
    plan->gt = c.take(n * plan->m_pad * e);
    plan->xt = c.take(k * plan->m_pad * e);
    plan->wt = c.take(k * plan->n_pad * e);
    plan->sums = static_cast<float*>(c.take(static_cast<size_t>(plan->m_pad / 64) * n * 4));
    plan->parts = static_cast<float*>(c.take(plan->splits > 1 ? plan->splits * n * k * 4 : 0));
    return c.off;
}

template <typename T>
hipError_t backward(hipStream_t st, const LinearBackward& b) {
    const auto& s = b.s;
    const auto& a = b.a;
    const int n = s.out_features, k = s.in_features;
    auto zero = [&](void* dst, int64_t rows, int cols, int64_t stride) {
        hipLaunchKernelGGL((linear_zero_kernel<T>), dim3(static_cast<unsigned>(ceil_div(rows * cols, 256))), dim3(256), 0,
                           st, static_cast<T*>(dst), rows, cols, stride);
    };
    if (s.rows == 0) {
        if (a.dweight) zero(a.dweight, n, k, a.dweight_stride);
        if (a.dbias) zero(a.dbias, 1, n, n);
        return hipGetLastError();
    }
    BackwardPlan plan;
    (void)carve_backward(s, a.workspace, &plan);
    const size_t out = s.out_type == CHIMERA_F32 ? 4 : sizeof(T);
    const unsigned row_blocks = static_cast<unsigned>(plan.m_pad / 64);
    GradArgs g = {};
    g.dy = a.dy;
    g.y = a.y;
    g.saved = a.saved;
    g.norms = a.norms;
    g.dresidual = a.dresidual;
    g.g = a.dx ? plan.g : nullptr;
    g.gt = a.dweight ? plan.gt : nullptr;
    g.sums = a.dbias ? plan.sums : nullptr;
    g.dy_stride = a.dy_stride;
    g.y_stride = a.y_stride;
    g.saved_stride = a.saved_stride;
    g.dresidual_stride = a.dresidual_stride;
    g.gt_cols = plan.m_pad;
    g.m = s.rows;
    g.n = n;
    g.g_cols = plan.n_pad;
    g.act = s.activation;
    g.out_f32 = out == 4;
    g.normalize = s.normalize != 0;
    g.dy_vec = rows_aligned(a.dy, a.dy_stride, out);
    g.y_vec = rows_aligned(a.y, a.y_stride, out);
    g.saved_vec = rows_aligned(a.saved, a.saved_stride, sizeof(T));
    g.dresidual_vec = rows_aligned(a.dresidual, a.dresidual_stride, sizeof(T));
    hipLaunchKernelGGL((linear_grad_kernel<T>), dim3(row_blocks, static_cast<unsigned>(ceil_div(n, 128))), dim3(256), 0, st, g);
    auto join = [&](const float* src, int64_t parts, int64_t count, int cols, void* dst, int64_t stride) {
        hipLaunchKernelGGL((linear_join_kernel<T>), dim3(static_cast<unsigned>(ceil_div(count, kWave))), dim3(256), 0, st,
                           src, parts, count, cols, static_cast<T*>(dst), stride);
    };
    if (a.dbias) join(plan.sums, row_blocks, n, n, a.dbias, n);
    auto product = [&](const void* pa, int64_t m, int64_t sum, const void* pb, int cols, void* dst, int64_t stride,
                       int splits) {
        Product p = {};
        p.a = pa;
        p.b = pb;
        p.a_stride = p.b_stride = p.k_bytes = sum * static_cast<int64_t>(sizeof(T));
        p.m = m;
        p.n = cols;
        Epilogue e = {};
        e.y = dst;
        e.y_stride = stride;
        e.m = m;
        e.n = cols;
        e.out_f32 = sizeof(T) == 4;
        e.y_vec = rows_aligned(dst, stride, sizeof(T));
        if (splits > 1) {
            e.partial = plan.parts;
            e.y_vec = cols % 4 == 0;
        }
        e.vec = e.y_vec;
        launch_tiles<T>(st, p, e, splits);
        if (splits > 1) {
            const int64_t steps = ceil_div(p.k_bytes, kStepBytes);
            join(plan.parts, ceil_div(steps, ceil_div(steps, splits)), m * cols, cols, dst, stride);
        }
    };
    if (a.dx) {
        hipLaunchKernelGGL((linear_transpose_kernel<T>),
                           dim3(static_cast<unsigned>(plan.n_pad / 64), static_cast<unsigned>(ceil_div(k, 64))), dim3(256),
                           0, st, static_cast<const T*>(a.weight), a.weight_stride, static_cast<int64_t>(n), k,
                           static_cast<T*>(plan.wt), static_cast<int64_t>(plan.n_pad));
        product(plan.g, s.rows, plan.n_pad, plan.wt, k, a.dx, a.dx_stride, 1);
    }
    if (a.dweight) {
        hipLaunchKernelGGL((linear_transpose_kernel<T>), dim3(row_blocks, static_cast<unsigned>(ceil_div(k, 64))), dim3(256),
                           0, st, static_cast<const T*>(a.x), a.x_stride, s.rows, k, static_cast<T*>(plan.xt), plan.m_pad);
        product(plan.gt, n, plan.m_pad, plan.xt, k, a.dweight, a.dweight_stride, plan.splits);
    }
    return hipGetLastError();
}

template <typename Call>
hipError_t by_type(int type, Call&& call) {
    switch (type) {
        case CHIMERA_F32: return call(float{});
        case CHIMERA_F16: return call(_Float16{});
        default: return call(__bf16{});
    }
}

}  // namespace

size_t linear_forward_workspace(const chimera_linear_shape& s) {
    ForwardPlan plan;
    return carve_forward(s, nullptr, &plan);
}
size_t linear_backward_workspace(const chimera_linear_shape& s) {
    BackwardPlan plan;
    return carve_backward(s, nullptr, &plan);
}

hipError_t launch_linear_forward(hipStream_t st, const LinearForward& f) {
    return by_type(f.s.type, [&](auto t) { return forward<decltype(t)>(st, f); });
}
hipError_t launch_linear_backward(hipStream_t st, const LinearBackward& b) {
    return by_type(b.s.type, [&](auto t) { return backward<decltype(t)>(st, b); });
}

}  // namespace chimera
