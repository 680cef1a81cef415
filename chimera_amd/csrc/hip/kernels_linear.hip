// Dense layers that turn hidden states into token embeddings, forward and
// backward (include/chimera_operators.h):
//   Z = X W^T + b,  H = act(Z) + R,  Y = H or H / max(|H|, 1e-12)
//   dH = dY or (dY - Y <Y, dY>) / norm,  dZ = dH act'(Z),
//   dX = dZ W,  dW = dZ^T X,  db = sum of dZ's rows,  dR = dH
// The products read X, W and dZ as they lie, with rows along the summed axis
// or across it.
#include "operators.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace chimera {

namespace {

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
// c ^ (r % 8), so that the lanes that follow each other in an LDS read of 16
// bytes hit different banks.
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
    int at;  // first value of the sum in this lane's chunk (or its row), within a step
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
                const int chunk = place ^ (row & 7);
                off[i] = static_cast<uint32_t>(min(row, last)) * static_cast<uint32_t>(stride) + 16u * chunk;
            }
        }
        if constexpr (kAcross) {
            base = static_cast<const char*>(p) + first * static_cast<int64_t>(sizeof(T));
            step_bytes = kStepRows * stride;
        } else {
            // the same chunk for every piece: 8 rows each
            at = ((l & 7) ^ (l >> 3)) * kPer;
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
                const int first = kAcross ? (static_cast<int>(piece[i]) + 16 * l) / kRowBytes : at;
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
            off[0] = static_cast<uint32_t>(first + (l & 31)) * kStepBytes + (((l >> 5) ^ (l & 7)) << 4);
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

template <typename T, int BM, int BN, int WM, int WN, int kSlotsA, int kSlotsB, bool kAcrossA, bool kAcrossB, End kEnd>
__device__ __forceinline__ void tile_product(unsigned char* lds, const Product& p, const Epilogue& e, int id, int split) {
    constexpr bool kLayer = kEnd != kSums;
    constexpr bool kNormalize = kEnd == kNormalizedLayer;
    constexpr int W = WM * WN;
    constexpr int TM = BM / WM, TN = BN / WN;
    constexpr int IM = TM / 32, IN = TN / 32;
    using SideA = Side<T, BM, W, kAcrossA>;
    using SideB = Side<T, BN, W, kAcrossB>;
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
    Reader<T, IM, kAcrossA, SideA::kRowBytes> reader_a;
    Reader<T, IN, kAcrossB, SideB::kRowBytes> reader_b;
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
    constexpr int kMfmas = IM * IN * (sizeof(T) == 4 ? 4 : 1);
    constexpr int kReads = IM * decltype(reader_a)::kReads + IN * decltype(reader_b)::kReads;
    constexpr int kBetween = (kReads + kMfmas - 1) / kMfmas;
    auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int i = 0; i < IM; ++i)
#pragma unroll
            for (int j = 0; j < IN; ++j) acc[i][j] = mma32<T>(o.b[j], o.a[i], acc[i][j]);
#pragma unroll
        for (int g = 0; g < kReads / kBetween; ++g) {
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, kBetween, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    Operands even, odd;
    // the first three quarters of step s, whose first one is in `even`
    auto quarters = [&](int s) {
        read(s, 1, odd);
        multiply(even);
        __builtin_amdgcn_s_waitcnt(kWaitLds);  // said before the next reads, it does not wait for them
        read(s, 2, even);
        multiply(odd);
        __builtin_amdgcn_s_waitcnt(kWaitLds);
        read(s, 3, odd);
        multiply(even);
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
    read(0, 0, even);
    int s = 0;
    for (; s + kSlotsA < whole; ++s) {
        quarters(s);
        wait_and_meet<kUnderWay>();
        side_b.fetch(s + kSlotsB, ring_b + s % kSlotsB * SideB::kBytes, true, left, l);
        side_a.fetch(s + kSlotsA, lds + s % kSlotsA * SideA::kBytes, true, left, l);
        read(s + 1, 0, even);
        multiply(odd);
        __builtin_amdgcn_s_waitcnt(kWaitLds);
    }
    for (; s < steps; ++s) {
        quarters(s);
        wait_and_meet<0>();
        fetch_b(s + kSlotsB);
        fetch_a(s + kSlotsA);
        if (s + 1 < steps) read(s + 1, 0, even);
        multiply(odd);
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

template <typename T, int BM, int BN, int WM, int WN, int kSlotsA, int kSlotsB, bool kAcrossA, bool kAcrossB, End kEnd>
__global__ __launch_bounds__(WM* WN* kWave) void linear_tile_kernel(Product p, Epilogue e) {
    __shared__ __align__(1024) unsigned char lds[tile_lds<BM, BN, WM, WN, kSlotsA, kSlotsB>()];
    tile_product<T, BM, BN, WM, WN, kSlotsA, kSlotsB, kAcrossA, kAcrossB, kEnd>(lds, p, e, static_cast<int>(blockIdx.x),
                                                                                static_cast<int>(blockIdx.y));
}

// dW (its parts first, the longer blocks) and dX on tiles of 64 in one launch:
// neither alone fills the GPU where both take such tiles.
template <typename T>
__global__ __launch_bounds__(256) void linear_gradients_kernel(Product pw, Epilogue ew, int splits, Product px, Epilogue ex) {
    __shared__ __align__(1024) unsigned char lds[tile_lds<64, 64, 2, 2, 3, 2>()];
    const int id = static_cast<int>(blockIdx.x), tiles = pw.tiles_m * pw.tiles_n;
    if (id < tiles * splits)
        tile_product<T, 64, 64, 2, 2, 3, 2, true, true, kSums>(lds, pw, ew, id % tiles, id / tiles);
    else
        tile_product<T, 64, 64, 2, 2, 3, 2, false, true, kSums>(lds, px, ex, id - tiles * splits, 0);
}

// ---- few rows ------------------------------------------------------------------

constexpr int kFewRows = 4;     // rows of X that go this way
constexpr int kWaveOutputs = 4; // rows of W a wave

// Up to four rows of X (kRows) against W, bound by reading W once: a wave
// takes four rows of W, a kilobyte of each at a time over its lanes, and sums
// the products in 32 bits on the vector unit; no matrix tile is worth filling
// for so few rows (one row, 1024 -> 4096: 4 us, on tiles of 64 7).
template <typename T, int kRows>
__global__ __launch_bounds__(256) void linear_vector_kernel(Product p, Epilogue e) {
    const int l = lane_id();
    const int n0 = (static_cast<int>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(wave_id())) * kWaveOutputs;
    if (n0 >= p.n) return;
    const int k = static_cast<int>(p.sum);
    const T* w[kWaveOutputs];
#pragma unroll
    for (int o = 0; o < kWaveOutputs; ++o)
        w[o] = reinterpret_cast<const T*>(static_cast<const char*>(p.b) + min(n0 + o, p.n - 1) * p.b_stride);
    float sums[kRows][kWaveOutputs] = {};
    constexpr int kAtOnce = 2;  // 8 values a lane each
    for (int k0 = 8 * l; k0 < k; k0 += kAtOnce * 8 * kWave) {
        float x[kAtOnce][kRows][8], v[kAtOnce][kWaveOutputs][8];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int at = k0 + u * 8 * kWave;
            const int count = k - at;
#pragma unroll
            for (int o = 0; o < kWaveOutputs; ++o) load8(w[o] + at, count, v[u][o]);
#pragma unroll
            for (int m = 0; m < kRows; ++m)
                load8(reinterpret_cast<const T*>(static_cast<const char*>(p.a) + m * p.a_stride) + at, count, x[u][m]);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
            for (int m = 0; m < kRows; ++m)
#pragma unroll
                for (int o = 0; o < kWaveOutputs; ++o)
#pragma unroll
                    for (int j = 0; j < 8; ++j) sums[m][o] = fmaf(x[u][m][j], v[u][o][j], sums[m][o]);
    }
    // lane m * kWaveOutputs + o finishes that sum
    float z = 0.0f;
#pragma unroll
    for (int m = 0; m < kRows; ++m)
#pragma unroll
        for (int o = 0; o < kWaveOutputs; ++o) {
            const float s = wave_sum(sums[m][o]);
            z = l == m * kWaveOutputs + o ? s : z;
        }
    const int64_t m = l / kWaveOutputs;
    const int n = n0 + l % kWaveOutputs;
    if (m >= kRows || n >= p.n) return;
    if (e.bias) z += to_float(static_cast<const T*>(e.bias)[n]);
    if (e.saved) static_cast<T*>(e.saved)[m * e.saved_stride + n] = from_float<T>(z);
    float h = activation(z, e.act);
    if (e.residual) h += to_float(static_cast<const T*>(e.residual)[m * e.residual_stride + n]);
    if (e.out_f32)
        static_cast<float*>(e.y)[m * e.y_stride + n] = h;
    else
        static_cast<T*>(e.y)[m * e.y_stride + n] = from_float<T>(h);
}

// ---- layouts -------------------------------------------------------------------

// dst [rows][dst_cols] = src, zeros from column `cols` on: rows of any
// alignment laid out at multiples of 16 bytes. Bound by memory and its own
// launch: 10,007 x 777 and 520 x 777 16-bit values take 9 us. (Loading such
// rows into registers and from there to LDS spares the copy, but every tile
// pays: 16,384 x 1001 -> 1024 took 62 us instead of 52, 65,536 x 1024 -> 4096
// in odd strides 916 instead of 666.)
struct AlignJob {
    const void* src;
    void* dst;
    int64_t src_stride, rows;
    int cols, dst_cols, blocks;
};
// Two matrices a launch: the first job's blocks, then the second's.
template <typename T>
__global__ __launch_bounds__(256) void linear_align_kernel(AlignJob first, AlignJob second) {
    constexpr int kPer = 16 / sizeof(T);
    const bool one = static_cast<int>(blockIdx.x) < first.blocks;
    const AlignJob job = one ? first : second;
    const int block = static_cast<int>(blockIdx.x) - (one ? 0 : first.blocks);
    const int chunks = job.dst_cols / kPer;
    const int64_t total = job.rows * chunks;
    for (int64_t i = block * 256ll + threadIdx.x; i < total; i += job.blocks * 256ll) {
        const int64_t r = i / chunks;
        const int c = static_cast<int>(i - r * chunks) * kPer;
        const T* from = static_cast<const T*>(job.src) + r * job.src_stride + c;
        u32x4_t t;
        if (c + kPer <= job.cols) {
            __builtin_memcpy(&t, from, 16);  // at any alignment of elements
        } else {
            T v[kPer];
#pragma unroll
            for (int j = 0; j < kPer; ++j) v[j] = c + j < job.cols ? from[j] : from_float<T>(0.0f);
            __builtin_memcpy(&t, v, 16);
        }
        *reinterpret_cast<u32x4_t*>(static_cast<T*>(job.dst) + r * job.dst_cols + c) = t;
    }
}

// ---- the gradient before the products ------------------------------------------

struct GradArgs {
    const void* dy;
    const void* y;
    const void* saved;
    const float* norms;
    void* dresidual;
    void* g;      // dZ [m][g_cols], zeros from column n on, or NULL
    float* sums;  // column sums of dZ by blocks of rows [blocks][n], or NULL
    int64_t dy_stride, y_stride, saved_stride, dresidual_stride;
    int64_t m;
    int n, g_cols, act;
    int block_rows;  // a multiple of 16
    bool out_f32, normalize;
};

// 16 rows x 128 columns at a time, eight neighbouring columns a thread: with
// normalize (n <= 128) a row is 16 neighbouring lanes. Bound by memory: 16,384
// x 1024 bf16 values with GELU and dR, 134 MB read and written, take 28 us (4.8
// TB/s; the slope to 32 bits is 2 us of it).
template <typename T>
__global__ __launch_bounds__(256) void linear_grad_kernel(GradArgs a) {
    __shared__ float sums[16][129];
    const int tid = static_cast<int>(threadIdx.x);
    const int col = tid % 16 * 8, n0 = static_cast<int>(blockIdx.y) * 128 + col;
    const int64_t m_end = min((blockIdx.x + int64_t{1}) * a.block_rows, a.m);
    float sum[8] = {};
#pragma unroll 2
    for (int64_t m0 = static_cast<int64_t>(blockIdx.x) * a.block_rows; m0 < m_end; m0 += 16) {
        const int64_t m = m0 + tid / 16;
        const int count = m < m_end ? a.n - n0 : 0;
        float g[8] = {};
        auto load = [&](const void* p, int64_t stride, float(&v)[8]) {
            if (a.out_f32)
                load8(static_cast<const float*>(p) + m * stride + n0, count, v);
            else
                load8(static_cast<const T*>(p) + m * stride + n0, count, v);
        };
        if (count > 0) load(a.dy, a.dy_stride, g);
        if (a.normalize) {
            float y[8] = {};
            if (count > 0) load(a.y, a.y_stride, y);
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
            store8(static_cast<T*>(a.dresidual) + m * a.dresidual_stride + n0, count, g);
        if (a.act != CHIMERA_ACT_NONE && count > 0) {
            float z[8], slope[8];
            load8(static_cast<const T*>(a.saved) + m * a.saved_stride + n0, count, z);
            slope8(z, slope, a.act);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = j < count ? g[j] * slope[j] : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += g[j];
        if (a.g && m < m_end && n0 < a.g_cols) store8(static_cast<T*>(a.g) + m * a.g_cols + n0, 8, g);
    }
    if (!a.sums) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[tid / 16][col + j] = sum[j];
    __syncthreads();
    const int nb = static_cast<int>(blockIdx.y) * 128;
    if (tid < 128 && nb + tid < a.n) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += sums[i][tid];
        a.sums[static_cast<int64_t>(blockIdx.x) * a.n + nb + tid] = s;
    }
}

// What is left to sum, in order: dst[rows][cols] = the sum over the parts of
// src [parts][rows * cols] - the parts of dW's product, or db's column sums.
struct Join {
    const float* src;
    void* dst;
    int64_t dst_stride, count;
    int parts, cols;
};

// Blocks of 512 threads: the first take 2,048 values of dW each, four
// neighbours a thread (one, where rows are not multiples of four), then the
// others 64 columns of db each, a lane a column, the parts over eight waves.
// A fixed order, so gradients do not change from run to run. Bound by memory
// and its launch: eight parts of 1024 x 1024 take 7.6 us.
template <typename T>
__global__ __launch_bounds__(512) void linear_join_kernel(Join w, int w_blocks, Join b) {
    __shared__ float sums[8][kWave];
    if (static_cast<int>(blockIdx.x) < w_blocks) {
        const bool four = w.cols % 4 == 0;
        const int64_t i = (blockIdx.x * 512ll + threadIdx.x) * (four ? 4 : 1);
        if (i >= w.count) return;
        const int64_t row = i / w.cols;
        T* to = static_cast<T*>(w.dst) + row * w.dst_stride + (i - row * w.cols);
        if (four) {
            f32x4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int k = 0; k < w.parts; ++k) s += *reinterpret_cast<const f32x4_t*>(w.src + k * w.count + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) to[j] = from_float<T>(s[j]);
        } else {
            float s = 0.0f;
#pragma unroll 4
            for (int k = 0; k < w.parts; ++k) s += w.src[k * w.count + i];
            to[0] = from_float<T>(s);
        }
        return;
    }
    const int l = lane_id(), wave = wave_id();
    const int i = (static_cast<int>(blockIdx.x) - w_blocks) * kWave + l;
    const int share = (b.parts + 7) / 8;
    float s = 0.0f;
    if (i < b.cols) {
        const int end = min(b.parts, (wave + 1) * share);
#pragma unroll 8
        for (int k = wave * share; k < end; ++k) s += b.src[static_cast<int64_t>(k) * b.cols + i];
    }
    sums[wave][l] = s;
    __syncthreads();
    if (wave != 0 || i >= b.cols) return;
    s = 0.0f;
#pragma unroll
    for (int o = 0; o < 8; ++o) s += sums[o][l];
    static_cast<T*>(b.dst)[i] = from_float<T>(s);
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

constexpr int kCus = 256;

// Which tile a product takes, and into how many parts its sum is split (where
// that is allowed): the least of an estimate in microseconds,
//   3 + steps x (step time of the busiest CU) + (parts written and read back).
// A step (128 bytes of the sum) takes a CU that has one tile `alone`, and `full`
// for each tile where it has several or all CUs work. Fitted to products of
// 64 to 65,536 rows; measured / estimated, us, 16-bit operands:
//                                      256 x 256   128 x 128    64 x 64
//     1024 x 1024, sum 1024            25 / 25     12 / 12      8 / 7
//     4096 x 1024, sum 1024            27 / 27     14 / 13      17 / 18
//     10007 x 1024, sum 1024           32 / 36     31 / 30      39 / 38
//     16384 x 1024, sum 1024           37 / 36     43 / 43      66 / 60
//     65536 x 4096, sum 1024           527 / 528   619 / 638    859 / 905
// With rows across the sum the data come from beyond the L2 and one tile a CU
// waits for them: 1024 x 1024 of 16,384 rows takes 160 us in 256 tiles of 64,
// 61 in four parts of the sum each; 226 in 64 tiles of 128, 69 in four parts,
// 50 in eight. 32-bit operands are bound by the matrix cores, which small
// tiles keep busy more evenly: 6001 x 1024, sum 768 takes 102 us on tiles of
// 128, 86 of 64.
struct TileCost {
    int size;
    double alone, alone_across, full;  // us
};
constexpr TileCost kCosts16[] = {{256, 1.33, 1.55, 2.05}, {128, 0.51, 0.87, 0.62}, {64, 0.26, 0.60, 0.22}};
constexpr TileCost kCosts32[] = {{128, 2.00, 2.20, 2.20}, {64, 0.62, 0.62, 0.60}};

struct TilePlan {
    int size, splits;
};

// The least estimate among tiles, and among parts of the sum up to most_splits.
TilePlan tile_plan(int64_t m, int64_t n, int64_t sum, size_t elem, bool across, int64_t most_splits) {
    const int64_t all_steps = ceil_div(sum * static_cast<int64_t>(elem), kStepBytes);
    TilePlan best = {0, 1};
    double least = 0.0;
    auto consider = [&](const TileCost& c) {
        const double tiles = static_cast<double>(ceil_div(m, c.size)) * static_cast<double>(ceil_div(n, c.size));
        for (int64_t splits = 1; splits == 1 || (splits <= most_splits && all_steps / splits >= 8); splits *= 2) {
            const double share = tiles * static_cast<double>(splits) / kCus;  // tiles a CU
            const double alone = across ? c.alone_across : c.alone;
            // CUs hold one tile of 256 at a time, two of 128, four of 64
            const double rounds = c.size == 256   ? std::ceil(share)
                                  : c.size == 128 ? (share + std::ceil(share)) / 2
                                                  : share + 0.25;
            const double step = share <= 1.0 ? alone + std::max(0.0, c.full - alone) * share
                                             : std::max(alone, c.full * rounds);
            double us = 3.0 + static_cast<double>(ceil_div(all_steps, splits)) * step;
            if (splits > 1) us += 3.0 + static_cast<double>(splits * m * n) * 8.0 / 4.5e6;
            if (best.size == 0 || us < least) {
                least = us;
                best = {c.size, static_cast<int>(splits)};
            }
        }
    };
    if (elem == 4)
        for (const TileCost& c : kCosts32) consider(c);
    else
        for (const TileCost& c : kCosts16) consider(c);
    return best;
}

// Sets a product's steps for about `splits` parts of its sum; returns how many
// parts that makes.
template <typename T>
int split_steps(Product& p, int splits) {
    if (p.sum == 0) return 0;
    p.steps = static_cast<int>(ceil_div(p.sum * static_cast<int64_t>(sizeof(T)), kStepBytes));
    p.steps_per_split = static_cast<int>(ceil_div(p.steps, splits));
    return static_cast<int>(ceil_div(p.steps, p.steps_per_split));
}

template <typename T, bool kAcrossA, bool kAcrossB, End kEnd>
void launch_tiles(hipStream_t st, Product p, const Epilogue& e, TilePlan plan) {
    const int splits = split_steps<T>(p, plan.splits);
    auto launch = [&](auto bm, auto bn, auto wm, auto wn, auto slots_a, auto slots_b) {
        constexpr int BM = decltype(bm)::value, BN = decltype(bn)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
        p.tiles_m = static_cast<int>(ceil_div(p.m, BM));
        p.tiles_n = static_cast<int>(ceil_div(p.n, BN));
        const dim3 grid(static_cast<unsigned>(p.tiles_m * p.tiles_n), static_cast<unsigned>(splits));
        hipLaunchKernelGGL((linear_tile_kernel<T, BM, BN, WM, WN, decltype(slots_a)::value, decltype(slots_b)::value, kAcrossA, kAcrossB, kEnd>), grid, dim3(WM * WN * kWave),
                           0, st, p, e);
    };
    constexpr std::integral_constant<int, 1> k1;
    constexpr std::integral_constant<int, 2> k2;
    constexpr std::integral_constant<int, 3> k3;
    constexpr std::integral_constant<int, 4> k4;
    constexpr std::integral_constant<int, 32> k32;
    constexpr std::integral_constant<int, 64> k64;
    constexpr std::integral_constant<int, 96> k96;
    constexpr std::integral_constant<int, 128> k128;
    constexpr std::integral_constant<int, 256> k256;
    if constexpr (kEnd == kNormalizedLayer) {
        // a block has whole rows: 32 of them where 128 leave CUs idle (and
        // always of 32 bits), the columns in waves of 32
        if constexpr (sizeof(T) == 2) {
            const bool many = ceil_div(ceil_div(p.m, 32), kCus) * 32 >= ceil_div(ceil_div(p.m, 128), kCus) * 128;
            if (many) return launch(k128, k128, k4, k1, k3, k2);
        }
        if (p.n > 96)
            launch(k32, k128, k1, k4, k3, k3);
        else if (p.n > 64)
            launch(k32, k96, k1, k3, k3, k3);
        else
            launch(k64, k64, k2, k2, k3, k2);
    } else {
        if constexpr (sizeof(T) == 2) {
            if (plan.size == 256) return launch(k256, k256, k2, k4, k3, k2);
        }
        if (plan.size == 128)
            launch(k128, k128, k2, k2, k3, k2);
        else
            launch(k64, k64, k2, k2, k3, k2);
    }
}

// Whether a product's loads can take a matrix as it lies: rows that start at
// multiples of 16 bytes and end at one, a tile's rows within 32-bit offsets.
template <typename T>
bool takes_loads(const void* p, int64_t stride, int64_t cols) {
    return rows_aligned(p, stride, sizeof(T)) && cols * static_cast<int64_t>(sizeof(T)) % 16 == 0 &&
           stride * static_cast<int64_t>(sizeof(T)) <= (int64_t{1} << 22);
}

// A matrix as a product reads it: as it lies where its loads can take it, else
// laid out again in `copy` (rows x round_up(cols, 64)) by a job added to jobs.
template <typename T>
void aligned_rows(const void* src, int64_t stride, int64_t rows, int cols, void* copy, const void** p,
                  int64_t* stride_bytes, AlignJob* jobs, int* count) {
    if (takes_loads<T>(src, stride, cols)) {
        *p = src;
        *stride_bytes = stride * static_cast<int64_t>(sizeof(T));
        return;
    }
    const int wide = static_cast<int>(round_up(cols, 64));
    const int64_t chunks = rows * (wide * static_cast<int64_t>(sizeof(T)) / 16);
    jobs[(*count)++] = AlignJob{src, copy, stride, rows, cols, wide,
                                static_cast<int>(std::min<int64_t>(ceil_div(chunks, 256), 65536))};
    *p = copy;
    *stride_bytes = wide * static_cast<int64_t>(sizeof(T));
}

template <typename T>
void launch_align(hipStream_t st, const AlignJob* jobs, int count) {
    if (count == 0) return;
    const AlignJob none = {};
    const AlignJob& second = count > 1 ? jobs[1] : none;
    hipLaunchKernelGGL((linear_align_kernel<T>), dim3(static_cast<unsigned>(jobs[0].blocks + second.blocks)), dim3(256), 0, st,
                       jobs[0], second);
}

struct ForwardPlan {
    void* x;
    void* weight;
};
// Room for `rows` rows of X laid out again, and for W.
size_t carve_forward(const chimera_linear_shape& s, int64_t rows, void* base, ForwardPlan* plan) {
    Carve c{static_cast<char*>(base)};
    const size_t wide = round_up(s.in_features, 64) * type_bytes(s.type);
    plan->weight = c.take(static_cast<size_t>(s.out_features) * wide);
    plan->x = c.take(static_cast<size_t>(rows) * wide);
    return c.off;
}

bool few_rows(const chimera_linear_shape& s) { return s.rows <= kFewRows && !s.normalize; }

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
    e.act = s.activation == CHIMERA_ACT_GELU && out == 2 ? kRoundedGelu : s.activation;
    e.out_f32 = out == 4;
    e.normalize = s.normalize != 0;
    Product p = {};
    p.m = s.rows;
    p.n = s.out_features;
    if (few_rows(s)) {
        p.a = a.x;
        p.b = a.weight;
        p.a_stride = a.x_stride * static_cast<int64_t>(sizeof(T));
        p.b_stride = a.weight_stride * static_cast<int64_t>(sizeof(T));
        p.sum = s.in_features;
        const dim3 grid(static_cast<unsigned>(ceil_div(s.out_features, 4 * kWaveOutputs)));
        switch (s.rows) {
            case 1: hipLaunchKernelGGL((linear_vector_kernel<T, 1>), grid, dim3(256), 0, st, p, e); break;
            case 2: hipLaunchKernelGGL((linear_vector_kernel<T, 2>), grid, dim3(256), 0, st, p, e); break;
            case 3: hipLaunchKernelGGL((linear_vector_kernel<T, 3>), grid, dim3(256), 0, st, p, e); break;
            default: hipLaunchKernelGGL((linear_vector_kernel<T, 4>), grid, dim3(256), 0, st, p, e);
        }
        return hipGetLastError();
    }
    ForwardPlan plan;
    (void)carve_forward(s, s.rows, a.workspace, &plan);  // X's room comes last: it is not there where X needs none
    AlignJob jobs[2];
    int njobs = 0;
    aligned_rows<T>(a.x, a.x_stride, s.rows, s.in_features, plan.x, &p.a, &p.a_stride, jobs, &njobs);
    aligned_rows<T>(a.weight, a.weight_stride, s.out_features, s.in_features, plan.weight, &p.b, &p.b_stride, jobs, &njobs);
    launch_align<T>(st, jobs, njobs);
    // whole chunks: as the matrices lie, or both laid out again with zeros
    p.sum = round_up(s.in_features, 16 / sizeof(T));
    const TilePlan tiles = tile_plan(p.m, p.n, p.sum, sizeof(T), false, 1);
    if (e.normalize)
        launch_tiles<T, false, false, kNormalizedLayer>(st, p, e, tiles);
    else
        launch_tiles<T, false, false, kPlainLayer>(st, p, e, tiles);
    return hipGetLastError();
}

struct BackwardPlan {
    int n_pad;
    int block_rows;  // of the gradient kernel
    TilePlan dweight;
    void *g, *x, *weight;
    float *sums, *parts;
};

// Parts that dW's sum may have, and that the workspace has room for: those of
// a few tiles of 64 a CU (64 MB), or as many as take the room of X and dZ laid
// out again where that is more. Grows with the rows only, so that a workspace
// sized for some rows serves fewer; the least estimate without a bound lies
// beyond it for 2 of 60,000 random shapes, where it costs 1 and 3 %.
int64_t most_parts(int64_t rows, int64_t n, int64_t k, size_t elem) {
    const int64_t e = static_cast<int64_t>(elem);
    const int64_t tiles = ceil_div(n, 64) * ceil_div(k, 64);
    const int64_t most = std::min<int64_t>(
        {256, std::max<int64_t>(16 * kCus / tiles, rows * e * (n + k) / (4 * n * k)), ceil_div(rows * e, kStepBytes) / 8});
    int64_t parts = 1;
    while (parts * 2 <= most) parts *= 2;
    return parts;
}

size_t carve_backward(const chimera_linear_shape& s, void* base, BackwardPlan* plan) {
    Carve c{static_cast<char*>(base)};
    const size_t e = type_bytes(s.type);
    const size_t k = static_cast<size_t>(s.in_features), n = static_cast<size_t>(s.out_features);
    const size_t wide = round_up(s.in_features, 64) * e;
    plan->n_pad = static_cast<int>(round_up(s.out_features, 64));
    // about 1,024 blocks of 16 to 512 rows
    plan->block_rows = static_cast<int>(std::max<int64_t>(
        16, std::min<int64_t>(512, round_up(ceil_div(s.rows * ceil_div(s.out_features, 128), 1024), 16))));
    const int64_t most = most_parts(s.rows, s.out_features, s.in_features, e);
    plan->dweight = tile_plan(s.out_features, s.in_features, s.rows, e, true, most);
    // blocks of any number of rows up to these
    const int64_t most_blocks = std::min<int64_t>(
        ceil_div(s.rows, 16), std::max<int64_t>(ceil_div(1024, ceil_div(s.out_features, 128)), ceil_div(s.rows, 512)));
    plan->g = c.take(static_cast<size_t>(s.rows) * plan->n_pad * e);
    plan->x = c.take(static_cast<size_t>(s.rows) * wide);
    plan->weight = c.take(n * wide);
    plan->sums = static_cast<float*>(c.take(static_cast<size_t>(most_blocks) * n * 4));
    plan->parts = static_cast<float*>(c.take(most > 1 ? static_cast<size_t>(most) * n * k * 4 : 0));
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
    const size_t out = type_bytes(s.out_type);
    // where dZ is dY as it lies, the products read dY
    const bool as_it_is = s.activation == CHIMERA_ACT_NONE && !s.normalize && out == sizeof(T) &&
                          takes_loads<T>(a.dy, a.dy_stride, n);
    const bool products = a.dx || a.dweight;
    GradArgs g = {};
    g.dy = a.dy;
    g.y = a.y;
    g.saved = a.saved;
    g.norms = a.norms;
    g.dresidual = a.dresidual;
    g.g = products && !as_it_is ? plan.g : nullptr;
    g.sums = a.dbias ? plan.sums : nullptr;
    g.dy_stride = a.dy_stride;
    g.y_stride = a.y_stride;
    g.saved_stride = a.saved_stride;
    g.dresidual_stride = a.dresidual_stride;
    g.m = s.rows;
    g.n = n;
    g.g_cols = plan.n_pad;
    g.act = s.activation;
    g.block_rows = plan.block_rows;
    g.out_f32 = out == 4;
    g.normalize = s.normalize != 0;
    const int64_t blocks = ceil_div(s.rows, plan.block_rows);
    if (g.g || g.sums || g.dresidual)
        hipLaunchKernelGGL((linear_grad_kernel<T>),
                           dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(ceil_div(n, 128))), dim3(256), 0, st, g);
    const void* dz = as_it_is ? a.dy : plan.g;
    const int64_t dz_stride = (as_it_is ? a.dy_stride : plan.n_pad) * static_cast<int64_t>(sizeof(T));
    auto product_to = [&](Product& p, Epilogue& e, int64_t m, int cols, int64_t sum, void* dst, int64_t stride) {
        p.a = dz;
        p.a_stride = dz_stride;
        p.m = e.m = m;
        p.n = e.n = cols;
        p.sum = sum;
        e.y = dst;
        e.y_stride = stride;
        e.out_f32 = sizeof(T) == 4;
    };
    Product px = {}, pw = {};
    Epilogue ex = {}, ew = {};
    TilePlan tiles_x = {};
    AlignJob jobs[2];
    int njobs = 0;
    if (a.dx) {
        product_to(px, ex, s.rows, k, n, a.dx, a.dx_stride);
        tiles_x = tile_plan(px.m, px.n, px.sum, sizeof(T), true, 1);
        aligned_rows<T>(a.weight, a.weight_stride, n, k, plan.weight, &px.b, &px.b_stride, jobs, &njobs);
    }
    if (a.dweight) {
        product_to(pw, ew, n, k, s.rows, a.dweight, a.dweight_stride);
        aligned_rows<T>(a.x, a.x_stride, s.rows, k, plan.x, &pw.b, &pw.b_stride, jobs, &njobs);
        if (plan.dweight.splits > 1) ew.partial = plan.parts;
    }
    launch_align<T>(st, jobs, njobs);
    const int parts = split_steps<T>(pw, plan.dweight.splits);
    if (a.dx && a.dweight && tiles_x.size == 64 && plan.dweight.size == 64) {
        split_steps<T>(px, 1);
        for (Product* p : {&pw, &px}) {
            p->tiles_m = static_cast<int>(ceil_div(p->m, 64));
            p->tiles_n = static_cast<int>(ceil_div(p->n, 64));
        }
        const int64_t blocks = static_cast<int64_t>(pw.tiles_m) * pw.tiles_n * parts + static_cast<int64_t>(px.tiles_m) * px.tiles_n;
        hipLaunchKernelGGL((linear_gradients_kernel<T>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, pw, ew, parts,
                           px, ex);
    } else {
        if (a.dx) launch_tiles<T, false, true, kSums>(st, px, ex, tiles_x);
        if (a.dweight) launch_tiles<T, true, true, kSums>(st, pw, ew, plan.dweight);
    }
    Join jw = {}, jb = {};
    int64_t w_blocks = 0, b_blocks = 0;
    if (ew.partial) {
        jw = Join{plan.parts, a.dweight, a.dweight_stride, static_cast<int64_t>(n) * k, parts, k};
        w_blocks = ceil_div(jw.count, k % 4 == 0 ? 2048 : 512);
    }
    if (a.dbias) {
        jb = Join{plan.sums, a.dbias, n, n, static_cast<int>(blocks), n};
        b_blocks = ceil_div(n, kWave);
    }
    if (w_blocks + b_blocks > 0)
        hipLaunchKernelGGL((linear_join_kernel<T>), dim3(static_cast<unsigned>(w_blocks + b_blocks)), dim3(512), 0, st, jw,
                           static_cast<int>(w_blocks), jb);
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

size_t linear_forward_workspace(const chimera_linear_shape& s) {
    ForwardPlan plan;
    return carve_forward(s, s.rows, nullptr, &plan);
}
size_t linear_forward_workspace(const LinearForward& f) {
    const bool taken = by_type(f.s.type, [&](auto t) { return takes_loads<decltype(t)>(f.a.x, f.a.x_stride, f.s.in_features); });
    ForwardPlan plan;
    return carve_forward(f.s, taken || few_rows(f.s) ? 0 : f.s.rows, nullptr, &plan);
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
