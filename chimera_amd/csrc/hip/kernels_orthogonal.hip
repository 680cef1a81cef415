// The update of a weight made orthogonal by Newton-Schulz products
// (include/chimera_operators.h):
//   M' = mu M + G,  U = G, M' or G + mu M',  X = U / |U|
//   X <- a X + (b A + c A^2) X with A = X X^T, `steps` times
//   W' = (1 - decay) W - rate X
// X lies on its shorter side [m, k], m <= k, and its transpose beside it, so
// that the rows of all products lie along their sums.
//
// Small singular values grow up to a^steps times, and with them every error,
// so X, A and B = b A + c A^2 are held to 22 bits: a value is two fp16 parts,
// times 2^8, which leaves room up to 255, the lower one times another 2^11. So
// both are normal numbers down to 2^-22, below which values are 2^-43 apart.
// (With one factor for both, values are 2^-32 apart from 2^-11 down; 1024 x 1024
// with rows that are 1e-5 of one row was off by 4.9e-5 of the result instead of
// 5e-7, and took 164 us instead of 167.) A product is hi hi + (hi lo + lo hi)
// 2^-11 on the matrix cores, two sums in 32 bits. That is as near to 64 bits as
// 32-bit products are (1e-7 to 2e-6 of the result's size at 300 to 1,024
// columns, those 3e-8 to 1e-5; one fp16 part gives 2e-3), at twice their rate:
// 4096 x 4096 takes 894 us a step, 310 TF of results where 32 bits reach 154.
#include "dense_tile.hpp"

namespace chimera {

namespace {

constexpr float kPairScale = 256.0f;
constexpr float kUnscale = 1.0f / kPairScale, kUnscaleSum = kUnscale * kUnscale;
constexpr float kLowScale = 2048.0f, kUnscaleLow = 1.0f / kLowScale;

// ---- pairs ---------------------------------------------------------------------

// A row of pairs is steps of 128 bytes with 32 values each: chunks of eight,
// hi 0..7, hi 8..15, lo 0..7, lo 8..15 and the same of the other 16, so that a
// quarter of a step is 16 values' upper or lower parts. Columns up to the end
// of a step are zeros.
struct Pairs {
    unsigned char* p;
    int64_t stride;  // bytes, a multiple of 128
};
__device__ __forceinline__ int64_t pair_chunk(int col) {  // the bytes of eight upper parts; the lower ones are 32 on
    return static_cast<int64_t>(col / 32) * 128 + (col & 16) * 4 + (col & 8) * 2;
}
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    const float s = v * kPairScale;
    hi = from_float<_Float16>(s);
    lo = from_float<_Float16>((s - to_float(hi)) * kLowScale);
}
__device__ __forceinline__ float join(_Float16 hi, _Float16 lo) { return fmaf(to_float(lo), kUnscaleLow, to_float(hi)); }
__device__ __forceinline__ void store_pairs(const Pairs& m, int64_t row, int col, const float (&v)[8]) {
    _Float16 hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) split(v[i], hi[i], lo[i]);
    unsigned char* to = m.p + row * m.stride + pair_chunk(col);
    *reinterpret_cast<u32x4_t*>(to) = *reinterpret_cast<const u32x4_t*>(hi);
    *reinterpret_cast<u32x4_t*>(to + 32) = *reinterpret_cast<const u32x4_t*>(lo);
}
// ---- what goes before the products ---------------------------------------------

struct Update {
    const void* gradient;
    const float* momentum;
    float* new_momentum;
    float* u;       // [rows][cols]
    double* parts;  // [blocks]: sums of U^2
    int64_t gradient_stride, momentum_stride, new_momentum_stride;
    int rows, cols;
    int blocks;
    float mu;
    bool nesterov;
};

// U, the new momentum, and the sums of U^2 by blocks in 64 bits: squares of
// any 32-bit values fit, and the norm is right to the last bit of 32, which
// matters because all singular values move with it.
template <typename T>
__global__ __launch_bounds__(256) void orthogonal_update_kernel(Update a) {
    __shared__ double sums[4];
    const int units = (a.cols + 7) / 8;
    const int64_t total = static_cast<int64_t>(a.rows) * units;
    double sum = 0.0;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += a.blocks * 256ll) {
        const int64_t r = i / units;
        const int c = static_cast<int>(i - r * units) * 8, count = a.cols - c;
        float g[8];
        load8(static_cast<const T*>(a.gradient) + r * a.gradient_stride + c, count, g);
        if (a.momentum) {
            float m[8];
            load8(a.momentum + r * a.momentum_stride + c, count, m);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                m[j] = fmaf(a.mu, m[j], g[j]);
                g[j] = a.nesterov ? fmaf(a.mu, m[j], g[j]) : m[j];
            }
            store8(a.new_momentum + r * a.new_momentum_stride + c, count, m);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) sum = fma(static_cast<double>(g[j]), static_cast<double>(g[j]), sum);
        store8(a.u + r * a.cols + c, count, g);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (lane_id() == 0) sums[wave_id()] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.parts[blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// A tile of values as pairs: rows [row0, row0 + rows) of `along` from column
// col0 on, and the transposed tile of `across`. Columns up to the end of a step
// are written, from values that are zeros there.
template <int BM, int BN, int kThreads>
__device__ __forceinline__ void put_tile(const float* tile, int rows, int cols, const Pairs& along, int64_t row0,
                                         const Pairs& across, int64_t col0) {
    constexpr int kPitch = BN + 1;
    const int wide = (cols + 31) / 32 * 32, high = (rows + 31) / 32 * 32;
    for (int i = static_cast<int>(threadIdx.x); i < BM * BN / 8; i += kThreads) {
        const int r = i / (BN / 8), c = i % (BN / 8) * 8;
        if (r >= rows || c >= wide) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tile[r * kPitch + c + j];
        store_pairs(along, row0 + r, static_cast<int>(col0) + c, v);
    }
    for (int i = static_cast<int>(threadIdx.x); i < BM * BN / 8; i += kThreads) {
        const int c = i / (BM / 8), r = i % (BM / 8) * 8;
        if (c >= cols || r >= high) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = tile[(r + j) * kPitch + c];
        store_pairs(across, col0 + c, static_cast<int>(row0) + r, v);
    }
}

constexpr int kMostBlocks = 256;  // of the update, whose sums a block of the scaling adds up

// X = U / |U| as pairs, along and across; a U of zeros stays zeros.
__global__ __launch_bounds__(256) void orthogonal_scale_kernel(const float* u, const double* parts, int count, int rows,
                                                               int cols, Pairs along, Pairs across) {
    constexpr int kPitch = 65;
    __shared__ float tile[64 * kPitch];
    __shared__ double sums[4];
    const int row0 = static_cast<int>(blockIdx.y) * 64, col0 = static_cast<int>(blockIdx.x) * 64;
    const int r0 = static_cast<int>(threadIdx.x) / 8, c0 = static_cast<int>(threadIdx.x) % 8 * 8;
    float v[2][8] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (row0 + r0 + 32 * i < rows && col0 + c0 < cols)
            load8(u + static_cast<int64_t>(row0 + r0 + 32 * i) * cols + col0 + c0, cols - col0 - c0, v[i]);
    double sum = static_cast<int>(threadIdx.x) < count ? parts[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (lane_id() == 0) sums[wave_id()] = sum;
    __syncthreads();
    sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const double by = sum == 0.0 ? 0.0 : 1.0 / sqrt(sum);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[(r0 + 32 * i) * kPitch + c0 + j] = static_cast<float>(v[i][j] * by);
    __syncthreads();
    put_tile<64, 64, 256>(tile, min(64, rows - row0), min(64, cols - col0), along, row0, across, col0);
}

// ---- products ------------------------------------------------------------------

enum Kind { kGram, kSquare, kApply, kLast };

struct Finish {
    void* out;            // or NULL
    const float* weight;  // or NULL
    float* new_weight;
    void* rounded;  // or NULL
    int64_t out_stride, weight_stride, new_weight_stride, rounded_stride;
    float keep, rate;
    int type;
    bool out_f32, turned;  // turned: X is the transpose of what is asked for
};

struct Schulz {
    Product p;      // of pairs: p.sum and steps in steps of 32 values
    Pairs from;     // what the sums are added to: A, or X
    Pairs along;    // the result
    Pairs across;   // its transpose
    float from_by, sum_by;
    float linear_by, square_by;  // B = linear_by A + square_by A^2, where a kernel makes it itself
    Finish f;
};

// Which tile of a symmetric result the t-th on and below the diagonal is.
__device__ __forceinline__ void below_diagonal(int t, int* tm, int* tn) {
    int m = static_cast<int>((sqrtf(8.0f * static_cast<float>(t) + 1.0f) - 1.0f) * 0.5f);
    while ((m + 1) * (m + 2) / 2 <= t) ++m;
    while (m * (m + 1) / 2 > t) --m;
    *tm = m;
    *tn = t - m * (m + 1) / 2;
}

// Eight neighbours of a row of the result.
template <typename T>
__device__ __forceinline__ void put8(const Finish& f, int64_t row, int64_t col, int count, const float (&v)[8]) {
    if (f.out) {
        if (f.out_f32)
            store8(static_cast<float*>(f.out) + row * f.out_stride + col, count, v);
        else
            store8(static_cast<T*>(f.out) + row * f.out_stride + col, count, v);
    }
    if (f.weight) {
        float w[8];
        load8(f.weight + row * f.weight_stride + col, count, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = fmaf(f.keep, w[j], -f.rate * v[j]);
        store8(f.new_weight + row * f.new_weight_stride + col, count, w);
        if (f.rounded) store8(static_cast<T*>(f.rounded) + row * f.rounded_stride + col, count, w);
    }
}
__device__ __forceinline__ void finish8(const Finish& f, int64_t row, int64_t col, int count, const float (&v)[8]) {
    switch (f.type) {
        case CHIMERA_F32: put8<float>(f, row, col, count, v); break;
        case CHIMERA_F16: put8<_Float16>(f, row, col, count, v); break;
        default: put8<__bf16>(f, row, col, count, v);
    }
}

template <Kind kKind>
constexpr bool kSymmetric = kKind == kGram || kKind == kSquare;

struct Place {
    int tm, tn;
};

// Blocks go round the 8 XCDs; each takes a run of tiles, so that an L2 holds what
// its blocks share.
template <Kind kKind>
__device__ __forceinline__ Place place(const Schulz& a) {
    const int id = static_cast<int>(blockIdx.x), xcd = id % 8, tiles = static_cast<int>(gridDim.x);
    const int tile = xcd * (tiles / 8) + min(xcd, tiles % 8) + id / 8;
    Place o;
    if constexpr (kSymmetric<kKind>) {
        below_diagonal(tile, &o.tm, &o.tn);
    } else {
        o.tm = tile % a.p.tiles_m;
        o.tn = tile / a.p.tiles_m;
    }
    return o;
}

// A tile's result from the sums in LDS, of kSums equal parts: C = from_by F +
// sum_by C, stored along and across. A thread takes eights of a row; F's are
// loaded before the sums are there.
template <Kind kKind, int B, int kSums, int kThreads>
struct Result {
    static constexpr int kPitch = B + 4, kTurned = B + 1, kSumBytes = kSums * B * kPitch * 4;
    static constexpr int kBytes = kSumBytes + B * kTurned * 4;
    static constexpr int kEights = (B * B / 8 + kThreads - 1) / kThreads;
    static constexpr bool kAdds = kKind != kGram;
    int rows, cols;  // of the tile, and with those up to the end of a step
    int high, wide;
    int64_t m0, n0;
    f16x8_t hi[kEights], lo[kEights];

    __device__ __forceinline__ int row(int i) const { return (i * kThreads + static_cast<int>(threadIdx.x)) / (B / 8); }
    __device__ __forceinline__ int col(int i) const { return (i * kThreads + static_cast<int>(threadIdx.x)) % (B / 8) * 8; }
    __device__ __forceinline__ void init(const Schulz& a, const Place& at) {
        m0 = static_cast<int64_t>(at.tm) * B;
        n0 = static_cast<int64_t>(at.tn) * B;
        rows = static_cast<int>(min(a.p.m - m0, int64_t{B}));
        cols = static_cast<int>(min(a.p.n - n0, int64_t{B}));
        high = static_cast<int>(min((a.p.m + 31) / 32 * 32 - m0, int64_t{B}));
        wide = static_cast<int>(min((a.p.n + 31) / 32 * 32 - n0, int64_t{B}));
    }
    __device__ __forceinline__ void load(const Schulz& a) {
        if constexpr (kAdds) {
#pragma unroll
            for (int i = 0; i < kEights; ++i) {
                hi[i] = lo[i] = f16x8_t{};
                if (row(i) < rows && col(i) < cols) {
                    const unsigned char* from = a.from.p + (m0 + row(i)) * a.from.stride + pair_chunk(static_cast<int>(n0) + col(i));
                    hi[i] = *reinterpret_cast<const f16x8_t*>(from);
                    lo[i] = *reinterpret_cast<const f16x8_t*>(from + 32);
                }
            }
        }
    }
    // four neighbours of a row
    static __device__ __forceinline__ void put(unsigned char* lds, int sum, int row, int col, const f32x4_t& v) {
        *reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(lds) + (sum * B + row) * kPitch + col) = v;
    }
    // 16 values of a lane: of row `row` of the tile and of part `sum`
    static __device__ __forceinline__ void put(unsigned char* lds, int sum, int row, int col0, const f32x16_t& v) {
        float* to = reinterpret_cast<float*>(lds) + (sum * B + row) * kPitch + col0 + 4 * (lane_id() >> 5);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4_t*>(to + 8 * q) = f32x4_t{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    }
    __device__ __forceinline__ void store(const Schulz& a, const Place& at, unsigned char* lds) const {
        const float* sums = reinterpret_cast<const float*>(lds);
        float* turned = reinterpret_cast<float*>(lds + kSumBytes);
        const bool across = kKind == kLast ? a.f.turned : !(kSymmetric<kKind> && at.tm == at.tn);
#pragma unroll
        for (int i = 0; i < kEights; ++i) {
            const int r = row(i), c = col(i);
            if (r >= high) break;
            float v[8] = {};
#pragma unroll
            for (int o = 0; o < kSums; ++o) {
                const f32x4_t* from = reinterpret_cast<const f32x4_t*>(sums + (o * B + r) * kPitch + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += from[j / 4][j % 4];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] *= a.sum_by;
                if constexpr (kAdds) v[j] = fmaf(a.from_by * kUnscale, join(hi[i][j], lo[i][j]), v[j]);
                v[j] = r < rows && c + j < cols ? v[j] : 0.0f;
            }
            if constexpr (kKind == kLast) {
                if (!across && r < rows && c < cols) finish8(a.f, m0 + r, n0 + c, cols - c, v);
            } else {
                if (r < rows && c < wide) store_pairs(a.along, m0 + r, static_cast<int>(n0) + c, v);
            }
            if (across) {
#pragma unroll
                for (int j = 0; j < 8; ++j) turned[r * kTurned + c + j] = v[j];
            }
        }
        if (!across) return;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEights; ++i) {
            const int c = row(i), r = col(i);
            if (c >= cols || r >= high) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = turned[(r + j) * kTurned + c];
            if constexpr (kKind == kLast) {
                if (r < rows) finish8(a.f, n0 + c, m0 + r, rows - r, v);
            } else {
                store_pairs(a.across, n0 + c, static_cast<int>(m0) + r, v);
            }
        }
    }
};

// The sums of I x J tiles: of the upper parts' products and of an upper and a
// lower part's, 2^11 times as large.
template <typename Tile, int I, int J = I>
struct Sums {
    Tile high[I][J] = {}, low[I][J] = {};

    __device__ __forceinline__ Tile value(int i, int j) const {
        Tile v;
#pragma unroll
        for (int q = 0; q < static_cast<int>(sizeof(Tile) / sizeof(float)); ++q) v[q] = fmaf(low[i][j][q], kUnscaleLow, high[i][j][q]);
        return v;
    }
};

// The parts of a half step that a wave multiplies: I x J tiles of 32 x 32.
template <int I, int J>
struct Halves {
    u32x4_t ah[I], al[I], bh[J], bl[J];

    __device__ __forceinline__ void multiply(Sums<f32x16_t, I, J>& sums) const {
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < I; ++i)
#pragma unroll
                for (int j = 0; j < J; ++j)
                    sums.low[i][j] = mma32<_Float16>(k == 1 ? bl[j] : bh[j], k == 0 ? al[i] : ah[i], sums.low[i][j]);
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) sums.high[i][j] = mma32<_Float16>(bh[j], ah[i], sums.high[i][j]);
        // with the reads of the half step after it in between
        constexpr int kMfmas = 3 * I * J, kReads = 2 * (I + J), kPer = (kReads + kMfmas - 1) / kMfmas;
#pragma unroll
        for (int g = 0; g < kReads / kPer; ++g) {
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, kPer, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
};

// A step's loads with the address in scalar registers and a lane's offset beside
// it: where the compiler can see the address it keeps each load's sum of the two
// in vector registers over the loop, and spills (768 x 768 159 us, so 143).
template <typename Part>
__device__ __forceinline__ void fetch_step(const Part& part, int s, unsigned char* to, int l) {
    Part from = part;
    asm volatile("" : "+s"(from.base));
    from.fetch(s, to, true, 0, l);
}

// Until at most kUnderWay of this wave's loads are under way and its LDS reads have come.
template <int kUnderWay>
__device__ __forceinline__ void arrived() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((kUnderWay & 15) | (kUnderWay >> 4 << 14) | (7 << 4));
    asm volatile("" ::: "memory");
}

// C = P Q^T of pairs on a tile of B x B, for results of few tiles. Each of kWaves
// waves takes the whole tile and every kWaves-th step of the sum, with LDS slots
// of its own that the operands go straight to, so that the loop has no meeting.
// With two slots half a step's parts, upper and lower, are read while the half
// before it is multiplied; with one a step is read, and the next one's loads
// pass under its products. Of the symmetric results only tiles on and below the
// diagonal are computed. A step of a tile of 64 is 256 cycles of loads into LDS
// (64 bytes a cycle) and 96 of the matrix cores. 1024 x 1024 x 1024 takes 9 us
// in its blocks: 2 until the first loads are there, 4.3 of loop (50 bytes a
// cycle), and 2 for the sums and what is stored, which waves without a share of
// the sum (kAll in all) halve.
template <Kind kKind, int B, int kWaves, int kSlots, int kAll = kWaves>
__global__ __launch_bounds__(kAll* kWave) void orthogonal_few_kernel(Schulz a) {
    constexpr int I = B / 32;
    using Part = Side<float, B, 1, false>;
    using End = Result<kKind, B, kWaves, kAll * kWave>;
    constexpr int kSlot = 2 * Part::kBytes, kLoads = 2 * Part::kLoads, kRings = kWaves * kSlots * kSlot;
    __shared__ __align__(1024) unsigned char lds[kRings > End::kBytes ? kRings : End::kBytes];
    const Product& p = a.p;
    const int l = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
    const Place at = place<kKind>(a);
    End end;
    end.init(a, at);
    const int steps = w < kWaves ? (p.steps - w + kWaves - 1) / kWaves : 0;  // of this wave
    Part side_a, side_b;
    side_a.init(p.a, p.a_stride, end.m0, p.m, w, 0, l);
    side_b.init(p.b, p.b_stride, end.n0, p.n, w, 0, l);
    Reader<float, I, false, kStepBytes> reader;
    reader.init(0, l);
    unsigned char* const ring = lds + w * kSlots * kSlot;
    auto fetch = [&](int s) {
        unsigned char* to = ring + s % kSlots * kSlot;
        side_a.fetch(kWaves * s, to, true, 0, l);
        side_b.fetch(kWaves * s, to + Part::kBytes, true, 0, l);
    };
    auto read = [&](int s, int h, Halves<I, I>& o) {
        const unsigned char* from = ring + s % kSlots * kSlot;
        reader.read(from, 2 * h + 1, o.al);
        reader.read(from + Part::kBytes, 2 * h, o.bh);
        reader.read(from, 2 * h, o.ah);
        reader.read(from + Part::kBytes, 2 * h + 1, o.bl);
    };
    end.load(a);
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
        if (s < steps) fetch(s);
    Sums<f32x16_t, I> acc;
    if (steps > 0) {
        Halves<I, I> even, odd;
        if (steps >= kSlots)
            arrived<(kSlots - 1) * kLoads>();
        else
            arrived<0>();
        read(0, 0, even);
        int s = 0;
        for (; s + kSlots < steps; ++s) {
            read(s, 1, odd);
            if constexpr (kSlots > 1) even.multiply(acc);
            arrived<63>();  // the reads: the slot takes new loads
            fetch(s + kSlots);
            if constexpr (kSlots == 1) {
                even.multiply(acc);
                odd.multiply(acc);
            }
            arrived<(kSlots - 1) * kLoads>();  // the next step's loads
            read(s + 1, 0, even);
            if constexpr (kSlots > 1) odd.multiply(acc);
        }
        for (; s < steps; ++s) {
            read(s, 1, odd);
            even.multiply(acc);
            arrived<0>();
            if (s + 1 < steps) read(s + 1, 0, even);
            odd.multiply(acc);
        }
    }
    __syncthreads();
    if (w < kWaves) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < I; ++j) End::put(lds, w, 32 * i + (l & 31), 32 * j, acc.value(i, j));
    }
    __syncthreads();
    end.store(a, at, lds);
}

// The same for tiles of 48, in products of 16 x 16: of symmetric results up to 22
// such tiles a side each CU then has one, where tiles of 64 leave half of the CUs
// idle and load a third more for each. A step is read while the one before it is
// multiplied.
template <Kind kKind>
__global__ __launch_bounds__(512) void orthogonal_few48_kernel(Schulz a) {
    constexpr int B = 48, I = B / 16, kWaves = 4, kSlots = 3;
    using Part = Side<float, B, 1, false>;
    using End = Result<kKind, B, kWaves, 512>;
    constexpr int kSlot = 2 * Part::kBytes, kLoads = 2 * Part::kLoads, kRings = kWaves * kSlots * kSlot;
    __shared__ __align__(1024) unsigned char lds[kRings > End::kBytes ? kRings : End::kBytes];
    const Product& p = a.p;
    const int l = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
    const Place at = place<kKind>(a);
    End end;
    end.init(a, at);
    const int steps = w < kWaves ? (p.steps - w + kWaves - 1) / kWaves : 0;  // of this wave
    Part side_a, side_b;
    side_a.init(p.a, p.a_stride, end.m0, p.m, w, 0, l);
    side_b.init(p.b, p.b_stride, end.n0, p.n, w, 0, l);
    unsigned char* const ring = lds + w * kSlots * kSlot;
    auto fetch = [&](int s) {
        unsigned char* to = ring + s % kSlots * kSlot;
        fetch_step(side_a, kWaves * s, to, l);
        fetch_step(side_b, kWaves * s, to + Part::kBytes, l);
    };
    // lane l's eight of row l % 16 is the l / 16-th of the step, upper parts
    // here, lower ones two chunks on
    const int group = l >> 4, place16 = ((group >> 1) * 4 + (group & 1)) ^ ((l >> 1) & 7);
    const int off = (l & 15) * kStepBytes + (place16 << 4);
    struct Operands {
        u32x4_t ah[I], al[I], bh[I], bl[I];
    };
    auto read = [&](int s, Operands& o) {
        const unsigned char* from = ring + s % kSlots * kSlot;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const unsigned char *x = from + 16 * i * kStepBytes, *y = x + Part::kBytes;
            o.al[i] = *reinterpret_cast<const u32x4_t*>(x + (off ^ 32));
            o.bh[i] = *reinterpret_cast<const u32x4_t*>(y + off);
            o.ah[i] = *reinterpret_cast<const u32x4_t*>(x + off);
            o.bl[i] = *reinterpret_cast<const u32x4_t*>(y + (off ^ 32));
        }
    };
    Sums<f32x4_t, I> acc;
    auto multiply = [&](const Operands& o) {
        auto product = [](u32x4_t x, u32x4_t y, f32x4_t sum) {
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, x), __builtin_bit_cast(f16x8_t, y), sum, 0, 0, 0);
        };
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int i = 0; i < I; ++i)
#pragma unroll
                for (int j = 0; j < I; ++j)
                    acc.low[i][j] = product(k == 1 ? o.bl[j] : o.bh[j], k == 0 ? o.al[i] : o.ah[i], acc.low[i][j]);
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < I; ++j) acc.high[i][j] = product(o.bh[j], o.ah[i], acc.high[i][j]);
#pragma unroll
        for (int g = 0; g < 4 * I; ++g) {
            __builtin_amdgcn_sched_group_barrier(kSchedMfma, 2, 0);
            __builtin_amdgcn_sched_group_barrier(kSchedLdsRead, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    end.load(a);
#pragma unroll
    for (int s = 0; s < kSlots; ++s)
        if (s < steps) fetch(s);
    if (steps > 0) {
        Operands even, odd;
        if (steps >= kSlots)
            arrived<(kSlots - 1) * kLoads>();
        else
            arrived<0>();
        read(0, even);
        // `now` has come from LDS for step s; the next step's into `then`
        auto turn = [&](int s, Operands& now, Operands& then) {
            arrived<63>();  // the reads: the slot takes new loads
            if (s + kSlots < steps) {
                fetch(s + kSlots);
                arrived<(kSlots - 1) * kLoads>();
            } else {
                arrived<0>();
            }
            if (s + 1 < steps) read(s + 1, then);
            multiply(now);
        };
        int s = 0;
        for (; s + 1 < steps; s += 2) {
            turn(s, even, odd);
            turn(s + 1, odd, even);
        }
        if (s < steps) turn(s, even, odd);
    }
    __syncthreads();
    if (w < kWaves) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < I; ++j) End::put(lds, w, 16 * i + (l & 15), 16 * j + 4 * group, acc.value(i, j));
    }
    __syncthreads();
    end.store(a, at, lds);
}

// X' = a X + B X for a shorter side of at most 128 with B = b A + c A^2 made on
// the way, which saves a launch: 5 us where the two take 8. A block takes 32 x 32 of X'; a wave makes 32
// columns of B's 32 rows, whose places in the lanes are, after one exchange of
// the half waves, those of the next product's operand: its 32 values of the sum.
template <Kind kKind>
__global__ __launch_bounds__(256) void orthogonal_both_kernel(Schulz a) {
    constexpr int B = 32, kSteps = 4;  // a wave each
    using Part = Side<float, B, 1, false>;
    using End = Result<kKind, B, kSteps, 256>;
    constexpr int kShared = kSteps * Part::kBytes, kOwn = (kSteps + 1) * Part::kBytes, kAll = kShared + kSteps * kOwn;
    __shared__ __align__(1024) unsigned char lds[kAll > End::kBytes ? kAll : End::kBytes];
    const Product& p = a.p;
    const int l = lane_id(), half = l >> 5, w = __builtin_amdgcn_readfirstlane(wave_id());
    const Place at = place<kKind>(a);
    End end;
    end.init(a, at);
    end.load(a);
    unsigned char* const own = lds + kShared + w * kOwn;
    const bool works = w < p.steps;
    if (works) {
        Part rows, columns, values;
        rows.init(p.a, p.a_stride, end.m0, p.m, 0, 0, l);
        rows.fetch(w, lds + w * Part::kBytes, true, 0, l);
        columns.init(p.a, p.a_stride, 32 * w, p.m, 0, 0, l);
        for (int s = 0; s < p.steps; ++s) columns.fetch(s, own + s * Part::kBytes, true, 0, l);
        values.init(p.b, p.b_stride, end.n0, p.n, 0, 0, l);
        values.fetch(w, own + kSteps * Part::kBytes, true, 0, l);
    }
    __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // all loads
    __syncthreads();
    Reader<float, 1, false, kStepBytes> reader;
    reader.init(0, l);
    Sums<f32x16_t, 1> acc;
    if (works) {
        Halves<1, 1> even, odd, x[2];
        auto read = [&](int s, int h, Halves<1, 1>& o) {
            reader.read(lds + s * Part::kBytes, 2 * h + 1, o.al);
            reader.read(own + s * Part::kBytes, 2 * h, o.bh);
            reader.read(lds + s * Part::kBytes, 2 * h, o.ah);
            reader.read(own + s * Part::kBytes, 2 * h + 1, o.bl);
        };
        read(0, 0, even);
        for (int s = 0; s < p.steps; ++s) {
            read(s, 1, odd);
            even.multiply(acc);
            if (s + 1 < p.steps) read(s + 1, 0, even);
            odd.multiply(acc);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            reader.read(own + kSteps * Part::kBytes, 2 * h, x[h].bh);
            reader.read(own + kSteps * Part::kBytes, 2 * h + 1, x[h].bl);
        }
        // this lane's values of B: row l % 32, columns 8 q + 4 half + i of the step
        const f32x16_t square = acc.value(0, 0);
        uint32_t hi[8], lo[8];
        const unsigned char* from = lds + w * Part::kBytes + (l & 31) * kStepBytes;
        const int turn = ((l & 31) >> 1) & 7;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // eights 0 and 1 of the upper parts, of the lower ones, then 2 and 3
            const int chunk = q / 2 * 4 + q % 2;
            const f16x4_t ah = *reinterpret_cast<const f16x4_t*>(from + ((chunk ^ turn) << 4) + 8 * half);
            const f16x4_t al = *reinterpret_cast<const f16x4_t*>(from + (((chunk + 2) ^ turn) << 4) + 8 * half);
            _Float16 h[4], r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                split(fmaf(a.linear_by, join(ah[i], al[i]), a.square_by * square[4 * q + i]), h[i], r[i]);  // as Result's
            __builtin_memcpy(&hi[2 * q], h, 8);
            __builtin_memcpy(&lo[2 * q], r, 8);
        }
        acc = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            auto operand = [&](const uint32_t* u) {
                const auto x = __builtin_amdgcn_permlane32_swap(u[4 * h], u[4 * h + 2], false, false);
                const auto y = __builtin_amdgcn_permlane32_swap(u[4 * h + 1], u[4 * h + 3], false, false);
                return u32x4_t{x[0], y[0], x[1], y[1]};
            };
            x[h].ah[0] = operand(hi);
            x[h].al[0] = operand(lo);
            x[h].multiply(acc);
        }
    }
    __syncthreads();
    End::put(lds, w, l & 31, 0, acc.value(0, 0));
    __syncthreads();
    end.store(a, at, lds);
}

// The same for many tiles: the block's WM x WN waves divide the tile and share a
// ring of kSlots slots, with one meeting a step. The loads of a step are issued
// in two halves between the products.
template <Kind kKind, int B, int WM, int WN, int kSlots>
__global__ __launch_bounds__(WM* WN* kWave) void orthogonal_tile_kernel(Schulz a) {
    constexpr int W = WM * WN, TM = B / WM, TN = B / WN, I = TM / 32, J = TN / 32;
    using Part = Side<float, B, W, false>;
    using End = Result<kKind, B, 1, W * kWave>;
    constexpr int kSlot = 2 * Part::kBytes, kLoads = 2 * Part::kLoads, kRing = kSlots * kSlot;
    __shared__ __align__(1024) unsigned char lds[kRing > End::kBytes ? kRing : End::kBytes];
    const Product& p = a.p;
    const int l = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id()), wm = w / WN, wn = w % WN;
    const Place at = place<kKind>(a);
    End end;
    end.init(a, at);
    const int steps = p.steps;
    Part side_a, side_b;
    side_a.init(p.a, p.a_stride, end.m0, p.m, 0, w, l);
    side_b.init(p.b, p.b_stride, end.n0, p.n, 0, w, l);
    Reader<float, I, false, kStepBytes> reader_a;
    Reader<float, J, false, kStepBytes> reader_b;
    reader_a.init(wm * TM, l);
    reader_b.init(wn * TN, l);
    auto fetch_a = [&](int s) { side_a.fetch(s, lds + s % kSlots * kSlot, true, 0, l); };
    auto fetch_b = [&](int s) { side_b.fetch(s, lds + s % kSlots * kSlot + Part::kBytes, true, 0, l); };
    auto read = [&](int s, int h, Halves<I, J>& o) {
        const unsigned char* from = lds + s % kSlots * kSlot;
        reader_a.read(from, 2 * h, o.ah);
        reader_b.read(from + Part::kBytes, 2 * h, o.bh);
        reader_a.read(from, 2 * h + 1, o.al);
        reader_b.read(from + Part::kBytes, 2 * h + 1, o.bl);
    };
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
        if (s < steps) fetch_a(s);
        if (s + 1 < kSlots && s < steps) fetch_b(s);
    }
    if (steps >= kSlots)
        wait_and_meet<(kSlots - 2) * kLoads + Part::kLoads>();
    else
        wait_and_meet<0>();
    Sums<f32x16_t, I, J> acc;
    Halves<I, J> even, odd;
    read(0, 0, even);
    int s = 0;
    for (; s + kSlots < steps; ++s) {
        fetch_b(s + kSlots - 1);
        read(s, 1, odd);
        even.multiply(acc);
        wait_and_meet<(kSlots - 2) * kLoads>();
        fetch_a(s + kSlots);
        read(s + 1, 0, even);
        odd.multiply(acc);
        __builtin_amdgcn_s_waitcnt(kWaitLds);
    }
    end.load(a);
    for (; s < steps; ++s) {
        if (s + kSlots - 1 < steps) fetch_b(s + kSlots - 1);
        read(s, 1, odd);
        even.multiply(acc);
        wait_and_meet<0>();
        if (s + 1 < steps) read(s + 1, 0, even);
        odd.multiply(acc);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j) End::put(lds, 0, wm * TM + 32 * i + (l & 31), wn * TN + 32 * j, acc.value(i, j));
    __syncthreads();
    end.store(a, at, lds);
}

// ---- plan ----------------------------------------------------------------------

struct Plan {
    int m, k, blocks;
    float* u;
    double* parts;
    Pairs x[2], xt[2], a, b;
};

size_t carve(const chimera_orthogonal_shape& s, void* base, Plan* plan) {
    Carve c{static_cast<char*>(base)};
    const int m = std::min(s.rows, s.cols), k = std::max(s.rows, s.cols);
    plan->m = m;
    plan->k = k;
    plan->blocks = static_cast<int>(std::min<int64_t>(ceil_div(static_cast<int64_t>(s.rows) * ceil_div(s.cols, 8), 256), kMostBlocks));
    auto pairs = [&](int rows, int cols) {
        const int64_t stride = ceil_div(cols, 32) * 128;
        return Pairs{static_cast<unsigned char*>(c.take(static_cast<size_t>(rows) * stride)), stride};
    };
    plan->u = static_cast<float*>(c.take(static_cast<size_t>(m) * k * sizeof(float)));
    plan->parts = static_cast<double*>(c.take(plan->blocks * sizeof(double)));
    for (int i = 0; i < 2; ++i) {
        plan->x[i] = pairs(m, k);
        plan->xt[i] = pairs(k, m);
    }
    plan->a = pairs(m, m);
    plan->b = pairs(m, m);
    return c.off;
}

void operands(Schulz* a, const Pairs& p, int64_t m, const Pairs& q, int n, int sum) {
    a->p.a = p.p;
    a->p.a_stride = p.stride;
    a->p.b = q.p;
    a->p.b_stride = q.stride;
    a->p.m = m;
    a->p.n = n;
    a->p.steps = static_cast<int>(ceil_div(sum, 32));
    a->sum_by *= kUnscaleSum;
}

// Whether X' = a X + B X makes B itself: a block more for each 32 x 32 of X makes
// all of its rows, which pays while each CU has one. All five steps of 64 x 64
// take 64 us with two launches and 47 so, 128 x 768 78 and 62, 128 x 2048 93
// and 78.
bool both_at_once(int m, int k) { return m <= 128 && ceil_div(m, 32) * ceil_div(k, 32) <= kCus; }

template <Kind kKind>
void launch_both(hipStream_t st, Schulz a, const Pairs& p, int64_t m, const Pairs& q, int n) {
    operands(&a, p, m, q, n, static_cast<int>(m));
    a.linear_by *= kUnscale;
    a.square_by *= kUnscaleSum;
    a.p.tiles_m = static_cast<int>(ceil_div(m, 32));
    a.p.tiles_n = static_cast<int>(ceil_div(n, 32));
    hipLaunchKernelGGL((orthogonal_both_kernel<kKind>), dim3(static_cast<unsigned>(a.p.tiles_m * a.p.tiles_n)), dim3(256), 0, st, a);
}

template <Kind kKind>
void launch_product(hipStream_t st, Schulz a, const Pairs& p, int64_t m, const Pairs& q, int n, int sum) {
    operands(&a, p, m, q, n, sum);
    // whether tiles of 48 cover the rows' padding too
    auto ends_with_steps = [](int64_t v) { return ceil_div(v, 48) * 48 >= ceil_div(v, 32) * 32; };
    auto tiles_of = [&](int tile) {
        a.p.tiles_m = static_cast<int>(ceil_div(m, tile));
        a.p.tiles_n = static_cast<int>(ceil_div(n, tile));
        return kSymmetric<kKind> ? int64_t{a.p.tiles_m} * (a.p.tiles_m + 1) / 2 : int64_t{a.p.tiles_m} * a.p.tiles_n;
    };
    auto launch = [&](auto kernel, int tile, int threads) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles_of(tile))), dim3(static_cast<unsigned>(threads)), 0, st, a);
    };
    // As long as each CU has at most one block whose waves divide the sum (of
    // tiles of 32 for X, two), that kernel, on tiles as small as that allows; then
    // tiles of 64 that waves share, and of 128 once they fill the CUs. us of A, B
    // and X: 512 x 2048 9.8, 5.7, 11.1; 768 x 768 8.8, 10.1, 9.5; 1024 x 1024 10.3,
    // 10.2, 14.1; 1024 x 4096 23.5, 9.7, 35.6; 4096 x 4096 283, 289, 446 (920 TF of
    // products, a plain fp16 product reaches 1,300). What was compared, when the
    // lower parts' products went into the same sum as the upper ones': 512 x 2048
    // 9.5, 5.7, 10.3 and in tiles of 64 17.9, 9.4, 10.7; 768 x 768 8.7, 10.8, 9.7
    // (64: 10.8, 12.4, 11.2); 1024 x 1024 11.1, 11.3, 13.7 (64: 11.3, 12.7; shared
    // tiles of 64 11.9, 13.0, 14.8; 32 19, 21, 23); 1024 x 4096 23.8, 10.3, 35.0
    // (64: 29.0, 11.6; X in tiles of 64 38, by waves that divide the sum 48; A in
    // four parts of its sum 25 and 5 for their join); 4096 x 4096 271, 268, 429 (by
    // eight waves of 64 x 32, which read a third more from LDS, 285, 291, 439).
    // Eight waves a tile of 32 take 0.3 us less for A and B and 0.3 more for X.
    if (tiles_of(32) <= (kSymmetric<kKind> ? 256 : 400)) {
        launch(orthogonal_few_kernel<kKind, 32, kSymmetric<kKind> ? 8 : 4, kSymmetric<kKind> ? 1 : 2>, 32,
               kSymmetric<kKind> ? 512 : 256);
    } else if (tiles_of(48) <= kCus && ends_with_steps(m) && ends_with_steps(n)) {
        launch(orthogonal_few48_kernel<kKind>, 48, 512);
    } else if (tiles_of(64) <= kCus) {
        launch(orthogonal_few_kernel<kKind, 64, 4, 2, 8>, 64, 512);
    } else if (tiles_of(128) < 224) {
        launch(orthogonal_tile_kernel<kKind, 64, 2, 2, 4>, 64, 256);
    } else if (kKind == kLast) {  // whose end, with the weight, is more of its time: 36 us with 1024 x 4096, 42 by four waves
        launch(orthogonal_tile_kernel<kKind, 128, 2, 4, 4>, 128, 512);
    } else {
        launch(orthogonal_tile_kernel<kKind, 128, 2, 2, 4>, 128, 256);
    }
}

}  // namespace

size_t orthogonal_workspace(const chimera_orthogonal_shape& s) {
    Plan plan;
    return carve(s, nullptr, &plan);
}

hipError_t launch_orthogonal(hipStream_t st, const chimera_orthogonal_shape& s, const chimera_orthogonal_update& g) {
    Plan plan;
    (void)carve(s, g.workspace, &plan);
    Update u = {};
    u.gradient = g.gradient;
    u.momentum = g.momentum;
    u.new_momentum = g.new_momentum;
    u.u = plan.u;
    u.parts = plan.parts;
    u.gradient_stride = g.gradient_stride;
    u.momentum_stride = g.momentum_stride;
    u.new_momentum_stride = g.new_momentum_stride;
    u.rows = s.rows;
    u.cols = s.cols;
    u.blocks = plan.blocks;
    u.mu = g.mu;
    u.nesterov = g.nesterov != 0;
    const dim3 blocks(static_cast<unsigned>(plan.blocks));
    switch (s.type) {
        case CHIMERA_F32: hipLaunchKernelGGL((orthogonal_update_kernel<float>), blocks, dim3(256), 0, st, u); break;
        case CHIMERA_F16: hipLaunchKernelGGL((orthogonal_update_kernel<_Float16>), blocks, dim3(256), 0, st, u); break;
        default: hipLaunchKernelGGL((orthogonal_update_kernel<__bf16>), blocks, dim3(256), 0, st, u);
    }
    const bool turned = s.rows > s.cols;
    hipLaunchKernelGGL(orthogonal_scale_kernel,
                       dim3(static_cast<unsigned>(ceil_div(s.cols, 64)), static_cast<unsigned>(ceil_div(s.rows, 64))), dim3(256),
                       0, st, plan.u, plan.parts, plan.blocks, s.rows, s.cols, turned ? plan.xt[0] : plan.x[0],
                       turned ? plan.x[0] : plan.xt[0]);
    for (int i = 0; i < s.steps; ++i) {
        const Pairs &x = plan.x[i % 2], &xt = plan.xt[i % 2];
        Schulz gram = {};
        gram.along = gram.across = plan.a;
        gram.sum_by = 1.0f;
        launch_product<kGram>(st, gram, x, plan.m, x, plan.m, plan.k);
        const bool both = both_at_once(plan.m, plan.k);
        if (!both) {
            Schulz square = {};
            square.from = plan.a;
            square.from_by = s.b;
            square.sum_by = s.c;
            square.along = square.across = plan.b;
            launch_product<kSquare>(st, square, plan.a, plan.m, plan.a, plan.m, plan.m);
        }
        Schulz apply = {};
        apply.from = x;
        apply.from_by = s.a;
        apply.sum_by = 1.0f;
        apply.along = plan.x[1 - i % 2];
        apply.across = plan.xt[1 - i % 2];
        apply.linear_by = s.b;
        apply.square_by = s.c;
        if (i + 1 < s.steps) {
            if (both)
                launch_both<kApply>(st, apply, plan.a, plan.m, xt, plan.k);
            else
                launch_product<kApply>(st, apply, plan.b, plan.m, xt, plan.k, plan.m);
            continue;
        }
        Finish& f = apply.f;
        f.out = g.out;
        f.weight = g.weight;
        f.new_weight = g.new_weight;
        f.rounded = g.rounded;
        f.out_stride = g.out_stride;
        f.weight_stride = g.weight_stride;
        f.new_weight_stride = g.new_weight_stride;
        f.rounded_stride = g.rounded_stride;
        f.keep = 1.0f - g.decay;
        f.rate = g.rate;
        f.type = s.type;
        f.out_f32 = s.out_type == CHIMERA_F32;
        f.turned = turned;
        if (both)
            launch_both<kLast>(st, apply, plan.a, plan.m, xt, plan.k);
        else
            launch_product<kLast>(st, apply, plan.b, plan.m, xt, plan.k, plan.m);
    }
    return hipGetLastError();
}

}  // namespace chimera
