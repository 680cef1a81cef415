// The update of a weight made orthogonal by Newton-Schulz products
// (include/chimera_operators.h):
//   M' = mu M + G,  U = G, M' or G + mu M',  X = U / |U|
//   X <- a X + (b A + c A^2) X with A = X X^T, `steps` times
//   W' = (1 - decay) W - rate X
// X lies on its shorter side [m, k], m <= k, and its transpose beside it, so
// that the rows of all products lie along their sums.
//
// Small singular values grow up to a^steps times, and with them every error,
// so X, A and B = b A + c A^2 are held to 22 bits: a value is two fp16 parts
// (times 2^8, which keeps the lower part of values down to 2^-11 a normal
// number and leaves room up to 255), and a product is hi hi + hi lo + lo hi
// on the matrix cores, summed in 32 bits. That is as near to 64 bits as 32-bit
// products are (2e-6 to 1e-5 of the result's size at 256 to 2,048 columns; one
// fp16 part gives 2e-3), at five times their rate.
#include "dense_tile.hpp"

namespace chimera {

namespace {

constexpr float kPairScale = 256.0f;
constexpr float kUnscale = 1.0f / kPairScale, kUnscaleSum = kUnscale * kUnscale;

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
__device__ __forceinline__ void store_pairs(const Pairs& m, int64_t row, int col, const float (&v)[8]) {
    _Float16 hi[8], lo[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = v[i] * kPairScale;
        hi[i] = from_float<_Float16>(s);
        lo[i] = from_float<_Float16>(s - to_float(hi[i]));
    }
    unsigned char* to = m.p + row * m.stride + pair_chunk(col);
    *reinterpret_cast<u32x4_t*>(to) = *reinterpret_cast<const u32x4_t*>(hi);
    *reinterpret_cast<u32x4_t*>(to + 32) = *reinterpret_cast<const u32x4_t*>(lo);
}
__device__ __forceinline__ void load_pairs(const Pairs& m, int64_t row, int col, float (&v)[8]) {
    const unsigned char* from = m.p + row * m.stride + pair_chunk(col);
    const f16x8_t hi = *reinterpret_cast<const f16x8_t*>(from), lo = *reinterpret_cast<const f16x8_t*>(from + 32);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (to_float(hi[i]) + to_float(lo[i])) * kUnscale;
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

// A tile of 64 x 64 values as pairs: rows [row0, row0 + 64) of `along` from
// column col0 on, and the transposed tile of `across`. Columns up to the end of
// a step are written, from values that are zeros there.
constexpr int kTilePitch = 65;
template <int kThreads>
__device__ __forceinline__ void put_tile(const float* tile, int rows, int cols, const Pairs& along, int64_t row0,
                                         const Pairs& across, int64_t col0) {
    for (int i = static_cast<int>(threadIdx.x); i < 64 * 8; i += kThreads) {
        const int r = i / 8, c = i % 8 * 8;
        float v[8];
        if (along.p && r < rows && c < (cols + 31) / 32 * 32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = tile[r * kTilePitch + c + j];
            store_pairs(along, row0 + r, static_cast<int>(col0) + c, v);
        }
        if (across.p && r < cols && c < (rows + 31) / 32 * 32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = tile[(c + j) * kTilePitch + r];
            store_pairs(across, col0 + r, static_cast<int>(row0) + c, v);
        }
    }
}

// X = U / |U| as pairs, along and across; a U of zeros stays zeros.
__global__ __launch_bounds__(256) void orthogonal_scale_kernel(const float* u, const double* parts, int count, int rows,
                                                               int cols, Pairs along, Pairs across) {
    __shared__ float tile[64 * kTilePitch];
    __shared__ double sums[4];
    double sum = 0.0;
    for (int i = static_cast<int>(threadIdx.x); i < count; i += 256) sum += parts[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    if (lane_id() == 0) sums[wave_id()] = sum;
    __syncthreads();
    sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const double by = sum == 0.0 ? 0.0 : 1.0 / sqrt(sum);
    const int row0 = static_cast<int>(blockIdx.y) * 64, col0 = static_cast<int>(blockIdx.x) * 64;
    for (int i = static_cast<int>(threadIdx.x); i < 64 * 64; i += 256) {
        const int r = i / 64, c = i % 64;
        const bool in = row0 + r < rows && col0 + c < cols;
        tile[r * kTilePitch + c] = in ? static_cast<float>(u[static_cast<int64_t>(row0 + r) * cols + col0 + c] * by) : 0.0f;
    }
    __syncthreads();
    put_tile<256>(tile, min(64, rows - row0), min(64, cols - col0), along, row0, across, col0);
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
    Finish f;
};

template <typename T>
__device__ __forceinline__ void put_as(void* p, int64_t at, float v) {
    static_cast<T*>(p)[at] = from_float<T>(v);
}
__device__ __forceinline__ void put(void* p, int64_t at, float v, int type) {
    if (type == CHIMERA_F32)
        put_as<float>(p, at, v);
    else if (type == CHIMERA_F16)
        put_as<_Float16>(p, at, v);
    else
        put_as<__bf16>(p, at, v);
}

// C = P Q^T of pairs on a tile of 64 x 64, four waves, the operands straight
// to a ring of LDS slots. C becomes from_by F + sum_by C, stored along and
// across; of the symmetric results only tiles on and below the diagonal are
// computed.
constexpr int kSlots = 4;
template <Kind kKind>
__global__ __launch_bounds__(256) void orthogonal_tile_kernel(Schulz a) {
    using Part = Side<float, 64, 4, false>;
    constexpr int kRing = kSlots * 2 * Part::kBytes;
    static_assert(kRing >= 64 * kTilePitch * 4, "the tile goes through the ring's memory");
    __shared__ __align__(1024) unsigned char lds[kRing];
    const Product& p = a.p;
    const int l = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
    int tm, tn;
    if constexpr (kKind == kGram || kKind == kSquare) {
        const int id = static_cast<int>(blockIdx.x);
        tm = static_cast<int>((sqrtf(8.0f * static_cast<float>(id) + 1.0f) - 1.0f) * 0.5f);
        while ((tm + 1) * (tm + 2) / 2 <= id) ++tm;
        while (tm * (tm + 1) / 2 > id) --tm;
        tn = id - tm * (tm + 1) / 2;
    } else {
        tm = static_cast<int>(blockIdx.x) % p.tiles_m;
        tn = static_cast<int>(blockIdx.x) / p.tiles_m;
    }
    const int64_t m0 = tm * 64ll, n0 = tn * 64ll;
    Part side_a, side_b;
    side_a.init(p.a, p.a_stride, m0, p.m, 0, w, l);
    side_b.init(p.b, p.b_stride, n0, p.n, 0, w, l);
    Reader<float, 1, false, kStepBytes> reader_a, reader_b;
    reader_a.init(w / 2 * 32, l);
    reader_b.init(w % 2 * 32, l);
    auto fetch = [&](int s) {
        unsigned char* to = lds + s % kSlots * 2 * Part::kBytes;
        side_a.fetch(s, to, true, 0, l);
        side_b.fetch(s, to + Part::kBytes, true, 0, l);
    };
    f32x16_t acc = {};
    auto step = [&](int s) {
        const unsigned char* from = lds + s % kSlots * 2 * Part::kBytes;
        u32x4_t x[4][1], y[4][1];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            reader_a.read(from, q, x[q]);
            reader_b.read(from + Part::kBytes, q, y[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
            acc = mma32<_Float16>(y[q + 1][0], x[q][0], acc);
            acc = mma32<_Float16>(y[q][0], x[q + 1][0], acc);
            acc = mma32<_Float16>(y[q][0], x[q][0], acc);
        }
    };
    const int steps = p.steps;
    for (int s = 0; s < kSlots - 1 && s < steps; ++s) fetch(s);
    int s = 0;
    for (; s + kSlots - 1 < steps; ++s) {
        wait_and_meet<(kSlots - 2) * 2 * Part::kLoads>();
        fetch(s + kSlots - 1);
        step(s);
    }
    for (; s < steps; ++s) {
        wait_and_meet<0>();
        step(s);
    }
    __syncthreads();
    float* tile = reinterpret_cast<float*>(lds);
    const int rows = static_cast<int>(min(p.m - m0, int64_t{64})), cols = static_cast<int>(min(p.n - n0, int64_t{64}));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int i = w / 2 * 32 + (l & 31), j = w % 2 * 32 + 8 * (r >> 2) + 4 * (l >> 5) + (r & 3);
        tile[i * kTilePitch + j] = i < rows && j < cols ? acc[r] * a.sum_by : 0.0f;
    }
    __syncthreads();
    if constexpr (kKind != kGram) {
        for (int i = static_cast<int>(threadIdx.x); i < 64 * 8; i += 256) {
            const int r = i / 8, c = i % 8 * 8;
            if (r >= rows || c >= cols) continue;
            float v[8];
            load_pairs(a.from, m0 + r, static_cast<int>(n0) + c, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) tile[r * kTilePitch + c + j] = fmaf(a.from_by, v[j], tile[r * kTilePitch + c + j]);
        }
        __syncthreads();
    }
    if constexpr (kKind != kLast) {
        Pairs across = a.across;
        if ((kKind == kGram || kKind == kSquare) && tm == tn) across.p = nullptr;
        put_tile<256>(tile, rows, cols, a.along, m0, across, n0);
    } else {
        const Finish& f = a.f;
        for (int i = static_cast<int>(threadIdx.x); i < 64 * 64; i += 256) {
            // neighbouring threads write neighbouring columns of the results
            const int r = f.turned ? i % 64 : i / 64, c = f.turned ? i / 64 : i % 64;
            if (r >= rows || c >= cols) continue;
            const float v = tile[r * kTilePitch + c];
            const int64_t row = f.turned ? n0 + c : m0 + r, col = f.turned ? m0 + r : n0 + c;
            if (f.out) put(f.out, row * f.out_stride + col, v, f.out_f32 ? CHIMERA_F32 : f.type);
            if (f.weight) {
                const float next = fmaf(f.keep, f.weight[row * f.weight_stride + col], -f.rate * v);
                f.new_weight[row * f.new_weight_stride + col] = next;
                if (f.rounded) put(f.rounded, row * f.rounded_stride + col, next, f.type);
            }
        }
    }
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
    plan->blocks = static_cast<int>(std::min<int64_t>(ceil_div(static_cast<int64_t>(s.rows) * ceil_div(s.cols, 8), 256), 1024));
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

template <Kind kKind>
void launch_product(hipStream_t st, Schulz a, const Pairs& p, int64_t m, const Pairs& q, int n, int sum) {
    a.p.a = p.p;
    a.p.a_stride = p.stride;
    a.p.b = q.p;
    a.p.b_stride = q.stride;
    a.p.m = m;
    a.p.n = n;
    a.p.steps = static_cast<int>(ceil_div(sum, 32));
    a.p.tiles_m = static_cast<int>(ceil_div(m, 64));
    a.p.tiles_n = static_cast<int>(ceil_div(n, 64));
    a.sum_by *= kUnscaleSum;
    const int tiles = kKind == kGram || kKind == kSquare ? a.p.tiles_m * (a.p.tiles_m + 1) / 2 : a.p.tiles_m * a.p.tiles_n;
    hipLaunchKernelGGL((orthogonal_tile_kernel<kKind>), dim3(static_cast<unsigned>(tiles)), dim3(256), 0, st, a);
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
        Schulz square = {};
        square.from = plan.a;
        square.from_by = s.b;
        square.sum_by = s.c;
        square.along = square.across = plan.b;
        launch_product<kSquare>(st, square, plan.a, plan.m, plan.a, plan.m, plan.m);
        Schulz apply = {};
        apply.from = x;
        apply.from_by = s.a;
        apply.sum_by = 1.0f;
        apply.along = plan.x[1 - i % 2];
        apply.across = plan.xt[1 - i % 2];
        if (i + 1 < s.steps) {
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
        launch_product<kLast>(st, apply, plan.b, plan.m, xt, plan.k, plan.m);
    }
    return hipGetLastError();
}

}  // namespace chimera
