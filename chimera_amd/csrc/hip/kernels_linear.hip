// Dense layers that turn hidden states into token embeddings, forward and
// backward (include/chimera_operators.h):
//   Z = X W^T + b,  H = act(Z) + R,  Y = H or H / max(|H|, 1e-12)
//   dH = dY or (dY - Y <Y, dY>) / norm,  dZ = dH act'(Z),
//   dX = dZ W,  dW = dZ^T X,  db = sum of dZ's rows,  dR = dH
// The products read X, W and dZ as they lie, with rows along the summed axis
// or across it.
#include "dense_tile.hpp"

#include <algorithm>
#include <cmath>

namespace chimera {

namespace {

template <typename T, int BM, int BN, int WM, int WN, int kSlotsA, int kSlotsB, bool kAcrossA, bool kAcrossB, End kEnd>
__global__ __launch_bounds__(WM* WN* kWave) void linear_tile_kernel(Product p, Epilogue e) {
    __shared__ __align__(1024) unsigned char lds[tile_lds<BM, BN, WM, WN, kSlotsA, kSlotsB>()];
    tile_product<T, T, BM, BN, WM, WN, kSlotsA, kSlotsB, kAcrossA, kAcrossB, kEnd>(lds, p, e, static_cast<int>(blockIdx.x),
                                                                                   static_cast<int>(blockIdx.y));
}

// dW (its parts first, the longer blocks) and dX on tiles of 64 in one launch:
// neither alone fills the GPU where both take such tiles.
template <typename T>
__global__ __launch_bounds__(256) void linear_gradients_kernel(Product pw, Epilogue ew, int splits, Product px, Epilogue ex) {
    __shared__ __align__(1024) unsigned char lds[tile_lds<64, 64, 2, 2, 3, 2>()];
    const int id = static_cast<int>(blockIdx.x), tiles = pw.tiles_m * pw.tiles_n;
    if (id < tiles * splits)
        tile_product<T, T, 64, 64, 2, 2, 3, 2, true, true, kSums>(lds, pw, ew, id % tiles, id / tiles);
    else
        tile_product<T, T, 64, 64, 2, 2, 3, 2, false, true, kSums>(lds, px, ex, id - tiles * splits, 0);
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
