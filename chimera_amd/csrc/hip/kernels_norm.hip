// Layer norm and its gradients (include/chimera_operators.h):
//   z = (x - mean) rstd,  rstd = (mean of (x - mean)^2 + eps)^-1/2,  y = z w + b
//   g = dy w,  dx = rstd (g - mean of g - z mean of g z),
//   dw = the sum over rows of dy z,  db = that of dy
#include "operators.hpp"

#include <algorithm>
#include <type_traits>

namespace chimera {

namespace {

int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

// Rows whose squares pass the 32-bit range are taken times kSmall, and so are
// those in the backward pass whose rstd is below kLowRstd.
constexpr float kSmall = 0x1p-80f, kLarge = 0x1p80f, kLowRstd = 0x1p-60f;
// What the rounding of a row's mean left out, over the row's deviation, from
// which on it is taken away, and how often at the most: each turn leaves 2^-17
// of it.
constexpr float kSmallRest = 0x1p-4f;
constexpr int kMostTurns = 16;

struct NormArgs {
    const void* x;
    const void* weight;
    const void* bias;
    const void* dy;
    void* y;  // or dx
    float* mean;
    float* rstd;
    float* parts;  // [blocks][2][cols]: sums of dy z and of dy
    int64_t x_stride, y_stride, dy_stride;
    int64_t rows;
    int cols;
    float eps;
    bool wants_dx;
};

// ---- sums over the threads of a row --------------------------------------------

// A row is kLanes neighbouring lanes, or the whole block of kLanes threads.
template <int kLanes, int kCount>
__device__ __forceinline__ void row_sums(float (&v)[kCount], float* lds) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
        if constexpr (kLanes >= kWave) {
            v[i] = wave_sum(v[i]);
        } else {
            static_assert(kLanes == 16, "");
            v[i] += lane_move<kSwap1>(v[i]);
            v[i] += lane_move<kSwap2>(v[i]);
            v[i] += lane_move<kMirror8>(v[i]);
            v[i] += lane_move<kRotate8>(v[i]);
        }
    }
    if constexpr (kLanes > kWave) {
        constexpr int kWaves = kLanes / kWave;
        __syncthreads();  // the sums before these have been read
        if (lane_id() == 0) {
#pragma unroll
            for (int i = 0; i < kCount; ++i) lds[wave_id() * kCount + i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) s += lds[w * kCount + i];
            v[i] = s;
        }
    }
}

// Threads of a block that has rows of kLanes threads.
constexpr int block_threads(int lanes) { return lanes > 256 ? lanes : 256; }
constexpr int kBackThreads = 256;

// ---- a thread's columns --------------------------------------------------------

// Eights of neighbours, as they lie in memory until they are taken: a row's are
// loaded while the row before it is worked on.
template <typename T>
struct Eight {
    u32x4_t v[sizeof(T) / 2];

    __device__ __forceinline__ void load(const T* p) {
        typedef T vec_t __attribute__((ext_vector_type(16 / sizeof(T))));
        typedef vec_t any_t __attribute__((aligned(sizeof(T))));
#pragma unroll
        for (int h = 0; h < static_cast<int>(sizeof(T)) / 2; ++h)
            v[h] = __builtin_bit_cast(u32x4_t, static_cast<vec_t>(reinterpret_cast<const any_t*>(p)[h]));
    }
    __device__ __forceinline__ void load(const T* p, int count) {
        T x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i < count ? p[i] : T(0.0f);
        __builtin_memcpy(v, x, sizeof(v));
    }
    __device__ __forceinline__ void take(float (&x)[8]) const {
        typedef T eight_t __attribute__((ext_vector_type(8)));
        eight_t u;
        __builtin_memcpy(&u, v, sizeof(v));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float(static_cast<T>(u[i]));
    }
};

// How rows fit their threads. kWhole: all threads have eights of their own.
// kRagged: an eight that passes the row's end lies at its end instead, and those
// of threads past it too; columns that two threads have get the same values from
// both, and count in the sums of one. So all loads are whole, and none is
// conditional. kNarrow: rows below eight columns, which the first thread takes.
enum Fit { kWhole, kRagged, kNarrow };

template <Fit kFit, int kLanes, int kChunks>
struct Columns {
    int t, cols;

    __device__ __forceinline__ Columns(int cols) : t(static_cast<int>(threadIdx.x) % kLanes), cols(cols) {}
    __device__ __forceinline__ int base(int j) const { return (j * kLanes + t) * 8; }
    __device__ __forceinline__ int first(int j) const {
        return kFit == kWhole ? base(j) : kFit == kNarrow ? 0 : min(base(j), cols - 8);
    }
    __device__ __forceinline__ bool there(int j) const { return kFit == kWhole || base(j) < cols; }
    // whether column first(j) + i counts here
    __device__ __forceinline__ bool counts(int j, int i) const {
        return kFit == kWhole || (kFit == kNarrow ? t == 0 && i < cols : i >= base(j) - first(j));
    }
    template <typename T>
    __device__ __forceinline__ void load(const T* row, Eight<T> (&v)[kChunks]) const {
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            if constexpr (kFit == kNarrow)
                v[j].load(row, cols);
            else
                v[j].load(row + first(j));
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(T* row, int j, const float (&v)[8]) const {
        if (there(j)) store8(row + first(j), kFit == kNarrow ? cols : 8, v);
    }
    // columns of a vector of the row's length, or `other`
    template <typename T>
    __device__ __forceinline__ void load(const T* p, float other, int j, float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = other;
        if (!p) return;
        Eight<T> u;
        if constexpr (kFit == kNarrow)
            u.load(p, cols);
        else
            u.load(p + first(j));
        u.take(v);
    }
};

// ---- forward -------------------------------------------------------------------

// A row's values stay in registers, 8 kChunks a thread, and are read once; the
// next row's are under way meanwhile, and the weights stay for all rows. Bound
// by memory: 65,536 x 1024 bf16 53 us, 5.1 TB/s (a copy 5.4); 65,536 x 768 41 (a
// wave for each row, without what it keeps: 50, and 60 with loads that wait for
// the row before them). A row of 64 lanes needs no LDS; longer ones meet twice.
// The variance is taken about a mean that is corrected by what is left of the
// row's sum after it, so that rows far from zero keep their digits. Where that
// rest is not small beside the row's deviation (rows of one value, or of a few
// neighbouring ones, far from zero) it is taken away and the sums are made
// again, in turns, from the caches. (In registers all rows would need more of
// them: 65,536 x 1024 53.4 us, not 51.8, and 500 x 65,536 of 32 bits 87, not 81;
// without the turns these take 51.8 and 70.)
template <typename T, typename Out, int kLanes, int kChunks, Fit kFit>
__global__ __launch_bounds__(block_threads(kLanes)) void norm_forward_kernel(NormArgs a) {
    constexpr int kRows = block_threads(kLanes) / kLanes;
    __shared__ float lds[kLanes > kWave ? kLanes / kWave * 2 : 1];
    const Columns<kFit, kLanes, kChunks> at(a.cols);
    const float inv = 1.0f / static_cast<float>(a.cols);
    int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + static_cast<int>(threadIdx.x) / kLanes;
    if (r >= a.rows) return;
    const T* const x0 = static_cast<const T*>(a.x);
    const T *const weight = static_cast<const T*>(a.weight), *const bias = static_cast<const T*>(a.bias);
    constexpr bool kAhead = kLanes <= 256;  // else a row takes the registers
    Eight<T> next[kChunks];
    float w[kAhead ? kChunks : 1][8], b[kAhead ? kChunks : 1][8];
    if constexpr (kAhead) {
        at.load(x0 + r * a.x_stride, next);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            at.load(weight, 1.0f, j, w[j]);
            at.load(bias, 0.0f, j, b[j]);
        }
    }
    for (; r < a.rows; r += static_cast<int64_t>(gridDim.x) * kRows) {
        float x[kChunks][8];
        if constexpr (!kAhead) at.load(x0 + r * a.x_stride, next);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) next[j].take(x[j]);
        const int64_t after = r + static_cast<int64_t>(gridDim.x) * kRows;
        if constexpr (kAhead) at.load(x0 + (after < a.rows ? after : r) * a.x_stride, next);
        float mean, rest, var;
        auto spread = [&](float (&s)[2]) {  // from the sums of x - mean and of its squares
            row_sums<kLanes>(s, lds);
            rest = s[0] * inv;
            // what rounding leaves of one value is no deviation
            var = fmaxf(fmaf(-rest, rest, s[1] * inv), rest * rest * 0x1p-18f);
            return s[1] - s[1] == 0.0f;  // neither infinite nor NaN
        };
        auto moments = [&] {  // x becomes x - mean
            float sum[1] = {0.0f};
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[0] += at.counts(j, i) ? x[j][i] : 0.0f;
            row_sums<kLanes>(sum, lds);
            mean = sum[0] * inv;
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[j][i] -= mean;
                    const float d = at.counts(j, i) ? x[j][i] : 0.0f;
                    s[0] += d;
                    s[1] = fmaf(d, d, s[1]);
                }
            return spread(s);
        };
        float scale = 1.0f;
        if (!moments()) {
            scale = kSmall;
            Eight<T> again[kChunks];
            at.load(x0 + r * a.x_stride, again);
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
                again[j].take(x[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[j][i] *= kSmall;
            }
            (void)moments();
        }
        const float eps = a.eps * scale * scale;
        float more = 0.0f;  // of the mean
        auto is_large = [&] { return rest * rest > kSmallRest * kSmallRest * (var + eps); };
        if (is_large()) {
            auto less = [&](int j, float (&v)[8]) {
                at.load(x0 + r * a.x_stride, 0.0f, j, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], scale, -mean) - more;
            };
            for (int turn = 0; turn < kMostTurns && is_large(); ++turn) {
                more += rest;
                float s[2] = {0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < kChunks; ++j) {
                    float v[8];
                    less(j, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float d = at.counts(j, i) ? v[i] : 0.0f;
                        s[0] += d;
                        s[1] = fmaf(d, d, s[1]);
                    }
                }
                (void)spread(s);
            }
#pragma unroll
            for (int j = 0; j < kChunks; ++j) less(j, x[j]);
        }
        const float square = var + eps;  // 0 for scaled rows of one value
        const float rstd = square == 0.0f ? 0.0f : 1.0f / sqrtf(square), by = -rest * rstd;
        if (at.t == 0) {
            if (a.mean) a.mean[r] = (mean + (more + rest)) * (scale == 1.0f ? 1.0f : kLarge);
            if (a.rstd) a.rstd[r] = square == 0.0f ? 1.0f / sqrtf(a.eps) : rstd * scale;
        }
        Out* to = static_cast<Out*>(a.y) + r * a.y_stride;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            if constexpr (!kAhead) {
                at.load(weight, 1.0f, j, w[0]);
                at.load(bias, 0.0f, j, b[0]);
            }
            constexpr int kOne = kAhead ? kChunks : 1;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf(fmaf(x[j][i], rstd, by), w[j % kOne][i], b[j % kOne][i]);
            at.store(to, j, v);
        }
    }
}

// ---- backward ------------------------------------------------------------------

// x and dy are read once and stay in registers, the next row's under way
// meanwhile: 16,384 x 1024 bf16 18.9 us, 5.3 TB/s (35 when each row's loads wait
// for the row before). So do the thread's columns of the sums over rows; these
// are joined over the block's rows in order and written for the join, 4 us. What
// the rounding of the mean left out is the sum of x - mean, and is taken away
// again, in turns where it is not small (see the forward pass; here from the
// registers, as loads in the branch make all rows wait for the next one's:
// 16,384 x 1024 29.4 us with the join, not 23.7; without the turns 23.4).
template <typename T, typename Out, int kLanes, int kChunks, Fit kFit>
__global__ __launch_bounds__(kBackThreads) void norm_backward_kernel(NormArgs a) {
    constexpr int kRows = kBackThreads / kLanes;
    __shared__ float lds[kLanes > kWave ? kLanes / kWave * 3 * kRows : 1];
    __shared__ float sums[kRows > 1 ? kBackThreads * 8 : 1];
    const Columns<kFit, kLanes, kChunks> at(a.cols);
    const int t = at.t, in_block = static_cast<int>(threadIdx.x) / kLanes;
    const float inv = 1.0f / static_cast<float>(a.cols);
    float w[kChunks][8], dw[kChunks][8] = {}, db[kChunks][8] = {};
#pragma unroll
    for (int j = 0; j < kChunks; ++j) at.load(static_cast<const T*>(a.weight), 1.0f, j, w[j]);
    const T* const x0 = static_cast<const T*>(a.x);
    const Out* const dy0 = static_cast<const Out*>(a.dy);
    Eight<T> next_x[kChunks];
    Eight<Out> next_dy[kChunks];
    float next_rstd = 0.0f, next_mean = 0.0f;
    auto load = [&](int64_t r) {
        at.load(x0 + r * a.x_stride, next_x);
        at.load(dy0 + r * a.dy_stride, next_dy);
        next_rstd = a.rstd[r];
        next_mean = a.mean[r];
    };
    int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + in_block;
    if (r < a.rows) load(r);
    for (; r < a.rows; r += static_cast<int64_t>(gridDim.x) * kRows) {
        float x[kChunks][8], dy[kChunks][8];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            next_x[j].take(x[j]);
            next_dy[j].take(dy[j]);
        }
        const float rstd = next_rstd;
        const bool low = rstd < kLowRstd;
        const float scale = low ? kSmall : 1.0f, mean = next_mean * scale, by = low ? rstd * kLarge : rstd;
        const int64_t after = r + static_cast<int64_t>(gridDim.x) * kRows;
        load(after < a.rows ? after : r);
        float s[3], rest;
        auto sum_up = [&](float more) {  // of x - mean - more
            s[0] = s[1] = s[2] = 0.0f;
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = at.counts(j, i) ? x[j][i] - more : 0.0f;
                    const float g = at.counts(j, i) ? dy[j][i] * w[j][i] : 0.0f;
                    s[0] += d;
                    s[1] += g;
                    s[2] = fmaf(g, d, s[2]);
                }
            row_sums<kLanes>(s, lds);
            rest = s[0] * inv;
        };
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[j][i] = fmaf(x[j][i], scale, -mean);
        sum_up(0.0f);
        float more = 0.0f;
        for (int turn = 0; turn < kMostTurns && fabsf(rest) * by > kSmallRest; ++turn) {
            more += rest;
            sum_up(more);
        }
        const float mean_g = s[1] * inv, mean_gz = by * fmaf(-rest, s[1], s[2]) * inv, off = -rest * by;
        T* to = static_cast<T*>(a.y) + r * a.y_stride;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = fmaf(x[j][i] - more, by, off);
                v[i] = rstd * fmaf(-z, mean_gz, fmaf(dy[j][i], w[j][i], -mean_g));
                dw[j][i] = fmaf(dy[j][i], z, dw[j][i]);
                db[j][i] += dy[j][i];
            }
            if (a.wants_dx) at.store(to, j, v);
        }
    }
    if (!a.parts) return;
    // rows of the block in order, then the block's sums
    float* part = a.parts + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = which ? db[j][i] : dw[j][i];
            if constexpr (kRows > 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) sums[(in_block * 8 + i) * kLanes + t] = v[i];
                __syncthreads();
                if (in_block == 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float sum = 0.0f;
#pragma unroll
                        for (int o = 0; o < kRows; ++o) sum += sums[(o * 8 + i) * kLanes + t];
                        v[i] = sum;
                    }
                }
            }
            if (in_block == 0) at.store(part + which * a.cols, j, v);
        }
}

// Rows too long for registers: two passes over a row, the second from the
// caches. `rests` [rows][2] gets what the saved mean left out, in two parts: what
// was taken away in turns, and what is left.
template <typename T, typename Out>
__global__ __launch_bounds__(1024) void norm_wide_kernel(NormArgs a, float* rests) {
    __shared__ float lds[16 * 3];
    const float inv = 1.0f / static_cast<float>(a.cols);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        float more = 0.0f;
        const T* from = static_cast<const T*>(a.x) + r * a.x_stride;
        const Out* grad = static_cast<const Out*>(a.dy) + r * a.dy_stride;
        const float rstd = a.rstd[r];
        const bool low = rstd < kLowRstd;
        const float scale = low ? kSmall : 1.0f, mean = a.mean[r] * scale, by = low ? rstd * kLarge : rstd;
        auto each = [&](auto&& visit) {
            for (int c = static_cast<int>(threadIdx.x) * 8; c < a.cols; c += 8192) {
                const int count = a.cols - c;
                float x[8], dy[8], w[8];
                load8(from + c, count, x);
                load8(grad + c, count, dy);
                if (a.weight) load8(static_cast<const T*>(a.weight) + c, count, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[i] = i < count ? fmaf(x[i], scale, -mean) - more : 0.0f;
                    dy[i] = i < count ? a.weight ? dy[i] * w[i] : dy[i] : 0.0f;
                }
                visit(c, count, x, dy);
            }
        };
        float s[3], rest;
        auto sum_up = [&] {
            s[0] = s[1] = s[2] = 0.0f;
            each([&](int, int, float(&d)[8], float(&g)[8]) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    s[0] += d[i];
                    s[1] += g[i];
                    s[2] = fmaf(g[i], d[i], s[2]);
                }
            });
            row_sums<1024>(s, lds);
            rest = s[0] * inv;
        };
        sum_up();
        for (int turn = 0; turn < kMostTurns && fabsf(rest) * by > kSmallRest; ++turn) {
            more += rest;
            sum_up();
        }
        const float mean_g = s[1] * inv, mean_gz = by * fmaf(-rest, s[1], s[2]) * inv;
        if (rests && threadIdx.x == 0) {
            rests[2 * r] = more;
            rests[2 * r + 1] = rest;
        }
        if (!a.wants_dx) continue;
        T* to = static_cast<T*>(a.y) + r * a.y_stride;
        each([&](int c, int count, float(&d)[8], float(&g)[8]) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = rstd * fmaf(-(d[i] - rest) * by, mean_gz, g[i] - mean_g);
            store8(to + c, count, v);
        });
    }
}
// Their sums over rows: 2,048 columns a block, eight a thread, the rows of
// part blockIdx.y.
template <typename T, typename Out>
__global__ __launch_bounds__(256) void norm_wide_sums_kernel(NormArgs a, const float* rests, int64_t part_rows) {
    const int c = (static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x)) * 8;
    const int count = a.cols - c;
    if (count <= 0) return;
    float dw[8] = {}, db[8] = {};
    const int64_t begin = blockIdx.y * part_rows, end = min(begin + part_rows, a.rows);
    for (int64_t r = begin; r < end; ++r) {
        const float rstd = a.rstd[r];
        const bool low = rstd < kLowRstd;
        const float scale = low ? kSmall : 1.0f, mean = a.mean[r] * scale, by = low ? rstd * kLarge : rstd;
        const float more = rests[2 * r], rest = rests[2 * r + 1];
        float x[8], dy[8];
        load8(static_cast<const T*>(a.x) + r * a.x_stride + c, count, x);
        load8(static_cast<const Out*>(a.dy) + r * a.dy_stride + c, count, dy);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            dw[i] = fmaf(dy[i], (fmaf(x[i], scale, -mean) - more - rest) * by, dw[i]);
            db[i] += dy[i];
        }
    }
    float* part = a.parts + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
    store8(part + c, count, dw);
    store8(part + a.cols + c, count, db);
}

// dw and db from the blocks' sums [parts][2][cols], in a fixed order: a block
// takes 32 of the 2 cols columns, its 16 half waves a share of the parts each.
template <typename T>
__global__ __launch_bounds__(512) void norm_join_kernel(const float* parts, int count, int cols, T* dweight, T* dbias) {
    __shared__ float lds[16][33];
    const int lane = static_cast<int>(threadIdx.x) % 32, share = static_cast<int>(threadIdx.x) / 32;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    const int each = (count + 15) / 16, end = min(count, (share + 1) * each);
    float s = 0.0f;
    if (i < 2 * cols) {
#pragma unroll 8
        for (int p = share * each; p < end; ++p) s += parts[static_cast<int64_t>(p) * 2 * cols + i];
    }
    lds[share][lane] = s;
    __syncthreads();
    if (share != 0 || i >= 2 * cols) return;
    s = 0.0f;
#pragma unroll
    for (int o = 0; o < 16; ++o) s += lds[o][lane];
    T* to = i < cols ? dweight : dbias;
    if (to) to[i < cols ? i : i - cols] = from_float<T>(s);
}

template <typename T>
__global__ __launch_bounds__(256) void norm_zero_kernel(T* dweight, T* dbias, int cols) {
    const int i = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
    if (i >= cols) return;
    if (dweight) dweight[i] = from_float<T>(0.0f);
    if (dbias) dbias[i] = from_float<T>(0.0f);
}

// ---- plans ---------------------------------------------------------------------

constexpr int kMostRegisters = 8192;  // columns of a backward pass in registers
constexpr int kMostParts = 512;       // 1,024 take 1 us longer at 16,384 x 1,024, and their join too; 256 1 us longer
constexpr int kMostThreads = 2048 * 256;  // 8 waves a SIMD

// Parts of the sums over rows, as many as blocks: grows with the rows.
int64_t parts_of(int64_t rows, int cols) {
    if (cols > kMostRegisters) return std::min<int64_t>(rows, 64);
    const int lanes = cols <= 128 ? 16 : cols <= 1024 ? 64 : 256;
    return std::min<int64_t>(ceil_div(rows, 256 / lanes), kMostParts);
}

template <int kValue>
using Int = std::integral_constant<int, kValue>;

template <int kLanes, int kChunks, typename Call>
void by_fit(int cols, Call&& call) {
    if (kLanes >= kWave && cols == kLanes * kChunks * 8) return call(std::integral_constant<Fit, kLanes >= kWave ? kWhole : kRagged>{});
    if (kLanes < kWave && cols < 8) return call(std::integral_constant<Fit, kLanes < kWave ? kNarrow : kRagged>{});
    return call(std::integral_constant<Fit, kRagged>{});
}

template <typename T, typename Out>
hipError_t forward(hipStream_t st, const NormArgs& a) {
    auto launch = [&](auto lanes, auto chunks) {
        constexpr int kLanes = decltype(lanes)::value, kChunks = decltype(chunks)::value, kThreads = block_threads(kLanes);
        const int64_t blocks = std::min<int64_t>(ceil_div(a.rows, kThreads / kLanes), kMostThreads / kThreads);
        by_fit<kLanes, kChunks>(a.cols, [&](auto fit) {
            hipLaunchKernelGGL((norm_forward_kernel<T, Out, kLanes, kChunks, decltype(fit)::value>),
                               dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, a);
        });
        return hipGetLastError();
    };
    if (a.cols <= 128) return launch(Int<16>{}, Int<1>{});
    if (a.cols <= 512) return launch(Int<64>{}, Int<1>{});
    if (a.cols <= 1024) return launch(Int<64>{}, Int<2>{});
    if (a.cols <= 2048) return launch(Int<256>{}, Int<1>{});
    if (a.cols <= 4096) return launch(Int<256>{}, Int<2>{});
    if (a.cols <= 8192) return launch(Int<256>{}, Int<4>{});
    if (a.cols <= 16384) return launch(Int<1024>{}, Int<2>{});
    if (a.cols <= 32768) return launch(Int<1024>{}, Int<4>{});
    return launch(Int<1024>{}, Int<8>{});
}

template <typename T, typename Out>
hipError_t backward(hipStream_t st, NormArgs a, const chimera_norm_backward& b) {
    T *dweight = static_cast<T*>(b.dweight), *dbias = static_cast<T*>(b.dbias);
    const bool sums = dweight || dbias;
    if (a.rows == 0) {
        if (sums)
            hipLaunchKernelGGL((norm_zero_kernel<T>), dim3(static_cast<unsigned>(ceil_div(a.cols, 256))), dim3(256), 0, st,
                               dweight, dbias, a.cols);
        return hipGetLastError();
    }
    if (!sums && !a.wants_dx) return hipSuccess;
    const int64_t parts = parts_of(a.rows, a.cols);
    a.parts = sums ? static_cast<float*>(b.workspace) : nullptr;
    auto launch = [&](auto lanes, auto chunks) {
        constexpr int kLanes = decltype(lanes)::value, kChunks = decltype(chunks)::value, kRows = kBackThreads / kLanes;
        const int64_t blocks = sums ? parts : std::min<int64_t>(ceil_div(a.rows, kRows), kMostThreads / kBackThreads);
        by_fit<kLanes, kChunks>(a.cols, [&](auto fit) {
            hipLaunchKernelGGL((norm_backward_kernel<T, Out, kLanes, kChunks, decltype(fit)::value>),
                               dim3(static_cast<unsigned>(blocks)), dim3(kBackThreads), 0, st, a);
        });
    };
    if (a.cols <= 128)
        launch(Int<16>{}, Int<1>{});
    else if (a.cols <= 512)
        launch(Int<64>{}, Int<1>{});
    else if (a.cols <= 1024)
        launch(Int<64>{}, Int<2>{});
    else if (a.cols <= 2048)
        launch(Int<256>{}, Int<1>{});
    else if (a.cols <= 4096)
        launch(Int<256>{}, Int<2>{});
    else if (a.cols <= kMostRegisters)
        launch(Int<256>{}, Int<4>{});
    else {
        float* rests = sums ? a.parts + parts * 2 * a.cols : nullptr;
        hipLaunchKernelGGL((norm_wide_kernel<T, Out>), dim3(static_cast<unsigned>(std::min<int64_t>(a.rows, 1 << 20))),
                           dim3(1024), 0, st, a, rests);
        if (sums)
            hipLaunchKernelGGL((norm_wide_sums_kernel<T, Out>),
                               dim3(static_cast<unsigned>(ceil_div(a.cols, 2048)), static_cast<unsigned>(parts)), dim3(256), 0,
                               st, a, rests, ceil_div(a.rows, parts));
    }
    if (sums)
        hipLaunchKernelGGL((norm_join_kernel<T>), dim3(static_cast<unsigned>(ceil_div(2 * a.cols, 32))), dim3(512), 0, st,
                           a.parts, static_cast<int>(parts), a.cols, dweight, dbias);
    return hipGetLastError();
}

template <typename Call>
auto by_types(int type, int out_type, Call&& call) {
    if (type == CHIMERA_F32) return call(float{}, float{});
    if (type == CHIMERA_F16) return out_type == CHIMERA_F32 ? call(_Float16{}, float{}) : call(_Float16{}, _Float16{});
    return out_type == CHIMERA_F32 ? call(__bf16{}, float{}) : call(__bf16{}, __bf16{});
}

}  // namespace

size_t norm_workspace(const chimera_norm_shape& s) {
    const int64_t rests = s.features > kMostRegisters ? 2 * s.rows : 0;
    return static_cast<size_t>(parts_of(s.rows, s.features) * 2 * s.features + rests) * sizeof(float);
}

hipError_t launch_norm_forward(hipStream_t st, const chimera_norm_shape& s, const chimera_norm_forward& f) {
    NormArgs a = {};
    a.x = f.x;
    a.weight = f.weight;
    a.bias = f.bias;
    a.y = f.y;
    a.mean = f.mean;
    a.rstd = f.rstd;
    a.x_stride = f.x_stride;
    a.y_stride = f.y_stride;
    a.rows = s.rows;
    a.cols = s.features;
    a.eps = s.eps;
    return by_types(s.type, s.out_type, [&](auto t, auto o) { return forward<decltype(t), decltype(o)>(st, a); });
}

hipError_t launch_norm_backward(hipStream_t st, const chimera_norm_shape& s, const chimera_norm_backward& b) {
    NormArgs a = {};
    a.x = b.x;
    a.weight = b.weight;
    a.dy = b.dy;
    a.y = b.dx;
    a.mean = const_cast<float*>(b.mean);
    a.rstd = const_cast<float*>(b.rstd);
    a.x_stride = b.x_stride;
    a.y_stride = b.dx_stride;
    a.dy_stride = b.dy_stride;
    a.rows = s.rows;
    a.cols = s.features;
    a.eps = s.eps;
    a.wants_dx = b.dx != nullptr;
    return by_types(s.type, s.out_type, [&](auto t, auto o) { return backward<decltype(t), decltype(o)>(st, a, b); });
}

}  // namespace chimera
