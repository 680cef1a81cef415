// Layer norm and its gradients (include/chimera_operators.h):
//   z = (x - mean) rstd,  rstd = (mean of (x - mean)^2 + eps)^-1/2,  y = z w + b
//   g = dy w,  dx = rstd (g - mean of g - z mean of g z),
//   dw = the sum over rows of dy z,  db = that of dy
#include "operators.hpp"

#include <algorithm>

namespace chimera {

namespace {

int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

// Rows whose squares pass the 32-bit range are taken times kSmall, and so are
// those in the backward pass whose rstd is below kLowRstd.
constexpr float kSmall = 0x1p-80f, kLarge = 0x1p80f, kLowRstd = 0x1p-60f;

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

// ---- forward -------------------------------------------------------------------

// A row's values stay in registers, 8 kChunks a thread, and are read once. The
// variance is taken about a mean that is corrected by what is left of the
// row's sum after it, so that rows far from zero keep their digits.
template <typename T, typename Out, int kLanes, int kChunks>
__global__ __launch_bounds__(block_threads(kLanes)) void norm_forward_kernel(NormArgs a) {
    constexpr int kRows = block_threads(kLanes) / kLanes;
    __shared__ float lds[kLanes > kWave ? kLanes / kWave * 2 : 1];
    const int t = static_cast<int>(threadIdx.x) % kLanes;
    const float inv = 1.0f / static_cast<float>(a.cols);
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + static_cast<int>(threadIdx.x) / kLanes; r < a.rows;
         r += static_cast<int64_t>(gridDim.x) * kRows) {
        float x[kChunks][8] = {};
        const T* from = static_cast<const T*>(a.x) + r * a.x_stride;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const int c = (j * kLanes + t) * 8;
            if (c < a.cols) load8(from + c, a.cols - c, x[j]);
        }
        float scale = 1.0f, mean, rest, rstd;
        for (;;) {
            float sum[1] = {0.0f};
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[0] += x[j][i] * scale;
            row_sums<kLanes>(sum, lds);
            mean = sum[0] * inv;
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < kChunks; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = (j * kLanes + t) * 8 + i < a.cols ? fmaf(x[j][i], scale, -mean) : 0.0f;
                    s[0] += d;
                    s[1] = fmaf(d, d, s[1]);
                }
            row_sums<kLanes>(s, lds);
            rest = s[0] * inv;
            const float var = fmaf(-rest, rest, s[1] * inv);
            rstd = 1.0f / sqrtf(var + a.eps * scale * scale);
            if (scale != 1.0f || s[1] - s[1] == 0.0f) break;
            scale = kSmall;
        }
        if (t == 0) {
            if (a.mean) a.mean[r] = (mean + rest) * (scale == 1.0f ? 1.0f : kLarge);
            if (a.rstd) a.rstd[r] = rstd * scale;
        }
        Out* to = static_cast<Out*>(a.y) + r * a.y_stride;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const int c = (j * kLanes + t) * 8;
            const int count = a.cols - c;
            if (count <= 0) break;
            float w[8], b[8] = {};
            if (a.weight)
                load8(static_cast<const T*>(a.weight) + c, count, w);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = 1.0f;
            if (a.bias) load8(static_cast<const T*>(a.bias) + c, count, b);
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf((fmaf(x[j][i], scale, -mean) - rest) * rstd, w[i], b[i]);
            store8(to + c, count, v);
        }
    }
}

// ---- backward ------------------------------------------------------------------

// x and dy are read once and stay in registers, as do the thread's columns of
// the sums over rows; these are joined over the block's rows in order and
// written for the join. What the rounding of the mean left out is the sum of
// x - mean, and is taken away again.
template <typename T, typename Out, int kLanes, int kChunks>
__global__ __launch_bounds__(block_threads(kLanes)) void norm_backward_kernel(NormArgs a) {
    constexpr int kRows = block_threads(kLanes) / kLanes;
    __shared__ float lds[kLanes > kWave ? kLanes / kWave * 3 : kRows > 1 ? kRows * kLanes * 8 : 1];
    const int t = static_cast<int>(threadIdx.x) % kLanes, in_block = static_cast<int>(threadIdx.x) / kLanes;
    const float inv = 1.0f / static_cast<float>(a.cols);
    float w[kChunks][8], dw[kChunks][8] = {}, db[kChunks][8] = {};
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
        const int c = (j * kLanes + t) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[j][i] = 1.0f;
        if (a.weight && c < a.cols) load8(static_cast<const T*>(a.weight) + c, a.cols - c, w[j]);
    }
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + in_block; r < a.rows;
         r += static_cast<int64_t>(gridDim.x) * kRows) {
        float x[kChunks][8] = {}, dy[kChunks][8] = {};
        const T* from = static_cast<const T*>(a.x) + r * a.x_stride;
        const Out* grad = static_cast<const Out*>(a.dy) + r * a.dy_stride;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            const int c = (j * kLanes + t) * 8;
            if (c < a.cols) {
                load8(from + c, a.cols - c, x[j]);
                load8(grad + c, a.cols - c, dy[j]);
            }
        }
        const float rstd = a.rstd[r];
        const bool low = rstd < kLowRstd;
        const float scale = low ? kSmall : 1.0f, mean = a.mean[r] * scale, by = low ? rstd * kLarge : rstd;
        float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool in = (j * kLanes + t) * 8 + i < a.cols;
                const float d = in ? fmaf(x[j][i], scale, -mean) : 0.0f;
                const float g = in ? dy[j][i] * w[j][i] : 0.0f;
                x[j][i] = d;
                s[0] += d;
                s[1] += g;
                s[2] = fmaf(g, d, s[2]);
            }
        row_sums<kLanes>(s, lds);
        const float rest = s[0] * inv, mean_g = s[1] * inv;
        const float mean_gz = by * fmaf(-rest, s[1], s[2]) * inv;
        T* to = static_cast<T*>(a.y) + r * a.y_stride;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = (x[j][i] - rest) * by;
                v[i] = rstd * fmaf(-z, mean_gz, fmaf(dy[j][i], w[j][i], -mean_g));
                dw[j][i] = fmaf(dy[j][i], z, dw[j][i]);
                db[j][i] += dy[j][i];
            }
            const int c = (j * kLanes + t) * 8;
            if (a.wants_dx && c < a.cols) store8(to + c, a.cols - c, v);
        }
    }
    if (!a.parts) return;
    // rows of the block in order, then the block's sums
    float* part = a.parts + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int c = (j * kLanes + t) * 8;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = which ? db[j][i] : dw[j][i];
            if constexpr (kRows > 1) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) lds[(in_block * 8 + i) * kLanes + t] = v[i];
                __syncthreads();
                if (in_block == 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        float sum = 0.0f;
#pragma unroll
                        for (int o = 0; o < kRows; ++o) sum += lds[(o * 8 + i) * kLanes + t];
                        v[i] = sum;
                    }
                }
            }
            if (in_block == 0 && c < a.cols) store8(part + which * a.cols + c, a.cols - c, v);
        }
}

// Rows too long for registers: two passes over a row, the second from the
// caches. `rests` [rows] gets what the saved mean left out.
template <typename T, typename Out>
__global__ __launch_bounds__(1024) void norm_wide_kernel(NormArgs a, float* rests) {
    __shared__ float lds[16 * 3];
    const float inv = 1.0f / static_cast<float>(a.cols);
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
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
                    x[i] = i < count ? fmaf(x[i], scale, -mean) : 0.0f;
                    dy[i] = i < count ? a.weight ? dy[i] * w[i] : dy[i] : 0.0f;
                }
                visit(c, count, x, dy);
            }
        };
        float s[3] = {0.0f, 0.0f, 0.0f};
        each([&](int, int, float(&d)[8], float(&g)[8]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[0] += d[i];
                s[1] += g[i];
                s[2] = fmaf(g[i], d[i], s[2]);
            }
        });
        row_sums<1024>(s, lds);
        const float rest = s[0] * inv, mean_g = s[1] * inv;
        const float mean_gz = by * fmaf(-rest, s[1], s[2]) * inv;
        if (rests && threadIdx.x == 0) rests[r] = rest;
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
        float x[8], dy[8];
        load8(static_cast<const T*>(a.x) + r * a.x_stride + c, count, x);
        load8(static_cast<const Out*>(a.dy) + r * a.dy_stride + c, count, dy);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            dw[i] = fmaf(dy[i], (fmaf(x[i], scale, -mean) - rests[r]) * by, dw[i]);
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
constexpr int kMostParts = 512;

// Parts of the sums over rows, as many as blocks: grows with the rows.
int64_t parts_of(int64_t rows, int cols) {
    if (cols > kMostRegisters) return std::min<int64_t>(rows, 64);
    const int lanes = cols <= 128 ? 16 : cols <= 1024 ? 64 : 256;
    return std::min<int64_t>(ceil_div(rows, 256 / lanes), kMostParts);
}

template <typename T, typename Out>
hipError_t forward(hipStream_t st, const NormArgs& a) {
    auto launch = [&](auto kernel, int lanes) {
        const int threads = block_threads(lanes);
        const int64_t blocks = ceil_div(a.rows, threads / lanes);
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min<int64_t>(blocks, 1 << 20))),
                           dim3(static_cast<unsigned>(threads)), 0, st, a);
        return hipGetLastError();
    };
    if (a.cols <= 128) return launch(norm_forward_kernel<T, Out, 16, 1>, 16);
    if (a.cols <= 512) return launch(norm_forward_kernel<T, Out, 64, 1>, 64);
    if (a.cols <= 1024) return launch(norm_forward_kernel<T, Out, 64, 2>, 64);
    if (a.cols <= 2048) return launch(norm_forward_kernel<T, Out, 256, 1>, 256);
    if (a.cols <= 4096) return launch(norm_forward_kernel<T, Out, 256, 2>, 256);
    if (a.cols <= 8192) return launch(norm_forward_kernel<T, Out, 256, 4>, 256);
    if (a.cols <= 32768) return launch(norm_forward_kernel<T, Out, 1024, 4>, 1024);
    return launch(norm_forward_kernel<T, Out, 1024, 8>, 1024);
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
    auto launch = [&](auto kernel, int lanes) {
        const int threads = block_threads(lanes);
        const int64_t blocks = sums ? parts : std::min<int64_t>(ceil_div(a.rows, threads / lanes), 1 << 20);
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(static_cast<unsigned>(threads)), 0, st, a);
    };
    if (a.cols <= 128)
        launch(norm_backward_kernel<T, Out, 16, 1>, 16);
    else if (a.cols <= 512)
        launch(norm_backward_kernel<T, Out, 64, 1>, 64);
    else if (a.cols <= 1024)
        launch(norm_backward_kernel<T, Out, 64, 2>, 64);
    else if (a.cols <= 2048)
        launch(norm_backward_kernel<T, Out, 256, 1>, 256);
    else if (a.cols <= 4096)
        launch(norm_backward_kernel<T, Out, 256, 2>, 256);
    else if (a.cols <= kMostRegisters)
        launch(norm_backward_kernel<T, Out, 256, 4>, 256);
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
    const int64_t rests = s.features > kMostRegisters ? s.rows : 0;
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
