// The quantised token cache (include/chimera_operators.h): rows written as
// codes with one scale per group of values, read back, and late interaction
//   score(q, d) = sum over tokens i of q of max over tokens t of d of <q_i, x_t>
// on the codes as they lie in the cache's pages.
#include "operators.hpp"

#include <algorithm>
#include <type_traits>

namespace chimera {

namespace {

int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

// A group whose largest magnitude is below this is stored as zeros: top / max
// and max / top stay within the normal 32-bit range (448 * 2^117 < 2^126).
constexpr float kLeastGroup = 0x1p-117f;

template <int kFormat>
constexpr float top_code() {
    return kFormat == CHIMERA_CACHE_INT8 ? 127.0f : kFormat == CHIMERA_CACHE_INT4 ? 7.0f : 448.0f;
}

struct CacheView {
    uint8_t* codes;
    float* scales;
    int64_t slots, num_pages;
    int dim, row_bytes, row_scales;
    int group_log2;  // of values per scale
    int page_log2;   // of tokens per page
};

CacheView view_of(const chimera_cache& c) {
    CacheView v;
    v.codes = c.codes;
    v.scales = c.scales;
    v.slots = c.num_pages * c.page_tokens;
    v.num_pages = c.num_pages;
    v.dim = c.dim;
    v.row_bytes = cache_row_bytes(c);
    v.row_scales = cache_row_scales(c);
    v.group_log2 = c.group == 32 ? 5 : c.group == 64 ? 6 : 7;
    v.page_log2 = __builtin_ctz(static_cast<unsigned>(c.page_tokens));
    return v;
}

// ---- writing -------------------------------------------------------------------

// scale = max |x| / top of a group, code = round(x * (top / max)). 16 lanes a
// row, eight neighbouring values a lane (whole 16-byte loads): a group is 4, 8
// or 16 neighbouring lanes, its maximum four exchanges in the vector unit. One
// pass, bound by memory, of which 64-byte code rows at random slots are the
// slow part: 2M rows of 128 bf16 values to 4-bit codes and four scales, 0.69
// GB, take 181 us (3.8 TB/s).
template <typename T, int kFormat, bool kOnce>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheView c, const T* __restrict__ rows, int64_t stride,
                                                          const int64_t* __restrict__ slots, int64_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
    const int col = static_cast<int>(threadIdx.x) % 16 * 8;
    const int64_t slot = i < n ? slots[i] : -1;
    const bool in = slot >= 0 && slot < c.slots;
    float x[8] = {};
    if (in && col < c.dim) load8<T, kOnce>(rows + i * stride + col, c.dim - col, x);
    float most = 0.0f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        most = fmaxf(most, fabsf(x[j]));
        bad |= !(fabsf(x[j]) <= 3.402823466e38f);
    }
    if (bad) most = INFINITY;
    const int lanes = 1 << (c.group_log2 - 3);
    for (int o = 1; o < lanes; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, kWave));
    constexpr float kTop = top_code<kFormat>();
    const bool finite = most <= 3.402823466e38f;
    const bool zero = most < kLeastGroup || !finite;
    const float inv = zero ? 0.0f : kTop * (1.0f / most);
    const float scale = !finite ? NAN : zero ? 0.0f : most * (1.0f / kTop);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = zero ? 0.0f : x[j] * inv;
        if (kFormat != CHIMERA_CACHE_FP8) v[j] = rintf(v[j]);
        v[j] = fminf(fmaxf(v[j], -kTop), kTop);
    }
    if (!in) return;
    if (col < (c.dim + 31) / 32 * 32) {
        uint8_t* dst = c.codes + slot * c.row_bytes;
        if constexpr (kFormat == CHIMERA_CACHE_INT4) {
            uint32_t u = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) u |= static_cast<uint32_t>(static_cast<int>(v[j]) + 8) << (4 * j);
            *reinterpret_cast<uint32_t*>(dst + col / 2) = u;
        } else {
            u32x2_t u = {0, 0};
            if constexpr (kFormat == CHIMERA_CACHE_INT8) {
#pragma unroll
                for (int j = 0; j < 8; ++j) u[j / 4] |= (static_cast<uint32_t>(static_cast<int>(v[j])) & 0xFFu) << (8 * (j % 4));
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j], v[4 * j + 1], 0, false);
                    p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j + 2], v[4 * j + 3], p, true);
                    u[j] = static_cast<uint32_t>(p);
                }
            }
            *reinterpret_cast<u32x2_t*>(dst + col) = u;
        }
    }
    if (col < c.dim && (col & ((1 << c.group_log2) - 1)) == 0)
        c.scales[slot * c.row_scales + (col >> c.group_log2)] = scale;
}

// ---- reading -------------------------------------------------------------------

// x = code * scale, laid out as for writing. Bound by memory: 2M rows of 128
// 4-bit codes to bf16, 0.69 GB, take 143 us (4.8 TB/s).
template <typename T, int kFormat, bool kOnce>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheView c, const int64_t* __restrict__ slots, int64_t n,
                                                         T* __restrict__ out, int64_t stride) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16;
    const int col = static_cast<int>(threadIdx.x) % 16 * 8;
    if (i >= n || col >= c.dim) return;
    const int64_t slot = slots[i];
    float v[8] = {};
    if (slot >= 0 && slot < c.slots) {
        const uint8_t* src = c.codes + slot * c.row_bytes;
        const float scale = c.scales[slot * c.row_scales + (col >> c.group_log2)];
        if constexpr (kFormat == CHIMERA_CACHE_INT4) {
            const uint32_t u = *reinterpret_cast<const uint32_t*>(src + col / 2);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(static_cast<int>((u >> (4 * j)) & 15u) - 8);
        } else {
            const u32x2_t u = *reinterpret_cast<const u32x2_t*>(src + col);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (kFormat == CHIMERA_CACHE_INT8)
                    v[j] = static_cast<float>(static_cast<int8_t>(u[j / 4] >> (8 * (j % 4))));
                else
                    v[j] = __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(u[j / 4] >> (8 * (j % 4))), 0);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= scale;
    }
    store8<T, kOnce>(out + i * stride + col, c.dim - col, v);
}

// ---- late interaction ----------------------------------------------------------

// Eight codes as fp16 values, exactly, in the order code_order() gives.
__device__ __forceinline__ f16x8_t int8_values(u32x2_t u) {
    // a byte plus 128 below the exponent of 1024 is 1152 + code
    const f16x2_t bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
    f16x8_t v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t x = u[j] ^ 0x80808080u;
        const f16x2_t lo = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - bias;
        const f16x2_t hi = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - bias;
        v[4 * j] = lo[0];
        v[4 * j + 1] = lo[1];
        v[4 * j + 2] = hi[0];
        v[4 * j + 3] = hi[1];
    }
    return v;
}
__device__ __forceinline__ f16x8_t int4_values(uint32_t u) {
    // a stored code below the exponent of 1024 is 1032 + code. (Its bits alone,
    // multiples of fp16's least value, cost as much and the products of such
    // values lost four bits in the matrix instruction's sums.)
    const f16x2_t bias = {static_cast<_Float16>(1032.0f), static_cast<_Float16>(1032.0f)};
    f16x8_t v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f16x2_t p = __builtin_bit_cast(f16x2_t, ((u >> (4 * j)) & 0x000F000Fu) | 0x64006400u) - bias;
        v[2 * j] = p[0];
        v[2 * j + 1] = p[1];
    }
    return v;
}
__device__ __forceinline__ f16x8_t fp8_values(u32x2_t u) {
    f16x8_t v;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u[j], 1.0f, false);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u[j], 1.0f, true);
        v[4 * j] = lo[0];
        v[4 * j + 1] = lo[1];
        v[4 * j + 2] = hi[0];
        v[4 * j + 3] = hi[1];
    }
    return v;
}
// Which of eight neighbouring values the j-th one is.
template <int kFormat>
__device__ __forceinline__ constexpr int code_order(int j) {
    return kFormat == CHIMERA_CACHE_INT4 ? (j & 1) * 4 + j / 2 : j;
}

struct MaxsimArgs {
    CacheView c;
    const void* queries;
    const int32_t* query_lens;
    const int64_t* page_start;
    const int32_t* doc_lens;
    const int32_t* pages;
    const int32_t* cand_ids;
    const int32_t* cand_counts;
    float* scores;
    float* parts;  // [nq * cap][splits][query rows] maxima where documents are split
    int64_t num_docs, num_page_entries;
    int nq, query_len, cap;
    int split_tokens, splits, max_tokens;
    int items;  // parts of documents a wave takes, 1..64
};

// The query row whose maximum lane l ends up with (maxima_to_rows).
__device__ __forceinline__ int row_of_lane(int l) {
    const int r = ((l >> 4) & 1) * 8 + ((l >> 3) & 1) * 4 + ((l >> 2) & 1) * 2 + ((l >> 1) & 1);
    return 8 * (r >> 2) + 4 * (l >> 5) + (r & 3);
}

// One query tile of 32 tokens as matrix operand (rows: query tokens), in fp16
// parts after a power of two per token that brings its largest value to
// [0.5, 1); kParts 2 keeps 22 bits of 32-bit queries. A token past the end is
// zeros.
template <typename T, int kFormat, int kParts>
struct QueryTile {
    f16x8_t part[kParts][4][2];
    float back;  // 2^e of row_of_lane's row; 0 in the lanes that do not count it

    __device__ __forceinline__ void load(const T* q, int rows, int dim, int l) {
        const int row = l & 31, half = l >> 5;
        float x[4][2][8];
        float most = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = 32 * g + 16 * half + 8 * h;
                const int count = row < rows ? dim - at : 0;
                load8(q + static_cast<int64_t>(row) * dim + at, count, x[g][h]);
#pragma unroll
                for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(x[g][h][j]));
            }
        most = fmaxf(most, __shfl_xor(most, 32, kWave));
        int e = 0;
        frexpf(most > 0.0f ? most : 1.0f, &e);
        // 2^e and 2^-e are normal numbers; the largest queries come to [2, 4) and
        // those below the normal numbers, which have fewer bits, to less than 0.5
        e = min(max(e, -126), 126);
        const float to = ldexpf(1.0f, -e);
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = x[g][h][code_order<kFormat>(j)] * to;
                    const _Float16 hi = static_cast<_Float16>(v);
                    part[0][g][h][j] = hi;
                    if constexpr (kParts == 2) part[1][g][h][j] = static_cast<_Float16>(v - static_cast<float>(hi));
                }
        back = __shfl(ldexpf(1.0f, e), row_of_lane(l), kWave);
        if ((l & 1) != 0 || row_of_lane(l) >= rows) back = 0.0f;
    }
};

// Maxima over the 32 lanes of each half of the wave of 16 values a lane: each
// step leaves a lane half of the values, the last one all lanes of a pair the
// same one (lane bits 4 to 1 choose it). All in the vector unit.
__device__ __forceinline__ float maxima_to_rows(float (&v)[16], int l) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[r]), __float_as_uint(v[r + 8]), false, false);
        v[r] = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    auto step = [&](int bit, int keep, auto ctrl) {
        const bool upper = (l & bit) != 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (r >= keep) continue;
            const float mine = upper ? v[r + keep] : v[r], theirs = upper ? v[r] : v[r + keep];
            v[r] = fmaxf(mine, lane_move<decltype(ctrl)::value>(theirs));
        }
    };
    step(8, 4, std::integral_constant<int, kRotate8>{});
    step(4, 2, std::integral_constant<int, kMirror8>{});
    step(2, 1, std::integral_constant<int, kSwap2>{});
    return fmaxf(v[0], lane_move<kSwap1>(v[0]));
}
// A wave scores `items` parts of documents (whole documents unless they are
// split) against one query, tile after tile of 32 tokens (matrix columns)
// with no break between documents: the codes of the next tile and the page
// numbers of the one after it are on their way while a tile is multiplied.
// Lane l holds of token l % 32 and each run of 32 values the 16 from
// 16 (l / 32) on; a tile's scores are 16 query rows a lane, of one token, so
// that the token's scale and the running maxima need no exchange before the
// document's end. Lanes past a document's last token take that token again;
// an absent token has NaN for its scale, which the maxima pass over.
// kRuns: runs of 32 values that share a scale: 1, 2, or 4 for one scale a row.
// Bound by reading the codes, whole pages in no order, and by the vector work
// a tile: 76,800 documents of 16 to 256 tokens, 8-bit codes, 32-bit queries of
// 32 tokens, 1.38 GB, take 320 us (4.3 TB/s); half as many of fp8 codes with
// bf16 queries 151, of 4-bit codes 142. Loads past the caches (453 us instead
// of 320) and other numbers of documents a wave were slower.
template <typename T, int kFormat, int kRuns>
__global__ __launch_bounds__(256) void cache_maxsim_kernel(MaxsimArgs a) {
    constexpr int kParts = sizeof(T) == 4 ? 2 : 1;
    constexpr int kScales = 4 / kRuns;
    const int l = lane_id();
    const int q = static_cast<int>(blockIdx.y);
    const int w = __builtin_amdgcn_readfirstlane(wave_id());
    const int64_t first_item = static_cast<int64_t>(blockIdx.x) * 4 * a.items + w;
    const int64_t total = static_cast<int64_t>(a.cap) * a.splits;

    // lane i: the wave's i-th item, number first_item + 4 i
    int my_begin = 0, my_end = 0, my_first_lo = 0, my_first_hi = 0;
    const int64_t my_item = first_item + 4 * l;
    bool scored = false;  // a score that is not -inf is still to come
    if (l < a.items && my_item < total) {
        const int j = static_cast<int>(my_item / a.splits), split = static_cast<int>(my_item - static_cast<int64_t>(j) * a.splits);
        const int64_t at = static_cast<int64_t>(q) * a.cap + j;
        const int count = a.cand_counts ? a.cand_counts[q] : a.cap;
        const int doc = j < count ? a.cand_ids[at] : -1;
        if (doc >= 0 && doc < a.num_docs) {
            const int len = min(a.doc_lens[doc], a.max_tokens);
            const int64_t first = a.page_start[doc];
            my_begin = split * a.split_tokens;
            my_end = min(len, my_begin + a.split_tokens);
            my_first_lo = static_cast<int>(first);
            my_first_hi = static_cast<int>(first >> 32);
            scored = my_begin < my_end;
        }
        if (!scored && a.splits == 1) a.scores[at] = -INFINITY;
    }
    const uint64_t work = __ballot(scored);
    if (work == 0) return;
    const int q_len = a.query_lens ? min(max(a.query_lens[q], 0), a.query_len) : a.query_len;
    const int groups = (a.c.dim + 31) / 32;
    const int half = l >> 5;
    const int rows_padded = (a.query_len + 31) / 32 * 32;

    struct Cursor {
        uint64_t left;  // items from this one on
        int item, t, end;
        int64_t first;
    };
    auto enter = [&](Cursor& c) {
        c.item = c.left ? __builtin_ctzll(c.left) : c.item;  // past the end: the last item again
        c.t = __builtin_amdgcn_readlane(my_begin, c.item);
        c.end = __builtin_amdgcn_readlane(my_end, c.item);
        c.first = (static_cast<int64_t>(__builtin_amdgcn_readlane(my_first_hi, c.item)) << 32) |
                  static_cast<uint32_t>(__builtin_amdgcn_readlane(my_first_lo, c.item));
    };
    auto advance = [&](Cursor& c) {
        c.t += 32;
        if (c.t < c.end) return;
        c.left &= c.left - 1;
        enter(c);
    };
    // the token's page number, -1 for none
    auto load_page = [&](const Cursor& c) {
        const int64_t entry = c.first + (min(c.t + (l & 31), c.end - 1) >> a.c.page_log2);
        return entry >= 0 && entry < a.num_page_entries ? a.pages[entry] : -1;
    };
    struct Tile {
        u32x4_t codes[kFormat == CHIMERA_CACHE_INT4 ? 2 : 4];
        float scale[kScales];
    };
    auto load_codes = [&](const Cursor& c, int page, Tile& tile) {
        const int t = min(c.t + (l & 31), c.end - 1);
        const bool in = page >= 0 && page < a.c.num_pages;
        const int64_t slot = in ? (static_cast<int64_t>(page) << a.c.page_log2) + (t & ((1 << a.c.page_log2) - 1)) : 0;
        const uint8_t* codes = a.c.codes + slot * a.c.row_bytes;
        if constexpr (kFormat == CHIMERA_CACHE_INT4) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (g < groups) {
                    const u32x2_t u = *reinterpret_cast<const u32x2_t*>(codes + 16 * g + 8 * half);
                    tile.codes[g / 2][2 * (g % 2)] = u[0];
                    tile.codes[g / 2][2 * (g % 2) + 1] = u[1];
                }
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (g < groups) tile.codes[g] = *reinterpret_cast<const u32x4_t*>(codes + 32 * g + 16 * half);
        }
        const float* scales = a.c.scales + slot * a.c.row_scales;
#pragma unroll
        for (int i = 0; i < kScales; ++i)
            if (i < a.c.row_scales) tile.scale[i] = in ? scales[i] : NAN;
    };

    for (int q0 = 0; q0 < rows_padded; q0 += 32) {
        if (q0 >= q_len && q0 > 0) break;
        QueryTile<T, kFormat, kParts> qt;
        qt.load(static_cast<const T*>(a.queries) + (static_cast<int64_t>(q) * a.query_len + q0) * a.c.dim, q_len - q0,
                a.c.dim, l);
        float best[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) best[r] = -INFINITY;

        auto run = [&](const Tile& tile, int g, f32x16_t acc) {
            f16x8_t v0, v1;
            if constexpr (kFormat == CHIMERA_CACHE_INT4) {
                v0 = int4_values(tile.codes[g / 2][2 * (g % 2)]);
                v1 = int4_values(tile.codes[g / 2][2 * (g % 2) + 1]);
            } else {
                const u32x4_t u = tile.codes[g];
                v0 = kFormat == CHIMERA_CACHE_INT8 ? int8_values(u32x2_t{u[0], u[1]}) : fp8_values(u32x2_t{u[0], u[1]});
                v1 = kFormat == CHIMERA_CACHE_INT8 ? int8_values(u32x2_t{u[2], u[3]}) : fp8_values(u32x2_t{u[2], u[3]});
            }
#pragma unroll
            for (int s = 0; s < kParts; ++s) {
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qt.part[s][g][0], v0, acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(qt.part[s][g][1], v1, acc, 0, 0, 0);
            }
            return acc;
        };
        auto multiply = [&](const Tile& tile) {
            f32x16_t sum;
#pragma unroll
            for (int i = 0; i < kScales; ++i) {
                if (i > 0 && i * kRuns >= groups) break;
                f32x16_t acc = run(tile, i * kRuns, f32x16_t{});
#pragma unroll
                for (int g = 1; g < kRuns; ++g)
                    if (i * kRuns + g < groups) acc = run(tile, i * kRuns + g, acc);
#pragma unroll
                for (int r = 0; r < 16; ++r) sum[r] = i == 0 ? acc[r] * tile.scale[0] : fmaf(acc[r], tile.scale[i], sum[r]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) best[r] = fmaxf(best[r], sum[r]);
        };
        // after an item's last tile
        auto finish = [&](const Cursor& c) {
            const float top = maxima_to_rows(best, l);
#pragma unroll
            for (int r = 0; r < 16; ++r) best[r] = -INFINITY;
            const float v = qt.back > 0.0f ? top * qt.back : 0.0f;
            const int64_t item = first_item + 4 * c.item;
            if (a.splits > 1) {
                if ((l & 1) == 0)
                    a.parts[(static_cast<int64_t>(q) * total + item) * rows_padded + q0 + row_of_lane(l)] = v;
                return;
            }
            float s = wave_sum(v);
            float* score = a.scores + static_cast<int64_t>(q) * a.cap + item;
            if (l == 0) *score = q0 > 0 ? *score + s : s;
        };

        Cursor now{work, 0, 0, 0, 0};
        enter(now);
        Cursor next = now;
        advance(next);
        Cursor after = next;
        advance(after);
        Tile t0, t1;
        load_codes(now, load_page(now), t0);
        int page = load_page(next);
        auto round = [&](Tile& mine, Tile& other) {
            load_codes(next, page, other);
            page = load_page(after);
            multiply(mine);
            if (next.item != now.item || next.left == 0) finish(now);
            now = next;
            next = after;
            advance(after);
        };
        while (true) {
            round(t0, t1);
            if (now.left == 0) break;
            round(t1, t0);
            if (now.left == 0) break;
        }
    }
}

// The parts of split documents: a block a candidate, a lane a query token
// (half a wave's lanes each of 32 tokens), the half waves share the parts.
__global__ __launch_bounds__(512) void cache_maxsim_join_kernel(MaxsimArgs a) {
    __shared__ float best[16][32];
    const int l = lane_id();
    const int row = l & 31, group = static_cast<int>(threadIdx.x) / 32;
    const int q = static_cast<int>(blockIdx.y), j = static_cast<int>(blockIdx.x);
    const int64_t at = static_cast<int64_t>(q) * a.cap + j;
    const int count = a.cand_counts ? a.cand_counts[q] : a.cap;
    const int doc = j < count ? a.cand_ids[at] : -1;
    const int len = doc >= 0 && doc < a.num_docs ? min(a.doc_lens[doc], a.max_tokens) : 0;
    const int q_len = a.query_lens ? min(max(a.query_lens[q], 0), a.query_len) : a.query_len;
    const int rows_padded = (a.query_len + 31) / 32 * 32;
    const int parts = (len + a.split_tokens - 1) / a.split_tokens;
    float total = 0.0f;
    for (int q0 = 0; q0 < q_len; q0 += 32) {
        float m = -INFINITY;
#pragma unroll 4
        for (int p = group; p < parts; p += 16) m = fmaxf(m, a.parts[(at * a.splits + p) * rows_padded + q0 + row]);
        best[group][row] = m;
        __syncthreads();
        if (threadIdx.x < 32) {
#pragma unroll
            for (int g = 1; g < 16; ++g) m = fmaxf(m, best[g][row]);
            total += q0 + row < q_len ? m : 0.0f;
        }
        __syncthreads();
    }
    if (threadIdx.x >= 32) return;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) total += __shfl_xor(total, o, kWave);
    if (threadIdx.x == 0) a.scores[at] = parts > 0 ? total : -INFINITY;
}

// The best k candidates of a query by score, ties to the larger id: one block
// of 1,024 threads sorts them all.
__global__ __launch_bounds__(1024) void cache_topk_kernel(const float* __restrict__ scores,
                                                          const int32_t* __restrict__ ids,
                                                          const int32_t* __restrict__ counts, int cap, int sort_cap, int k,
                                                          int64_t* __restrict__ top_ids, float* __restrict__ top_scores,
                                                          int32_t* __restrict__ top_counts) {
    extern __shared__ uint64_t keys[];
    const int64_t q = blockIdx.x;
    const int n = counts ? min(max(counts[q], 0), cap) : cap;
    for (int t = threadIdx.x; t < sort_cap; t += 1024) {
        uint64_t key = ~0ull;
        if (t < n) {
            // descending (score, id) as an ascending key; the sign bit makes
            // absent candidates' negative ids the smallest
            const uint32_t id = static_cast<uint32_t>(ids[q * cap + t]) ^ 0x80000000u;
            key = ~((static_cast<uint64_t>(float_to_ordered(scores[q * cap + t])) << 32) | id);
        }
        keys[t] = key;
    }
    __syncthreads();
    block_sort_u64(keys, sort_cap);
    for (int64_t t = threadIdx.x; t < k; t += 1024) {
        const uint64_t v = t < n ? ~keys[t] : 0ull;
        top_ids[q * k + t] = t < n ? static_cast<int32_t>(static_cast<uint32_t>(v) ^ 0x80000000u) : -1;
        if (top_scores) top_scores[q * k + t] = t < n ? ordered_to_float(static_cast<uint32_t>(v >> 32)) : 0.0f;
    }
    if (threadIdx.x == 0) top_counts[q] = min(k, n);
}

// How documents are split: four waves for each of the 1,024 SIMDs where there
// are fewer candidates, 128 tokens a part at least. Joining the parts is a launch
// of its own, so documents of less than 512 tokens stay whole. One query, us,
// by the least tokens of a part (128 / 256 / 512):
//     10 candidates of up to 4,000 tokens      11.7 / 14.2 / 20.0
//     8 of 30,000 to 60,000                    19.2 / 21.0 / 24.8
//     100 of up to 300                         11.2 / 11.0 / 11.0 (whole)
// and 1,000 of up to 300 split in two 17.2, whole 13.7. Candidates are counted
// by their capacity, which the host knows, and not by those that are filled,
// and from 2,049 on none is split, however long: a call with a few long
// documents does better with a capacity near their number.
struct Split {
    int tokens, count;
};
Split split_of(const chimera_cache_maxsim& m) {
    constexpr int64_t kWaves = 4096;
    const int64_t docs = static_cast<int64_t>(m.nq) * m.cand_cap;
    const int64_t longest = std::max(m.max_doc_tokens, 1);
    const int64_t count =
        longest < 512 ? 1 : std::max<int64_t>(1, std::min(kWaves / std::max<int64_t>(docs, 1), longest / 128));
    Split s;
    s.tokens = static_cast<int>(ceil_div(ceil_div(longest, count), 32) * 32);
    s.count = static_cast<int>(ceil_div(longest, s.tokens));
    return s;
}

// Parts of documents a wave takes: as many as leave 8,192 waves, at most 16.
int items_of(int64_t parts) { return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(parts / 8192, 16))); }

template <typename Call>
hipError_t by_format(int format, int type, Call&& call) {
    auto by_type = [&](auto f) {
        switch (type) {
            case CHIMERA_F32: call(f, float{}); break;
            case CHIMERA_F16: call(f, _Float16{}); break;
            default: call(f, __bf16{}); break;
        }
    };
    switch (format) {
        case CHIMERA_CACHE_INT8: by_type(std::integral_constant<int, CHIMERA_CACHE_INT8>{}); break;
        case CHIMERA_CACHE_INT4: by_type(std::integral_constant<int, CHIMERA_CACHE_INT4>{}); break;
        default: by_type(std::integral_constant<int, CHIMERA_CACHE_FP8>{}); break;
    }
    return hipGetLastError();
}

// Rows that fill the GPU's L2 (8 x 4 MB) several times over are neither kept in
// it nor fetched from it: 2M rows of 128 16-bit values written and read back
// take 402 us through the caches, 372 past them.
bool passes_caches(const chimera_cache& c, int64_t n, int type) {
    return n * c.dim * static_cast<int64_t>(type_bytes(type)) > (int64_t{128} << 20);
}

}  // namespace

hipError_t launch_cache_write(hipStream_t st, const chimera_cache& c, const void* rows, int type, int64_t stride,
                              const int64_t* slots, int64_t n) {
    const CacheView v = view_of(c);
    const unsigned blocks = static_cast<unsigned>(ceil_div(n, 16));
    const bool once = passes_caches(c, n, type);
    return by_format(c.format, type, [&](auto f, auto t) {
        using T = decltype(t);
        auto* kernel = once ? cache_write_kernel<T, decltype(f)::value, true> : cache_write_kernel<T, decltype(f)::value, false>;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, v, static_cast<const T*>(rows), stride, slots, n);
    });
}

hipError_t launch_cache_read(hipStream_t st, const chimera_cache& c, const int64_t* slots, int64_t n, void* out,
                             int type, int64_t stride) {
    const CacheView v = view_of(c);
    const unsigned blocks = static_cast<unsigned>(ceil_div(n, 16));
    const bool once = passes_caches(c, n, type);
    return by_format(c.format, type, [&](auto f, auto t) {
        using T = decltype(t);
        auto* kernel = once ? cache_read_kernel<T, decltype(f)::value, true> : cache_read_kernel<T, decltype(f)::value, false>;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, v, slots, n, static_cast<T*>(out), stride);
    });
}

size_t cache_maxsim_workspace(const chimera_cache_maxsim& m) {
    const Split s = split_of(m);
    if (s.count <= 1) return 0;
    return static_cast<size_t>(m.nq) * m.cand_cap * s.count * (ceil_div(m.query_len, 32) * 32) * sizeof(float);
}

hipError_t launch_cache_maxsim(hipStream_t st, const chimera_cache& c, const chimera_cache_maxsim& m) {
    const Split s = split_of(m);
    MaxsimArgs a = {};
    a.c = view_of(c);
    a.queries = m.queries;
    a.query_lens = m.query_lens;
    a.page_start = m.page_start;
    a.doc_lens = m.doc_lens;
    a.pages = m.pages;
    a.cand_ids = m.cand_ids;
    a.cand_counts = m.cand_counts;
    a.scores = m.scores;
    a.parts = static_cast<float*>(m.workspace);
    a.num_docs = m.num_docs;
    a.num_page_entries = m.num_page_entries;
    a.nq = m.nq;
    a.query_len = m.query_len;
    a.cap = m.cand_cap;
    a.split_tokens = s.tokens;
    a.splits = s.count;
    // without pages every token is absent, and no slot may be read
    a.max_tokens = c.num_pages > 0 && m.num_page_entries > 0 ? m.max_doc_tokens : 0;
    const int64_t parts = static_cast<int64_t>(m.cand_cap) * s.count;
    a.items = items_of(m.nq * parts);
    const dim3 grid(static_cast<unsigned>(ceil_div(parts, 4 * a.items)), static_cast<unsigned>(m.nq));
    hipError_t e = by_format(c.format, m.type, [&](auto f, auto t) {
        using T = decltype(t);
        constexpr int kFormat = decltype(f)::value;
        auto* kernel = a.c.row_scales == 1   ? cache_maxsim_kernel<T, kFormat, 4>
                       : a.c.group_log2 == 6 ? cache_maxsim_kernel<T, kFormat, 2>
                                             : cache_maxsim_kernel<T, kFormat, 1>;
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a);
    });
    if (e != hipSuccess) return e;
    if (s.count > 1) hipLaunchKernelGGL(cache_maxsim_join_kernel, dim3(static_cast<unsigned>(m.cand_cap), static_cast<unsigned>(m.nq)),
                       dim3(512), 0, st, a);
    if (m.k > 0) {
        // at least one key per thread of the block's merge sort
        int sort_cap = 1024;
        while (sort_cap < m.cand_cap) sort_cap *= 2;
        hipLaunchKernelGGL(cache_topk_kernel, dim3(static_cast<unsigned>(m.nq)), dim3(1024), static_cast<size_t>(sort_cap) * 8,
                           st, m.scores, m.cand_ids, m.cand_counts, m.cand_cap, sort_cap, m.k, m.top_ids, m.top_scores,
                           m.top_counts);
    }
    return hipGetLastError();
}

}  // namespace chimera
