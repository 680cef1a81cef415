// C ABI of the operators beside the index (include/chimera_operators.h): the
// checks of their arguments, then the launches.
#include "operators.hpp"

#include <string>

#include "capi_internal.hpp"

using namespace chimera;

namespace {

int invalid(const std::string& msg) { return api_fail(CHIMERA_ERR_INVALID_ARGUMENT, msg); }

int launched(hipError_t e, const char* what) {
    if (e == hipSuccess) return CHIMERA_OK;
    return api_fail(CHIMERA_ERR_HIP, std::string(what) + " failed: " + hipGetErrorString(e));
}

bool known_type(int type) { return type == CHIMERA_F32 || type == CHIMERA_F16 || type == CHIMERA_BF16; }

constexpr int kMostFeatures = 65536;
constexpr int kMostNormalized = 128;
// tiles of 128 x 128 that one launch may have (blocks of 32 rows stay within
// 2^32 threads), and values of a weight
constexpr int64_t kMostTiles = int64_t{1} << 21;
constexpr int64_t kMostWeights = int64_t{1} << 30;
constexpr int kMostCandidates = 8192;  // the top-k sorts a query's candidates in LDS

int check_shape(const chimera_linear_shape* s) {
    if (!s) return invalid("null shape");
    if (s->rows < 0) return invalid("negative row count");
    if (s->in_features < 1 || s->in_features > kMostFeatures || s->out_features < 1 || s->out_features > kMostFeatures)
        return invalid("features must be in [1, 65536]");
    if (!known_type(s->type)) return invalid("unknown element type");
    if (s->out_type != s->type && s->out_type != CHIMERA_F32) return invalid("the output has the layer's type or 32 bits");
    if (s->activation < CHIMERA_ACT_NONE || s->activation > CHIMERA_ACT_SILU) return invalid("unknown activation");
    if (s->normalize != 0 && s->normalize != 1) return invalid("normalize must be 0 or 1");
    if (s->normalize && s->out_features > kMostNormalized) return invalid("normalized rows have at most 128 features");
    const int64_t widest = s->in_features > s->out_features ? s->in_features : s->out_features;
    if (s->rows > (int64_t{1} << 31) || (s->rows + 127) / 128 * ((widest + 127) / 128) > kMostTiles)
        return invalid("too many rows for one call: rows * features / 16384 must not pass 2^21");
    if (static_cast<int64_t>(s->in_features) * s->out_features > kMostWeights)
        return invalid("a weight has at most 2^30 values");
    return CHIMERA_OK;
}

// A matrix argument: aligned to its elements, rows that do not overlap and
// whose offsets fit 62 bits.
int check_matrix(const char* name, const void* p, int64_t rows, int64_t cols, int64_t stride, size_t elem) {
    if (!p) return invalid(std::string("null argument: ") + name);
    if (reinterpret_cast<uintptr_t>(p) % elem) return invalid(std::string(name) + " is not aligned to its elements");
    if (stride < cols) return invalid(std::string("the row stride of ") + name + " is less than a row");
    if (stride > (int64_t{1} << 62) / (rows * static_cast<int64_t>(elem)))
        return invalid(std::string("the row stride of ") + name + " is too large");
    return CHIMERA_OK;
}
int check_vector(const char* name, const void* p, size_t elem) { return check_matrix(name, p, 1, 0, 0, elem); }

// What a call reads or writes, for the check that outputs lie apart.
struct Region {
    const char* name;
    const void* p;
    int64_t rows, row_bytes, stride_bytes;
};
Region region(const char* name, const void* p, int64_t rows, int64_t cols, int64_t stride, size_t elem) {
    return Region{name, p, rows, cols * static_cast<int64_t>(elem), stride * static_cast<int64_t>(elem)};
}
// Whether two matrices share a byte. Rows of the same stride may interleave
// (columns of one wider matrix); otherwise the ranges have to be apart.
bool overlap(const Region& a, const Region& b) {
    if (!a.p || !b.p || a.rows == 0 || b.rows == 0) return false;
    const char *pa = static_cast<const char*>(a.p), *pb = static_cast<const char*>(b.p);
    const char *ea = pa + (a.rows - 1) * a.stride_bytes + a.row_bytes, *eb = pb + (b.rows - 1) * b.stride_bytes + b.row_bytes;
    if (ea <= pb || eb <= pa) return false;
    if (a.stride_bytes != b.stride_bytes || a.stride_bytes == 0) return true;
    const int64_t apart = ((pb - pa) % a.stride_bytes + a.stride_bytes) % a.stride_bytes;
    return apart < a.row_bytes || apart + b.row_bytes > a.stride_bytes;
}
template <size_t kOut, size_t kIn>
int check_apart(const Region (&outs)[kOut], const Region (&ins)[kIn]) {
    for (size_t i = 0; i < kOut; ++i) {
        for (const Region& in : ins)
            if (overlap(outs[i], in)) return invalid(std::string(outs[i].name) + " overlaps " + in.name);
        for (size_t j = i + 1; j < kOut; ++j)
            if (overlap(outs[i], outs[j])) return invalid(std::string(outs[i].name) + " overlaps " + outs[j].name);
    }
    return CHIMERA_OK;
}

int check_workspace(const void* p, size_t have, size_t need) {
    if (need == 0) return CHIMERA_OK;
    if (!p || have < need)
        return api_fail(CHIMERA_ERR_CAPACITY, "the workspace has " + std::to_string(p ? have : 0) + " bytes, " +
                                                  std::to_string(need) + " are needed");
    if (reinterpret_cast<uintptr_t>(p) % 256) return invalid("the workspace is not aligned to 256 bytes");
    return CHIMERA_OK;
}

#define CK(expr)                         \
    do {                                 \
        const int r_ = (expr);           \
        if (r_ != CHIMERA_OK) return r_; \
    } while (0)

int check_cache(const chimera_cache* c) {
    if (!c) return invalid("null cache");
    if (c->format < CHIMERA_CACHE_INT8 || c->format > CHIMERA_CACHE_FP8) return invalid("unknown cache format");
    if (c->dim < 1 || c->dim > kDim) return invalid("the cache's dim must be in [1, 128]");
    if (c->group != 32 && c->group != 64 && c->group != 128) return invalid("the cache's group must be 32, 64 or 128");
    if (c->page_tokens < 1 || c->page_tokens > 4096 || (c->page_tokens & (c->page_tokens - 1)))
        return invalid("tokens per page must be a power of two in [1, 4096]");
    if (c->num_pages < 0 || c->num_pages > INT32_MAX) return invalid("the number of pages must be in [0, 2^31)");
    return CHIMERA_OK;
}
int check_cache_memory(const chimera_cache* c) {
    if (c->num_pages == 0) return CHIMERA_OK;
    if (!c->codes || !c->scales) return invalid("null cache memory");
    if (reinterpret_cast<uintptr_t>(c->codes) % 16 || reinterpret_cast<uintptr_t>(c->scales) % 16)
        return invalid("the cache's memory is not aligned to 16 bytes");
    return CHIMERA_OK;
}
constexpr int64_t kMostRows = int64_t{1} << 28;  // 16 rows a block of 256 threads

int check_rows(int64_t n) {
    if (n < 0) return invalid("negative row count");
    if (n > kMostRows - 16) return invalid("at most 2^28 - 16 rows per call");
    return CHIMERA_OK;
}

int check_maxsim_sizes(const chimera_cache_maxsim* m) {
    if (!m) return invalid("null argument");
    if (m->nq < 0 || m->nq > 65535) return invalid("the number of queries must be in [0, 65535]");
    if (m->query_len < 1 || m->query_len > 1024) return invalid("the query length must be in [1, 1024]");
    if (m->cand_cap < 1 || m->cand_cap > (1 << 24)) return invalid("candidate capacity must be in [1, 2^24]");
    if (m->max_doc_tokens < 0 || m->max_doc_tokens > (1 << 30)) return invalid("the longest document must have 0 to 2^30 tokens");
    return CHIMERA_OK;
}

}  // namespace

extern "C" {

int chimera_linear_workspace(const chimera_linear_shape* shape, int32_t training, size_t* bytes) {
    CK(check_shape(shape));
    if (!bytes) return invalid("null argument");
    const size_t f = linear_forward_workspace(*shape), b = training ? linear_backward_workspace(*shape) : 0;
    *bytes = f > b ? f : b;
    return CHIMERA_OK;
}

int chimera_linear_forward_device(chimera_ctx* ctx, const chimera_linear_shape* shape,
                                  const chimera_linear_forward* args) {
    hipStream_t st;
    CK(api_enter(ctx, &st));
    CK(check_shape(shape));
    if (!args) return invalid("null argument");
    if (shape->rows == 0) return CHIMERA_OK;
    const size_t e = type_bytes(shape->type), out = type_bytes(shape->out_type);
    CK(check_matrix("x", args->x, shape->rows, shape->in_features, args->x_stride, e));
    CK(check_matrix("weight", args->weight, shape->out_features, shape->in_features, args->weight_stride, e));
    CK(check_matrix("y", args->y, shape->rows, shape->out_features, args->y_stride, out));
    if (args->bias) CK(check_vector("bias", args->bias, e));
    if (args->residual) CK(check_matrix("residual", args->residual, shape->rows, shape->out_features, args->residual_stride, e));
    if (args->saved) CK(check_matrix("saved", args->saved, shape->rows, shape->out_features, args->saved_stride, e));
    if (args->norms) CK(check_vector("norms", args->norms, 4));
    if (args->norms && !shape->normalize) return invalid("norms are an output of normalized layers");
    const size_t need = linear_forward_workspace(LinearForward{*shape, *args});
    CK(check_workspace(args->workspace, args->workspace_bytes, need));
    const int64_t m = shape->rows, k = shape->in_features, n = shape->out_features, bytes = static_cast<int64_t>(need);
    const Region outs[] = {region("y", args->y, m, n, args->y_stride, out),
                           region("saved", args->saved, m, n, args->saved_stride, e),
                           region("norms", args->norms, 1, m, m, 4),
                           region("the workspace", args->workspace, 1, bytes, bytes, 1)};
    const Region ins[] = {region("x", args->x, m, k, args->x_stride, e),
                          region("weight", args->weight, n, k, args->weight_stride, e),
                          region("bias", args->bias, 1, n, n, e),
                          region("residual", args->residual, m, n, args->residual_stride, e)};
    CK(check_apart(outs, ins));
    return launched(launch_linear_forward(st, LinearForward{*shape, *args}), "linear forward kernels");
}

int chimera_linear_backward_device(chimera_ctx* ctx, const chimera_linear_shape* shape,
                                   const chimera_linear_backward* args) {
    hipStream_t st;
    CK(api_enter(ctx, &st));
    CK(check_shape(shape));
    if (!args) return invalid("null argument");
    const size_t e = type_bytes(shape->type), out = type_bytes(shape->out_type);
    if (args->dweight) CK(check_matrix("dweight", args->dweight, shape->out_features, shape->in_features, args->dweight_stride, e));
    if (args->dbias) CK(check_vector("dbias", args->dbias, e));
    if (shape->rows > 0) {
        CK(check_matrix("dy", args->dy, shape->rows, shape->out_features, args->dy_stride, out));
        if (args->dweight) CK(check_matrix("x", args->x, shape->rows, shape->in_features, args->x_stride, e));
        if (args->dx) {
            CK(check_matrix("weight", args->weight, shape->out_features, shape->in_features, args->weight_stride, e));
            CK(check_matrix("dx", args->dx, shape->rows, shape->in_features, args->dx_stride, e));
        }
        if (shape->activation != CHIMERA_ACT_NONE)
            CK(check_matrix("saved", args->saved, shape->rows, shape->out_features, args->saved_stride, e));
        if (shape->normalize) {
            CK(check_matrix("y", args->y, shape->rows, shape->out_features, args->y_stride, out));
            CK(check_vector("norms", args->norms, 4));
        }
        if (args->dresidual)
            CK(check_matrix("dresidual", args->dresidual, shape->rows, shape->out_features, args->dresidual_stride, e));
        const size_t need = linear_backward_workspace(*shape);
        CK(check_workspace(args->workspace, args->workspace_bytes, need));
        const int64_t m = shape->rows, k = shape->in_features, n = shape->out_features, bytes = static_cast<int64_t>(need);
        const bool act = shape->activation != CHIMERA_ACT_NONE, norm = shape->normalize != 0;
        const Region outs[] = {region("dx", args->dx, m, k, args->dx_stride, e),
                               region("dweight", args->dweight, n, k, args->dweight_stride, e),
                               region("dbias", args->dbias, 1, n, n, e),
                               region("dresidual", args->dresidual, m, n, args->dresidual_stride, e),
                               region("the workspace", args->workspace, 1, bytes, bytes, 1)};
        const Region ins[] = {region("x", args->dweight ? args->x : nullptr, m, k, args->x_stride, e),
                              region("weight", args->dx ? args->weight : nullptr, n, k, args->weight_stride, e),
                              region("dy", args->dy, m, n, args->dy_stride, out),
                              region("saved", act ? args->saved : nullptr, m, n, args->saved_stride, e),
                              region("y", norm ? args->y : nullptr, m, n, args->y_stride, out),
                              region("norms", norm ? args->norms : nullptr, 1, m, m, 4)};
        CK(check_apart(outs, ins));
    }
    return launched(launch_linear_backward(st, LinearBackward{*shape, *args}), "linear backward kernels");
}

int chimera_cache_row(const chimera_cache* cache, int32_t* row_bytes, int32_t* scales) {
    CK(check_cache(cache));
    if (!row_bytes || !scales) return invalid("null argument");
    *row_bytes = cache_row_bytes(*cache);
    *scales = cache_row_scales(*cache);
    return CHIMERA_OK;
}

int chimera_cache_write_device(chimera_ctx* ctx, const chimera_cache* cache, const void* d_rows, int32_t type,
                               int64_t row_stride, const int64_t* d_slots, int64_t n) {
    hipStream_t st;
    CK(api_enter(ctx, &st));
    CK(check_cache(cache));
    CK(check_cache_memory(cache));
    CK(check_rows(n));
    if (!known_type(type)) return invalid("unknown element type");
    if (n == 0) return CHIMERA_OK;
    CK(check_matrix("rows", d_rows, n, cache->dim, row_stride, type_bytes(type)));
    CK(check_vector("slots", d_slots, 8));
    return launched(launch_cache_write(st, *cache, d_rows, type, row_stride, d_slots, n), "cache write kernel");
}

int chimera_cache_read_device(chimera_ctx* ctx, const chimera_cache* cache, const int64_t* d_slots, int64_t n,
                              void* d_out, int32_t type, int64_t out_stride) {
    hipStream_t st;
    CK(api_enter(ctx, &st));
    CK(check_cache(cache));
    CK(check_cache_memory(cache));
    CK(check_rows(n));
    if (!known_type(type)) return invalid("unknown element type");
    if (n == 0) return CHIMERA_OK;
    CK(check_matrix("out", d_out, n, cache->dim, out_stride, type_bytes(type)));
    CK(check_vector("slots", d_slots, 8));
    return launched(launch_cache_read(st, *cache, d_slots, n, d_out, type, out_stride), "cache read kernel");
}

int chimera_cache_maxsim_workspace(const chimera_cache_maxsim* args, size_t* bytes) {
    CK(check_maxsim_sizes(args));
    if (!bytes) return invalid("null argument");
    *bytes = cache_maxsim_workspace(*args);
    return CHIMERA_OK;
}

int chimera_cache_maxsim_device(chimera_ctx* ctx, const chimera_cache* cache, const chimera_cache_maxsim* m) {
    hipStream_t st;
    CK(api_enter(ctx, &st));
    CK(check_cache(cache));
    CK(check_cache_memory(cache));
    CK(check_maxsim_sizes(m));
    if (!known_type(m->type)) return invalid("unknown element type");
    if (m->num_docs < 0 || m->num_page_entries < 0 || m->k < 0) return invalid("negative size");
    if (m->k > 0 && m->cand_cap > kMostCandidates) return invalid("a top-k takes at most 8192 candidates");
    if (m->nq == 0) return CHIMERA_OK;
    CK(check_vector("queries", m->queries, type_bytes(m->type)));
    CK(check_vector("cand_ids", m->cand_ids, 4));
    CK(check_vector("scores", m->scores, 4));
    if (m->num_docs > 0) {
        CK(check_vector("page_start", m->page_start, 8));
        CK(check_vector("doc_lens", m->doc_lens, 4));
    }
    if (m->num_page_entries > 0) CK(check_vector("pages", m->pages, 4));
    if (m->k > 0 && (!m->top_ids || !m->top_counts)) return invalid("null top-k argument");
    CK(check_workspace(m->workspace, m->workspace_bytes, cache_maxsim_workspace(*m)));
    return launched(launch_cache_maxsim(st, *cache, *m), "cache MaxSim kernels");
}

}  // extern "C"
