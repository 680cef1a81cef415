/*
 * chimera_operators.h - the operators next to an index: dense layers that
 * turn a language model's hidden states into token embeddings (forward and
 * backward), the layer norm between them, the update that turns a weight's
 * gradient into its next value, dense layers served in microscaled 4-bit
 * floating point, a quantised cache of token embeddings in pages, for
 * documents that come and go, and late interaction (MaxSim) on that cache.
 *
 * No counterpart in the reference, which takes embeddings as they are and
 * whose index does not change. Same conventions as chimera_hip.h: a status
 * code per call, chimera_last_error() for the message, device pointers,
 * asynchronous on the context's stream (order other streams' work on the same
 * memory against it: chimera_stream, chimera_synchronize). No call allocates
 * or waits, so all of them can be captured into a HIP graph; where one needs
 * scratch memory the caller gives it. Arguments are checked on the host before
 * anything is launched; what only the device sees (slots, candidate ids,
 * pages) is checked by the kernels, which take an entry out of range for an
 * absent one.
 */
#ifndef CHIMERA_OPERATORS_H_
#define CHIMERA_OPERATORS_H_

#include <stddef.h>
#include <stdint.h>

#include "chimera_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define CHIMERA_F32 0
#define CHIMERA_F16 1
#define CHIMERA_BF16 2

/* activations; gelu by the error function, gelu_tanh by its approximation */
#define CHIMERA_ACT_NONE 0
#define CHIMERA_ACT_RELU 1
#define CHIMERA_ACT_GELU 2
#define CHIMERA_ACT_GELU_TANH 3
#define CHIMERA_ACT_SILU 4

/* ---- dense layer ----
 *
 *   Z = X W^T + b          [rows, out_features]
 *   H = act(Z) + R
 *   Y = H, or H / max(|H|, 1e-12) row by row (normalize)
 *
 * X, W, b, R and the saved Z have one type, Y has it too or is 32-bit; sums
 * are held in 32 bits and rounded once. Before that, activations are within
 * 2^-20 of 1 + |z|; CHIMERA_ACT_GELU is within 2^-18 of its own size down to
 * z = -6 where Y has 16 bits, and within 2^-20 down to -12.9 where it has 32. A
 * length beyond the 32-bit range is infinite in norms. Matrices are row-major
 * with a row stride in elements; any stride of at least the row's length and
 * any alignment of whole elements will do, rows that start at multiples of 16
 * bytes are the fast ones. Outputs and workspace overlap neither inputs nor
 * each other (columns of one wider matrix do not overlap). */
typedef struct {
    int64_t rows;         /* >= 0; rows * features at most 2^35 */
    int32_t in_features;  /* 1..65536, in_features * out_features at most 2^30 */
    int32_t out_features; /* 1..65536; at most 128 with normalize */
    int32_t type;         /* CHIMERA_F32, _F16 or _BF16 */
    int32_t out_type;     /* type or CHIMERA_F32 */
    int32_t activation;   /* CHIMERA_ACT_* */
    int32_t normalize;    /* 0 or 1 */
} chimera_linear_shape;

typedef struct {
    const void* x;        /* [rows, in_features] */
    const void* weight;   /* [out_features, in_features] */
    const void* bias;     /* [out_features] or NULL */
    const void* residual; /* [rows, out_features] or NULL */
    void* y;              /* [rows, out_features], out_type */
    void* saved;          /* Z [rows, out_features] for the backward pass, or NULL */
    float* norms;         /* max(|H|, 1e-12) [rows] for the backward pass, or NULL */
    int64_t x_stride, weight_stride, residual_stride, y_stride, saved_stride;
    void* workspace;      /* chimera_linear_workspace bytes, 256-byte aligned */
    size_t workspace_bytes;
} chimera_linear_forward;

/* Gradients from dY: with dH = dY, or (dY - Y <Y, dY>) / norm with normalize
 * (dY / norm where the norm was held at its least value), dZ = dH act'(Z):
 *   dX = dZ W, dW = dZ^T X, db = the sum of dZ's rows, dR = dH.
 * Sums over rows have a fixed order. dZ is rounded to `type`, which is what the
 * matrix cores take, and Z was when it was saved, for half the memory: of a
 * bf16 layer with GELU, 1024 features, that makes 0.0017 of the size of dX and
 * dW, 0.0016 of it dZ's (their own rounding is 0.0017). Y is read as it was
 * written, so an out_type of 32 bits keeps it whole. With rows = 0, dW and db
 * are zeros. Outputs that are NULL are not computed. */
typedef struct {
    const void* x;        /* read for dweight */
    const void* weight;   /* read for dx */
    const void* dy;       /* out_type */
    const void* saved;    /* Z as the forward pass saved it; read unless activation is NONE */
    const void* y;        /* out_type; read with normalize */
    const float* norms;   /* read with normalize */
    void* dx;             /* [rows, in_features], type, or NULL */
    void* dweight;        /* [out_features, in_features], type, or NULL */
    void* dbias;          /* [out_features], type, or NULL */
    void* dresidual;      /* [rows, out_features], type, or NULL */
    int64_t x_stride, weight_stride, dy_stride, saved_stride, y_stride;
    int64_t dx_stride, dweight_stride, dresidual_stride;
    void* workspace;      /* chimera_linear_workspace bytes, 256-byte aligned */
    size_t workspace_bytes;
} chimera_linear_backward;

/* Bytes of workspace for calls of this shape (any strides and alignment):
 * the forward pass, or with training the larger of both passes. Grows with
 * rows, so that of the largest call serves all. Most of the forward pass's is
 * for X laid out again: a call whose rows of X start and end at multiples of
 * 16 bytes, with a stride of at most 4 MiB, or one of up to four rows without
 * normalize, needs no more than for rows = 0. Host arithmetic only. */
int chimera_linear_workspace(const chimera_linear_shape* shape, int32_t training, size_t* bytes);

int chimera_linear_forward_device(chimera_ctx* ctx, const chimera_linear_shape* shape,
                                  const chimera_linear_forward* args);
int chimera_linear_backward_device(chimera_ctx* ctx, const chimera_linear_shape* shape,
                                   const chimera_linear_backward* args);

/* ---- layer norm ----
 *
 *   z = (x - mean) rstd,  rstd = 1 / sqrt(mean of (x - mean)^2 + eps)
 *   y = z w + b           [rows, features]
 *
 * x, w and b have one type, y has it too or is 32-bit; statistics and sums are
 * held in 32 bits, results rounded once. The mean is corrected by what is left
 * of a row's sum after it, in turns where that is not small beside the row's
 * deviation, and rows whose squares pass the 32-bit range are scaled, so rows of
 * any finite values are normalized, those of one value too (z is zero and rstd
 * 1 / sqrt(eps)); a row with a value that is not finite becomes NaN. Rows may
 * lie apart and have any alignment of whole elements, as for dense layers.
 * Outputs and workspace overlap neither inputs nor each other. */
typedef struct {
    int64_t rows;     /* 0..2^31 */
    int32_t features; /* 1..65536 */
    int32_t type;     /* CHIMERA_F32, _F16 or _BF16 */
    int32_t out_type; /* type or CHIMERA_F32 */
    float eps;        /* 1e-30 or more */
} chimera_norm_shape;

typedef struct {
    const void* x;      /* [rows, features] */
    const void* weight; /* [features] or NULL: ones */
    const void* bias;   /* [features] or NULL: zeros */
    void* y;            /* [rows, features], out_type */
    float* mean;        /* [rows] for the backward pass, or NULL */
    float* rstd;        /* likewise */
    int64_t x_stride, y_stride;
} chimera_norm_forward;

/* Gradients from dY, with g = dY w:
 *   dx = rstd (g - mean of g - z mean of g z),
 *   dw = the sum over rows of dY z,  db = the sum over rows of dY,
 * in a fixed order. With rows = 0, dw and db are zeros. Outputs that are NULL
 * are not computed. */
typedef struct {
    const void* x;
    const void* weight; /* as in the forward pass */
    const void* dy;     /* out_type */
    const float* mean;  /* as the forward pass left them */
    const float* rstd;
    void* dx;           /* [rows, features], type, or NULL */
    void* dweight;      /* [features], type, or NULL */
    void* dbias;        /* [features], type, or NULL */
    int64_t x_stride, dy_stride, dx_stride;
    void* workspace;    /* chimera_norm_workspace bytes, 256-byte aligned; read with dweight or dbias */
    size_t workspace_bytes;
} chimera_norm_backward;

/* Bytes of workspace of the backward pass; grows with rows, so that of the
 * largest call serves all. Host arithmetic only. */
int chimera_norm_workspace(const chimera_norm_shape* shape, size_t* bytes);

int chimera_norm_forward_device(chimera_ctx* ctx, const chimera_norm_shape* shape, const chimera_norm_forward* args);
int chimera_norm_backward_device(chimera_ctx* ctx, const chimera_norm_shape* shape, const chimera_norm_backward* args);

/* ---- microscaled 4-bit floating point ----
 *
 * A row of features values is codes of 4 bits and, for each 32 neighbours, a
 * scale of 8 bits that is a power of two: value = code * 2^(scale - 127), with
 * codes 0, 0.5, 1, 1.5, 2, 3, 4 and 6 (0..7, plus 8 with a minus sign), the
 * even value in the low half of a byte. Quantising takes
 *   scale - 127 = the exponent of the largest magnitude - 2, at least -127,
 *   code = value / 2^(scale - 127) to the nearest, ties to the even code, 6
 *          at the most.
 * A block with a value that is not finite has the scale 255 and reads back as
 * NaN. Rows of codes are padded with zeros to whole blocks (16 bytes each),
 * rows of scales to a multiple of 8; what the padding's scales hold does not
 * matter where they are read. */

/* Bytes of a row's codes and of its scales. Host arithmetic only. */
int chimera_mx4_row(int32_t features, int32_t* row_bytes, int32_t* scales);

/* d_codes [n, row_bytes] (16-byte aligned) and d_scales [n, scales] (8-byte
 * aligned) of rows [n, features] of `type` (row stride in elements). */
int chimera_mx4_quantise_device(chimera_ctx* ctx, const void* d_rows, int32_t type, int64_t row_stride, int64_t n,
                                int32_t features, uint8_t* d_codes, uint8_t* d_scales);

/* d_out [n, features] of `type` = the values, rounded once to the type. */
int chimera_mx4_read_device(chimera_ctx* ctx, const uint8_t* d_codes, const uint8_t* d_scales, int64_t n,
                            int32_t features, void* d_out, int32_t type, int64_t out_stride);

/* A dense layer on a weight that is held so,
 *   Y = act(Q(X) W^T + b) + R, divided row by row by its length with normalize,
 * with Q(X) the values of X's rows quantised as above. Shape, types, epilogue
 * and limits are those of the dense layer, but for CHIMERA_ACT_GELU where Y has 16
 * bits: down to z = -6 it is within 2^-17 of its size in fp16, which ends there,
 * and 2^-16 in bf16; in bf16 from there to -12.9 within 2^-12. Products are exact
 * and sums held in 32 bits. */
typedef struct {
    const void* x;           /* [rows, in_features], type */
    const uint8_t* codes;    /* [out_features, row_bytes of in_features], 16-byte aligned */
    const uint8_t* scales;   /* [out_features, scales of in_features], 8-byte aligned */
    const void* bias;        /* [out_features], type, or NULL */
    const void* residual;    /* [rows, out_features], type, or NULL */
    void* y;                 /* [rows, out_features], out_type */
    int64_t x_stride, residual_stride, y_stride;
    void* workspace;         /* chimera_mx4_linear_workspace bytes, 256-byte aligned; NULL if 0 */
    size_t workspace_bytes;
} chimera_mx4_linear;

/* Grows with rows, so that of the largest call serves all. Host arithmetic
 * only. */
int chimera_mx4_linear_workspace(const chimera_linear_shape* shape, size_t* bytes);

int chimera_mx4_linear_device(chimera_ctx* ctx, const chimera_linear_shape* shape, const chimera_mx4_linear* args);

/* ---- orthogonal update of a weight ----
 *
 *   M' = mu M + G,  U = G without M, G + mu M' with nesterov, else M'
 *   X = U / |U| (the square root of the sum of squares; zeros stay zeros), then
 *   X <- a X + (b A + c A^2) X with A = X X^T, `steps` times,
 *   W' = (1 - decay) W - rate X
 *
 * which brings U's singular values near one and keeps its directions: what the
 * products do to a singular value s is a s + b s^3 + c s^5, step by step. G has
 * the layer's type, M and W are 32-bit; a 16-bit layer reads the rounded copy.
 * Products are sums in 32 bits of values that are held to 22 bits (those of
 * less than 2^-22 to 2^-44); sums of squares are held in 64. X, A and b A + c A^2
 * become infinite from 255 on, so the coefficients should keep singular values
 * s below 15 from step to step, and b s^2 + c s^4 within 255 of zero (the values
 * 3.4445, -4.7750, 2.0315 keep s below 1.3 and that above -2.9). A U that is not
 * finite gives X that is not. */
typedef struct {
    int32_t rows, cols; /* 1..65536; rows * cols at most 2^28, the smaller at most 8192 */
    int32_t type;       /* of the gradient and the rounded copy */
    int32_t out_type;   /* type or CHIMERA_F32 */
    int32_t steps;      /* 1..100 */
    float a, b, c;
} chimera_orthogonal_shape;

typedef struct {
    const void* gradient;  /* [rows, cols], type */
    const float* momentum; /* [rows, cols] or NULL */
    float* new_momentum;   /* [rows, cols], with momentum; may be momentum */
    float mu;
    int32_t nesterov;      /* 0 or 1 */
    void* out;             /* X [rows, cols], out_type, or NULL */
    const float* weight;   /* [rows, cols] or NULL */
    float* new_weight;     /* [rows, cols], with weight; may be weight */
    void* rounded;         /* W' [rows, cols], type, or NULL */
    float rate, decay;
    int64_t gradient_stride, momentum_stride, new_momentum_stride, out_stride;
    int64_t weight_stride, new_weight_stride, rounded_stride;
    void* workspace;       /* chimera_orthogonal_workspace bytes, 256-byte aligned */
    size_t workspace_bytes;
} chimera_orthogonal_update;

/* Host arithmetic only. */
int chimera_orthogonal_workspace(const chimera_orthogonal_shape* shape, size_t* bytes);

/* Outputs and workspace overlap neither inputs nor each other, but for
 * new_momentum = momentum and new_weight = weight with the same stride. */
int chimera_orthogonal_update_device(chimera_ctx* ctx, const chimera_orthogonal_shape* shape,
                                     const chimera_orthogonal_update* args);

/* ---- quantised token cache ----
 *
 * num_pages pages of page_tokens slots; a slot holds one token's embedding of
 * dim values as codes of 8 or 4 bits and one 32-bit scale for every `group`
 * values: value = code * scale. A row of codes is padded with zeros to a
 * multiple of 32 values: slot s has its codes at s * row_bytes with
 * row_bytes = ceil(dim / 32) * 32 * bits / 8, and its scales at
 * s * ceil(dim / group). Writing a row x takes, group by group,
 *   scale = max|x| * (1 / top),  code = round(x * (top * (1 / max|x|)))
 * in 32-bit arithmetic, ties to even, with top = 127 (INT8, two's
 * complement), 7 (INT4, stored plus 8, the even value in the low half of a
 * byte) or 448 (FP8, e4m3). A group whose largest magnitude is below 2^-117
 * is stored as zeros, with scale 0; a group with a value that is not finite
 * has the scale NaN and reads back as NaN. */
#define CHIMERA_CACHE_INT8 0
#define CHIMERA_CACHE_INT4 1
#define CHIMERA_CACHE_FP8 2

typedef struct {
    int32_t format;      /* CHIMERA_CACHE_* */
    int32_t dim;         /* 1..128 */
    int32_t group;       /* 32, 64 or 128 values per scale */
    int32_t page_tokens; /* a power of two, 1..4096 */
    int64_t num_pages;
    uint8_t* codes;      /* [num_pages * page_tokens][row_bytes], 16-byte aligned */
    float* scales;       /* [num_pages * page_tokens][ceil(dim / group)], 16-byte aligned */
} chimera_cache;

/* Bytes of a slot's codes and its number of scales. Host arithmetic only. */
int chimera_cache_row(const chimera_cache* cache, int32_t* row_bytes, int32_t* scales);

/* Quantises rows [n, dim] of `type` (row stride in elements) into slots
 * d_slots [n]; a slot outside the cache is skipped. Slots of one call must
 * differ from each other. */
int chimera_cache_write_device(chimera_ctx* ctx, const chimera_cache* cache, const void* d_rows, int32_t type,
                               int64_t row_stride, const int64_t* d_slots, int64_t n);

/* d_out [n, dim] of `type` = the values of slots d_slots [n], rounded once
 * to the type; zeros for a slot outside the cache. */
int chimera_cache_read_device(chimera_ctx* ctx, const chimera_cache* cache, const int64_t* d_slots, int64_t n,
                              void* d_out, int32_t type, int64_t out_stride);

/* Late interaction of nq queries with candidate documents in the cache:
 * d_scores[q * cand_cap + j] = sum over the tokens i of query q of the max
 * over the tokens t of document d_cand_ids[q * cand_cap + j] of <q_i, x_t>.
 * Token t of document d is in slot t % page_tokens of page
 * d_pages[d_page_start[d] + t / page_tokens], t < d_doc_lens[d]. A document
 * without tokens, an id outside [0, num_docs) and j >= d_cand_counts[q] score
 * -inf, in the last case without the candidate's being read; tokens on pages
 * outside the cache or the page list are absent, and so are tokens past
 * max_doc_tokens, which should be at least the longest candidate's length
 * (it decides how documents are split over the GPU). A product that is NaN
 * (a cached row that was not finite) is passed over; with a query token that
 * is not finite a query's scores mean nothing. A query without tokens scores
 * 0 where the document has some. d_query_lens [nq] is the number of
 * tokens of each query (the rest of its query_len rows are not read), NULL
 * for query_len each. Queries of 32-bit type are split into two fp16 parts
 * (22 bits), 16-bit ones are used as they are, in fp16 with a power of two
 * per token: within 2^-20 |q_i||x_t| per product.
 *
 * With k > 0, top_ids / top_scores [nq, k] get the k best candidates by
 * score descending, ties to the larger id (those that are no documents last,
 * with their -inf), padded with -1 / 0, and top_counts [nq] their number;
 * cand_cap is then at most 8192. */
typedef struct {
    const void* queries;          /* [nq, query_len, dim], contiguous */
    int32_t type;                 /* of queries */
    int32_t nq;                   /* 0..65535 */
    int32_t query_len;            /* 1..1024 */
    const int32_t* query_lens;    /* [nq] or NULL */
    const int64_t* page_start;    /* [num_docs] */
    const int32_t* doc_lens;      /* [num_docs] */
    const int32_t* pages;         /* [num_page_entries] */
    int64_t num_docs, num_page_entries;
    int32_t max_doc_tokens;       /* 0..2^30 */
    const int32_t* cand_ids;      /* [nq, cand_cap] */
    const int32_t* cand_counts;   /* [nq] or NULL: cand_cap each */
    int32_t cand_cap;             /* 1..2^24 */
    float* scores;                /* [nq, cand_cap] */
    int32_t k;                    /* 0: no top-k */
    int64_t* top_ids;
    float* top_scores;            /* or NULL */
    int32_t* top_counts;
    void* workspace;              /* chimera_cache_maxsim_workspace bytes, 256-byte aligned; NULL if 0 */
    size_t workspace_bytes;
} chimera_cache_maxsim;

/* Bytes of workspace of a call with these nq, query_len, cand_cap and
 * max_doc_tokens. Host arithmetic only. */
int chimera_cache_maxsim_workspace(const chimera_cache_maxsim* args, size_t* bytes);

int chimera_cache_maxsim_device(chimera_ctx* ctx, const chimera_cache* cache, const chimera_cache_maxsim* args);

#ifdef __cplusplus
}
#endif

#endif /* CHIMERA_OPERATORS_H_ */
