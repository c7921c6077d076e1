/*
 * lily_layers.h -- C ABI of what stands in front of the head: the norm of the last
 * layer's output and the matrix product of draft heads and unquantised heads, for engines
 * that call this library from the last layer's output on. (The reference has its own among its
 * model's kernels, src/kernels.)
 *
 * The conventions are those of lily_sampler.h: calls enqueue on `stream` and return,
 * the caller owns every buffer, negative = refused on the host before anything was
 * enqueued, no CPU fallback. Any handle of the device serves (its fault latch, error
 * text, status word and wait limit; nothing else of it is used), and calls that overlap on
 * the GPU share nothing. What they run is loaded when the device's first handle is made: a first call may
 * be captured, and none allocates. All pointers are device pointers.
 */
#ifndef LILY_LAYERS_H
#define LILY_LAYERS_H

#include "lily_sampler.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LILY_NORM_MAX_HIDDEN 32768u

/*
 * The residual's addition and the root-mean-square norm, a token at a time:
 *
 *   h = x + residual                       (residual NULL: h = x)
 *   y = h * (weight_offset + weight) * (1 / sqrt(mean(h^2) + eps))
 *
 * h, its sum of squares, both products (in this order) and y are binary32; `residual_out` gets h rounded to `dtype`, the
 * norm is taken of h as it is before that rounding. `out` is y rounded to F32 or BF16, or with
 * out_dtype LILY_E4M3 codes with one scale per token, y ~ code * scale:
 *
 *   m = max(|y|, 2^-64) over the token,  scale = m / 448,  code = e4m3(y * (448 / m)),
 *
 * of the same binary32 y that an F32 out gets (rows that lie alike), a rounding a step.
 *
 * A NaN or an infinity makes its token's values what the formulas make of them, and no other's.
 *
 * Any hidden size up to LILY_NORM_MAX_HIDDEN and any row pitch >= hidden; rows that all start on
 * 16-byte boundaries (weight too) are read and written 16 bytes at a time. `out` and
 * `residual_out` may each be x or residual themselves (the same address, pitch and type);
 * else no two buffers overlap.
 */
typedef struct lily_norm_args {
    uint32_t struct_size;    /* sizeof(lily_norm_args_t) */
    uint32_t tokens;
    uint32_t hidden;
    uint32_t dtype;          /* of x, residual, residual_out: LILY_F32 or LILY_BF16 */
    const void *x;           /* [tokens, x_ld] */
    uint64_t x_ld;           /* elements between rows, here and below */
    const void *residual;    /* [tokens, residual_ld] or NULL */
    uint64_t residual_ld;
    void *residual_out;      /* [tokens, residual_out_ld] or NULL */
    uint64_t residual_out_ld;
    const void *weight;      /* [hidden] */
    uint32_t weight_dtype;   /* LILY_F32 or LILY_BF16 */
    uint32_t out_dtype;      /* LILY_F32, LILY_BF16 or LILY_E4M3 */
    void *out;               /* [tokens, out_ld] */
    uint64_t out_ld;
    float *out_scales;       /* [tokens], with LILY_E4M3 and only then */
    float eps;               /* >= 0 */
    float weight_offset;     /* 0, or 1 for weights stored as their distance from 1 */
} lily_norm_args_t;

int32_t lily_add_rms_norm(lily_sampler_t *h, void *stream, const lily_norm_args_t *args);

enum lily_activation {
    LILY_ACT_NONE = 0,
    LILY_ACT_RELU = 1,
    LILY_ACT_SILU = 2,      /* v / (1 + exp(-v)) */
    LILY_ACT_GELU = 3,      /* v * (1 + erf(v / sqrt(2))) / 2 */
    LILY_ACT_GELU_TANH = 4  /* v * (1 + tanh(sqrt(2 / pi) * (v + 0.044715 v^3))) / 2 */
};

/*
 * A matrix product with everything that follows it in its epilogue:
 *
 *   out[t, n] = act(a_scales[t] * weight_scales[n] * sum_k a[t, k] * weight[n, k] + bias[n])
 *               + residual[t, n]
 *
 * a and weight are both BF16 (no scales) or both E4M3 (both scales set: one per token, as
 * lily_add_rms_norm writes them, and one per output). Products are summed on the tensor cores in
 * binary32, the epilogue is binary32, and `out` is rounded once.
 *
 * Any numbers of tokens, outputs and columns, up to 2^30 each. The rows of a and weight start on 16-byte
 * boundaries (their pitches multiples of 16 bytes); out, bias and residual need no alignment
 * beyond their elements'. `residual` may be `out` itself (the same address and pitch); else out
 * overlaps no other buffer. A call gives the same bits every time, and a token's do not depend
 * on the tokens beside it; up to 64 tokens they do not depend on their number either as long as
 * that stays within 1..16, ..32 or ..64. (The columns are added up in shares whose number is
 * chosen by the sizes.)
 */
typedef struct lily_linear_args {
    uint32_t struct_size;    /* sizeof(lily_linear_args_t) */
    uint32_t tokens;
    uint32_t columns;        /* k */
    uint32_t outputs;        /* n */
    uint32_t dtype;          /* of a and weight: LILY_BF16 or LILY_E4M3 */
    uint32_t out_dtype;      /* of out and residual: LILY_F32 or LILY_BF16 */
    const void *a;           /* [tokens, a_ld] */
    uint64_t a_ld;
    const void *weight;      /* [outputs, weight_ld] */
    uint64_t weight_ld;
    const float *a_scales;      /* [tokens] or NULL */
    const float *weight_scales; /* [outputs] or NULL */
    const void *bias;        /* [outputs] of bias_dtype, or NULL */
    uint32_t bias_dtype;     /* LILY_F32 or LILY_BF16 */
    uint32_t activation;     /* enum lily_activation */
    const void *residual;    /* [tokens, residual_ld] or NULL */
    uint64_t residual_ld;
    void *out;               /* [tokens, out_ld] */
    uint64_t out_ld;
} lily_linear_args_t;

int32_t lily_linear(lily_sampler_t *h, void *stream, const lily_linear_args_t *args);

#ifdef __cplusplus
}
#endif
#endif /* LILY_LAYERS_H */
