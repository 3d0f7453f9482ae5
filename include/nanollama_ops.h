/*
 * nanollama_ops.h -- C ABI of libnanollama_stack.so, third part: operators on device memory.  A feed-forward of experts in three calls:
 *
 *   nl_op_route           scores of every expert -> the experts of every token and their weights
 *   nl_op_experts         y = sum over a token's experts of weight * down(act(gate x) * up x), the tokens grouped by expert
 *   nl_op_residual_norm   what closes a block: norm behind it, gate, residual scale, norm in front of the next
 *
 * Layer-stack models call the same kernels for layers that nl_stack_experts (below) has given experts.
 *
 * Conventions.  Pointers are device memory of `device` that the caller owns, unless a comment says otherwise; nothing is kept behind a
 * return, and no call allocates, synchronises or copies to the host: work is queued on `stream` (a hipStream_t of `device`; NULL,
 * hipStreamLegacy, hipStreamPerThread: its default streams), and a call may be captured into a graph.  The caller's current device is as
 * it was behind every call.  Arrays are row-major and on a boundary of their elements; ld* are elements from a row to the next.  n == 0
 * queues nothing.  Calls on different threads and streams do not disturb each other as long as their outputs and workspaces do not
 * overlap.  0 or a negative nl_status; nl_last_error(NULL) has this thread's message.
 * Element type `dtype`: NL_DTYPE_BF16 or NL_DTYPE_F32 (nanollama_stack.h); sums, scores, weights and norms are 32-bit either way.
 */
#ifndef NANOLLAMA_OPS_H
#define NANOLLAMA_OPS_H

#include "nanollama_stack.h"

#ifdef __cplusplus
extern "C" {
#endif

#define NL_MAX_EXPERTS 1024
#define NL_MAX_PER_TOKEN 32

enum { NL_SCORE_SOFTMAX = 0, NL_SCORE_SIGMOID = 1 };

/* Which experts a token goes to.  An expert whose logit (or logit's place in `bias`) is -infinity or NaN is out.  Score s of the others:
 *   NL_SCORE_SOFTMAX   exp(l) / sum of exp(l) over the row          chosen by l
 *   NL_SCORE_SIGMOID   1 / (1 + exp(-l))                            chosen by l, or by s + bias
 * The per_token largest, largest first, equal ones by lower number.  weight = scale * s, or scale * s / (sum of the chosen s) with renorm.
 * Of logits of +infinity every one counts the same and the others nothing (softmax).  Places for which no expert is left get id -1 and
 * weight 0. */
typedef struct {
    int32_t experts, per_token;   /* per_token <= min(experts, NL_MAX_PER_TOKEN) */
    int32_t score;                /* NL_SCORE_* */
    int32_t renorm;
    float scale;
} nl_route_desc;
/* logits [n][ld], bias [experts] or NULL (sigmoid scores only), ids and weights [n][per_token]. */
NL_API int nl_op_route(int device, void *stream, const nl_route_desc *d, int n, const float *logits, int64_t ld, const float *bias,
                       int32_t *ids, float *weights);

typedef struct {
    int32_t experts, per_token;
    int32_t dim, ff;              /* width of tokens, width of an expert */
    int32_t act;                  /* NL_ACT_* */
    int32_t dtype;                /* of x, the matrices and y */
} nl_experts_desc;
/* x [n][ldx], ids and weights [n][per_token], gate and up [experts][ff][dim], down [experts][dim][ff], y [n][ldy].  An id outside
 * [0, experts) adds nothing, whatever its weight (a row without any: y = 0); an id twice in a row counts twice.  Rows of y behind n are
 * not touched.  bfloat16: y is rounded, and the activation where more than 8 tokens come to an expert on the average or rows are
 * not on 16-byte boundaries; nothing else is.  Fast where all rows of x and the matrices start on 16-byte boundaries
 * (pointers, and dim, ff and ldx times the element's size), 1.1 to 1.7 times as long where they start on 4-byte ones, 8 to 40 times with bfloat16 rows that
 * do not.
 * workspace: at least nl_op_experts_workspace bytes, on a 16-byte boundary, this call's alone until its work is done (two graphs that may
 * run at the same time need one each).  x and y must not overlap. */
NL_API int nl_op_experts(int device, void *stream, const nl_experts_desc *d, int n, const void *x, int64_t ldx, const int32_t *ids,
                         const float *weights, const void *gate, const void *up, const void *down, void *y, int64_t ldy, void *workspace,
                         uint64_t workspace_bytes);
/* bytes for calls of up to n tokens (host arithmetic); 0: the description is not one that nl_op_experts takes */
NL_API uint64_t nl_op_experts_workspace(const nl_experts_desc *d, int n);

/* x_out = x + scale * gate * v,  v = norm(d) * post, or d without post;    h = norm(x_out) * pre  (h NULL: not asked for)
 * norm(v) = v / sqrt(mean(v^2) + eps).  x, x_out: 32-bit; d, h: dtype.  gate: 32-bit, one row for all (ldgate 0) or a row a token; NULL: 1.
 * post, pre: 32-bit gains [dim].  x_out may be x; no other overlap.
 * Time beside a copy of as many bytes: rows of up to 4096 elements, which are read once, 1.2 times where they come in fours on boundaries
 * of four elements, else 1.4 to 2.5 times; longer ones, which are read again for every step, 3.2 to 4.4 times. */
typedef struct {
    int32_t dim, dtype;
    float eps, scale;
} nl_residual_norm_desc;
NL_API int nl_op_residual_norm(int device, void *stream, const nl_residual_norm_desc *d, int n, const float *x, int64_t ldx, const void *b,
                               int64_t ldb, const float *post, const float *gate, int64_t ldgate, const float *pre, float *x_out,
                               int64_t ldxo, void *h, int64_t ldh);

/* Experts as the feed-forward of a layer of a model that nl_create_stack made, before its tensors are uploaded:
 *     h = norm2 x;   x += experts(h), the choice by ff.router h;   with post_norm x += norm2_post(experts(h))
 * The layer's nl_layer_desc has ff == 0.  Tensors: norm2 (and norm2_post) as for a feed-forward, and
 *     layers.N.ff.router                       [experts, dim],  ff.router_bias [experts] with bias (sigmoid scores only, joins the choice alone)
 *     layers.N.ff.experts.gate / up            [experts * ff, dim], expert behind expert
 *     layers.N.ff.experts.down                 [experts * dim, ff]
 * A call that fails, for want of memory too, leaves the handle as it was.
 * In bfloat16 a token's choice can differ between decode and prompt launches where two keys lie within the rounding of the router's operand. */
typedef struct {
    int32_t experts, per_token, ff, act;        /* ff: width of an expert; act: NL_ACT_* */
    int32_t score, renorm, bias;                /* as in nl_route_desc */
    float scale;
} nl_stack_experts_desc;
NL_API int nl_stack_experts(nl_handle h, int layer, const nl_stack_experts_desc *d);

#ifdef __cplusplus
}
#endif
#endif /* NANOLLAMA_OPS_H */
