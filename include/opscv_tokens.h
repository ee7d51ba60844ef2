/*
 * Operators on token sequences -- two-phase C API, MI355X (gfx950) implementation.  No counterpart in the reference:
 * what a transformer block over the tokens of a picture, or a language model that reads such tokens, needs around its
 * matrix products.  They follow the conventions of the aclnn entry points beside them: the first phase
 * (...GetWorkspaceSize) is host-only, validates, plans and hands out the executor; the second enqueues kernels on
 * `stream` (a hipStream_t), allocates nothing, never synchronises, may be recorded into a HIP graph and always frees
 * the executor.
 *
 *   dtypes  : FLOAT, FLOAT16, BF16; the operands of one call have one type unless stated otherwise.  Sums, softmax
 *             statistics and norms are held in 32 bits.  The matrix products of attention take operands of the tensors'
 *             type: its weights, and in the gradients weights and gradients of the scores, are rounded to it (to nearest,
 *             a relative 2^-11 at most for FLOAT16, 2^-8 for BF16) before they are multiplied and summed up in 32 bits.
 *   formats : any (the order of the dimensions is fixed by the operator)
 *   views   : arbitrary strides and offsets are honoured.  Attention and rotary operands whose last dimension is dense
 *             are used in place whatever the strides of the others; other views are packed through the workspace.
 *             Outputs must not overlap themselves or, unless stated otherwise, an input.
 *   status  : 161001 for a NULL argument or data pointer, 161002 for anything else that does not fit.
 *   results : the same from call to call (no atomic additions; sums have a fixed order).
 */
#ifndef OPSCV_TOKENS_H_
#define OPSCV_TOKENS_H_

#include "opscv_acl_base.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Root-mean-square norm with the residual's addition:
 *   h = x + residual,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * weight
 * x, residual, y, sum : (..., width), one to five dimensions; weight : (width), of x's type or FLOAT.  h, its squares and
 * h * weight are numbers of 32 bits: their range is FLOAT's.
 *   residual : NULL: h = x
 *   y        : of x's type, or INT8.  INT8: y = round(h * weight * (127 / m)) to the nearest, ties to even, with
 *              m = max |h * weight| over the row, and `scale` (FLOAT, the leading dimensions) = m * rstd / 127, so that
 *              y * scale stands for the norm.  A row of zeros has scale 0; a row that holds an infinity or NaN has
 *              y = 0 and scale NaN.
 *   scale    : required with an INT8 y, else NULL
 *   sum      : NULL, or h rounded to x's type.  The norm is taken of h before that rounding.
 *   rstd     : NULL, or FLOAT, the leading dimensions: what the backward pass reads
 * sum may be x or residual (the same view): the addition in place.
 */
ACLNN_API aclnnStatus opscvResidualNormGetWorkspaceSize(const aclTensor* x, const aclTensor* residual,
                                                        const aclTensor* weight, double eps, aclTensor* y,
                                                        aclTensor* scale, aclTensor* sum, aclTensor* rstd,
                                                        uint64_t* workspaceSize, aclOpExecutor** executor);
ACLNN_API aclnnStatus opscvResidualNorm(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                        aclrtStream stream);

/*
 * Gradients of the norm.  n = sum * rstd, g = gradY * weight:
 *   gradX = (g - n * mean(g * n)) * rstd + gradSum,   gradWeight = sum over rows of gradY * n
 * gradX is the gradient of x and of the residual alike.
 *   sum, rstd  : what the forward pass wrote (sum = x where there was no residual)
 *   gradSum    : NULL, or the gradient that reaches `sum` on its other way
 *   gradWeight : NULL, or (width), of weight's type
 * gradX may be gradY or gradSum (the same view).
 */
ACLNN_API aclnnStatus opscvResidualNormBackwardGetWorkspaceSize(const aclTensor* gradY, const aclTensor* gradSum,
                                                                const aclTensor* sum, const aclTensor* weight,
                                                                const aclTensor* rstd, aclTensor* gradX,
                                                                aclTensor* gradWeight, uint64_t* workspaceSize,
                                                                aclOpExecutor** executor);
ACLNN_API aclnnStatus opscvResidualNormBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                                aclrtStream stream);

/* How opscvRotaryTable stretches its angles to contexts longer than a model was trained on. */
typedef enum {
    OPSCV_ROTARY_PLAIN = 0,    /* pair i turns by base^(-2i/rot) radians from one position to the next */
    OPSCV_ROTARY_LINEAR = 1,   /* every frequency divided by factor */
    OPSCV_ROTARY_BASE = 2,     /* base * factor^(rot / (rot - 2)): the lowest frequency is divided by factor, the
                                  highest kept */
    OPSCV_ROTARY_BY_PARTS = 3  /* frequencies that turn 32 times or more in originalLength positions kept, those that
                                  turn once or less divided by factor, a linear blend by turns between */
} opscvRotaryScaling;

/*
 * Table of cosines and sines: row p of `table` ((positions, rot), FLOAT, rot even) holds rot / 2 cosines and behind
 * them rot / 2 sines of the angles of position p, computed in 64 bits, times `magnitude` (1: a rotation).
 * factor >= 1; originalLength is read with OPSCV_ROTARY_BY_PARTS only; OPSCV_ROTARY_BASE needs rot > 2.
 */
ACLNN_API aclnnStatus opscvRotaryTableGetWorkspaceSize(double base, int64_t scaling, double factor,
                                                       int64_t originalLength, double magnitude, aclTensor* table,
                                                       uint64_t* workspaceSize, aclOpExecutor** executor);
ACLNN_API aclnnStatus opscvRotaryTable(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                       aclrtStream stream);

/*
 * Rotary positions: in the first rot features of every head, pair i = (a, b) of a token at position p becomes
 *   (a cos - b sin, b cos + a sin)   with cos = table[p][i], sin = table[p][rot / 2 + i]; other features are copied.
 *   query, queryOut : (batch, tokens, heads, d), d <= 1024
 *   key, keyOut     : (batch, tokens, kvHeads, d), or both NULL
 *   positions       : (batch, tokens), INT32 or INT64, or NULL: token t is at position t.  A token whose position is
 *                     not a row of the table gets NaN in its rotated features.
 *   table           : (positions, rot), FLOAT, rot even, rot <= d
 *   interleaved     : pair i is features (2i, 2i + 1); else (i, i + rot / 2)
 *   inverse         : the transposed map (sin negated): the gradient's way back
 * queryOut may be query and keyOut key (the same view): rotation in place.
 */
ACLNN_API aclnnStatus opscvRotaryGetWorkspaceSize(const aclTensor* query, const aclTensor* key,
                                                  const aclTensor* positions, const aclTensor* table, bool interleaved,
                                                  bool inverse, aclTensor* queryOut, aclTensor* keyOut,
                                                  uint64_t* workspaceSize, aclOpExecutor** executor);
ACLNN_API aclnnStatus opscvRotary(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor, aclrtStream stream);

/*
 * Attention to a window around each token and to the first tokens (sinks).
 *   query, out : (batch, tokens, heads, d);  key, value : (batch, kvTokens, kvHeads, d), kvHeads divides heads, d <= 256
 *   qLengths, kvLengths : (batch), INT32 or INT64, or NULL: all tokens.  Values are clamped to [0, tokens] and
 *       [0, kvTokens].  A sequence's queries are its last tokens: query i < qLength stands at
 *       p = kvLength - qLength + i.
 *   Query i sees key j if j < kvLength, j <= p + right, and (j >= p - left or j < sinks).
 *   out = softmax over the seen keys of (scale * query . key) applied to their values; what a key or value holds that a
 *       query does not see, or from kvLength on, is never read into its result, NaN included.  A query that
 *       sees nothing (i >= qLength among them) gives zeros.
 *   lse : NULL, or (batch, heads, tokens), FLOAT: ln of the sum of exp(scale * query . key) over the seen keys, minus
 *       infinity where nothing is seen
 *   left, right, sinks >= 0 (right = 0: causal; left = INT64_MAX: no window), scale > 0 and finite.
 * Prompts (many queries), chunks on a cache and single tokens take the same call.
 *   sizes : up to 2^28 tokens and kvTokens, 2^30 rows (tokens * heads) of a sequence, 2^31 - 1 batch * heads.  A sequence
 *       whose workgroups one launch does not hold is refused (161002): FLOAT heads of up to 64 features from 2^29
 *       rows on, and, in the gradients, kvTokens * kvHeads from 2^31 on.  Batches of any size take as many launches as they need.
 */
ACLNN_API aclnnStatus opscvWindowAttentionGetWorkspaceSize(const aclTensor* query, const aclTensor* key,
                                                           const aclTensor* value, const aclTensor* qLengths,
                                                           const aclTensor* kvLengths, double scale, int64_t left,
                                                           int64_t right, int64_t sinks, aclTensor* out, aclTensor* lse,
                                                           uint64_t* workspaceSize, aclOpExecutor** executor);
ACLNN_API aclnnStatus opscvWindowAttention(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                           aclrtStream stream);

/*
 * Gradients of the attention.  out and lse are what the forward call wrote for the same arguments; gradQuery, gradKey
 * and gradValue have the shapes of query, key and value and are written whole (zeros where nothing is seen).
 * What keys, values, queries and gradients hold past the sequences' lengths is never read into a result, nor is a key or
 * value that a query does not see into that query's gradient.  A query or its gradOut that is not finite reaches the
 * gradients of the keys that it sees, and may reach those of keys beside them.
 */
ACLNN_API aclnnStatus opscvWindowAttentionBackwardGetWorkspaceSize(
    const aclTensor* gradOut, const aclTensor* query, const aclTensor* key, const aclTensor* value,
    const aclTensor* out, const aclTensor* lse, const aclTensor* qLengths, const aclTensor* kvLengths, double scale,
    int64_t left, int64_t right, int64_t sinks, aclTensor* gradQuery, aclTensor* gradKey, aclTensor* gradValue,
    uint64_t* workspaceSize, aclOpExecutor** executor);
ACLNN_API aclnnStatus opscvWindowAttentionBackward(void* workspace, uint64_t workspaceSize, aclOpExecutor* executor,
                                                   aclrtStream stream);

#ifdef __cplusplus
}
#endif

#endif /* OPSCV_TOKENS_H_ */
