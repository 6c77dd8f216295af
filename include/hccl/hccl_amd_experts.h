/* Operators of an expert-parallel layer, next to HcclAlltoAllV, and of its training step, next to HcclAllReduce.  Nothing here exists in
 * the reference.
 *
 *   HcclAmdExpertRoute      logits -> experts, weights, per-expert counts, rows in expert order, balance loss
 *   HcclAmdExpertPack       tokens -> rows in expert order (an all-to-all-v's send buffer), copied or in 8 bits
 *   HcclAmdBlockMatmul      8-bit rows, group by group, times their experts' 8-bit weights
 *   HcclAmdExpertCombine    rows -> tokens, weighted and summed
 *   HcclAmdNormRows         rows + residual, normed by their root mean square, in their type and as 8-bit rows
 *   HcclAmdExpertRouteScored, HcclAmdExpertBias   experts by sigmoid or softmax scores, a balancing bias, in groups
 *   HcclAmdExpertGate       silu(gate) * up between two products, in the rows' type or as 8-bit rows
 *   HcclAmdGradSquares, HcclAmdGradClip   gradients of many tensors held to a norm over all of them (and all ranks)
 *   ...Grad, HcclAmdBlockMatmulGradWeight, HcclAmdBlockQuant...   their gradients and what these read
 *
 * All of them: device pointers unless said otherwise, of one GPU; no communicator; the work is queued on `stream` (a
 * hipStream_t, not null) and nothing is allocated, copied or waited for, so a call can be captured into a HIP graph.  An
 * output must not overlap an input or another output, except where a call says that the two may be the same.  Same inputs, same bits: no atomics whose order matters.  Strides are
 * in elements, from one row to the next, 2^40 at most; 0 stands for rows that follow each other without a gap.  Values in 16 bits are
 * widened, everything is summed in 32 bits, and rounded once at the end.  Indices and offsets read from device memory are
 * checked on the device: what points outside is skipped.
 * Errors: HCCL_E_PTR (a null pointer or stream), HCCL_E_PARA (a size, stride or alignment), HCCL_E_NOT_SUPPORT (a type),
 * HCCL_E_RUNTIME (the launch failed); nothing has been queued then, except that a failed launch may follow good ones.
 * No work (tokens, rows or width 0) returns HCCL_SUCCESS before the pointers of what is absent are looked at.
 *
 * 8-bit rows.  HCCL_DATA_TYPE_FP8E4M3 values (largest 448) with one scale per 128 consecutive values: value = q * scale.
 * Every row is padded with zeros to a multiple of 128 values, starts on a 16-byte boundary, and its stride is a multiple
 * of 16 below 2^23.  Of a block, a = max(largest finite magnitude, 2^-96); the scale is
 *   HCCL_AMD_SCALE_FP32   float a * (1 / 448), q = round(v * (1 / a * 448)), every quotient and product rounded to 32 bits
 *   HCCL_AMD_SCALE_E8M0   one byte b that stands for 2^(b - 127), the least power of two with a <= 448 * 2^(b - 127);
 *                         q = round(v / scale)
 * rounding to nearest, ties to even.  Infinities and NaN become the type's NaN and leave their block's scale alone. */
#ifndef HCCL_AMD_EXPERTS_H_
#define HCCL_AMD_EXPERTS_H_

#include <hccl/hccl_types.h>

#ifdef __cplusplus
extern "C" {
#endif

#define HCCL_AMD_MAX_EXPERTS 1024u   /* of a router */
#define HCCL_AMD_MAX_GROUPS 4096u    /* groups of rows, and weights, of one product */
#define HCCL_AMD_MAX_TOPK 16u
#define HCCL_AMD_MAX_EXPERT_GROUPS 64u   /* groups of experts of a router */
#define HCCL_AMD_MAX_NORM_WIDTH 32768u   /* of a row that is normed */

typedef enum HcclAmdScaleTypeDef {
    HCCL_AMD_SCALE_NONE = 0,
    HCCL_AMD_SCALE_FP32 = 1,
    HCCL_AMD_SCALE_E8M0 = 2
} HcclAmdScaleType;

/* Bytes of device workspace that HcclAmdExpertRoute needs (host pointer `bytes`). */
extern HcclResult HcclAmdExpertRouteWorkspace(uint64_t tokens, uint32_t experts, uint64_t *bytes);

/* Chooses topK of `experts` experts for every token and counts them.
 *   logits[tokens][logitStride]   FP32, FP16 or BFP16
 *   tokenMask[tokens]             0: the token takes no part (its logits are not looked at); NULL: all take part
 * The topK largest logits win, ties go to the lowest expert; a logit of -inf or NaN is never chosen.
 *   expertOf[tokens][topK]        the experts, largest logit first; -1 where there is none
 *   weights[tokens][topK]         softmax probabilities of the row; with `renormalise` divided by the sum of the chosen ones; 0 where expertOf is -1
 *   rowOf[tokens][topK]           the row of (token, choice) when all are sorted by expert, then by token; -1 where there is none
 *   counts[experts + 1]           rows per expert; at [experts] the number of tokens that chose any
 *   offsets[experts + 1]          first row of every expert; at [experts] the number of rows
 *   loss[1]                       lossScale * experts * sum over e of (counts[e] / rows) * (sum of the probabilities of e / tokens that chose);
 *                                 0 without rows
 * A NaN or +inf logit of a token that chose any makes all its probabilities, and with them its weights and the loss, NaN, as the formula has it.
 * topK <= experts.  workspace: 16-byte aligned, HcclAmdExpertRouteWorkspace bytes, free for other use once the stream is past the call. */
extern HcclResult HcclAmdExpertRoute(const void *logits, HcclDataType logitType, uint64_t tokens, uint32_t experts, uint64_t logitStride,
    uint32_t topK, uint32_t renormalise, const uint8_t *tokenMask, float lossScale, int32_t *expertOf, float *weights, int32_t *rowOf,
    int32_t *counts, int32_t *offsets, float *loss, void *workspace, uint64_t workspaceBytes, void *stream);

/* Gradient of the logits, from weightGrad[tokens][topK] and lossGrad[1] (either may be NULL: zero).  logits, tokenMask, sizes
 * and settings as given to HcclAmdExpertRoute; expertOf and counts as it left them.  Rows that chose nothing get zeros. */
extern HcclResult HcclAmdExpertRouteGrad(const void *logits, HcclDataType logitType, uint64_t tokens, uint32_t experts, uint64_t logitStride,
    uint32_t topK, uint32_t renormalise, const uint8_t *tokenMask, float lossScale, const int32_t *expertOf, const int32_t *counts,
    const float *weightGrad, const float *lossGrad, void *logitGrad, uint64_t logitGradStride, void *stream);

/* out[rowOf[t][j]] = x[t] for every token t and choice j with 0 <= rowOf[t][j] < rows.
 *   scaleType NONE          a copy, in x's type (FP32, FP16, BFP16)
 *   FP32, E8M0              8-bit rows (see above) and scales[rows][scaleStride], ceil(width / 128) to a row
 * rowOf NULL (topK 1): row t is token t.  Rows that no choice names are left as they are. */
extern HcclResult HcclAmdExpertPack(const void *x, HcclDataType type, uint64_t tokens, uint64_t width, uint64_t xStride, uint32_t topK,
    const int32_t *rowOf, HcclAmdScaleType scaleType, void *out, uint64_t rows, uint64_t outStride, void *scales, uint64_t scaleStride,
    void *stream);

/* y[t] = sum over j of weights[t][j] * x[rowOf[t][j]], over the choices with 0 <= rowOf < rows.  weights NULL: all 1, which is
 * the gradient of HcclAmdExpertPack.  rowOf NULL (topK 1): row t.  FP32, FP16 or BFP16, x and y alike. */
extern HcclResult HcclAmdExpertCombine(const void *x, HcclDataType type, uint64_t rows, uint64_t width, uint64_t xStride, uint64_t tokens,
    uint32_t topK, const int32_t *rowOf, const float *weights, void *y, uint64_t yStride, void *stream);

/* Gradients of HcclAmdExpertCombine: xGrad[rowOf[t][j]] = weights[t][j] * yGrad[t] and weightGrad[t][j] = <yGrad[t], x[rowOf[t][j]]>
 * (0 where there is no row).  Either output may be NULL.  Rows that no choice names are left as they are. */
extern HcclResult HcclAmdExpertCombineGrad(const void *yGrad, uint64_t yGradStride, const void *x, HcclDataType type, uint64_t rows,
    uint64_t width, uint64_t xStride, uint64_t tokens, uint32_t topK, const int32_t *rowOf, const float *weights, void *xGrad,
    uint64_t xGradStride, float *weightGrad, void *stream);

/* Weights in 8 bits, one scale for each block of 128 x 128 (blocks at the edge are smaller).
 *   w[experts][n][wStride]               FP32, FP16 or BFP16
 *   q[experts][n][ceil128(k)]            scales[experts][ceil(n/128)][ceil(k/128)]
 *   qT[experts][k][ceil128(n)]           the same values transposed, scalesT[experts][ceil(k/128)][ceil(n/128)]
 * Either pair may be NULL.  Limit: experts * ceil(n/128) * ceil(k/128) <= 2^23. */
extern HcclResult HcclAmdBlockQuantWeights(const void *w, HcclDataType type, uint32_t experts, uint64_t n, uint64_t k, uint64_t wStride,
    HcclAmdScaleType scaleType, void *q, void *scales, void *qT, void *scalesT, void *stream);

/* 8-bit columns: x[rows][xStride] of `width` columns, transposed, with one scale per column and 128 rows of a group.
 * offsets[groups + 1] are the groups' first rows, ascending.  In qT[width][columns] every group starts at a multiple of 128 and is
 * padded with zeros to one; group g starts at sum over h < g of ceil128(rows of h).  scales[columns / 128][width].
 * columns: a multiple of 128, at least (rows / 128 + groups) * 128 (rows / 128 rounded down) so that any offsets fit.
 * Limits: rows <= 2^28, (rows / 128 + groups) * ceil(width / 128) <= 2^23. */
extern HcclResult HcclAmdBlockQuantColumns(const void *x, HcclDataType type, uint64_t rows, uint64_t width, uint64_t xStride,
    uint32_t groups, const int32_t *offsets, HcclAmdScaleType scaleType, void *qT, uint64_t columns, void *scales, void *stream);

/* y[r] = a[r] * w[e]^T for the rows r of every group, e the group's expert.
 *   a[rows][aStride]             8-bit rows of k values, aScales[rows][aScaleStride]
 *   offsets[groups + 1]          first row of every group, ascending; NULL: one group of all rows
 *   expertOfGroup[groups]        the weights a group uses; NULL: group g uses weights g, groups <= experts
 *   w[experts][n][ceil128(k)]    8-bit weights, wScales[experts][ceil(n/128)][ceil(k/128)], as HcclAmdBlockQuantWeights leaves them
 *   y[rows][yStride]             yType FP32, FP16 or BFP16, n to a row
 * Rows outside all groups are left as they are.  The gradient of the rows is the same call with the transposed weights.
 * Sums: products are exact and added in 32 bits, whatever the type of the results.
 * Limits: rows <= 2^28, and (rows / 128 + the lesser of rows and groups) * ceil(n / 128) <= 2^22. */
extern HcclResult HcclAmdBlockMatmul(const void *a, uint64_t aStride, const void *aScales, uint64_t aScaleStride, uint64_t rows,
    uint32_t groups, const int32_t *offsets, const int32_t *expertOfGroup, const void *w, const void *wScales, uint32_t experts,
    uint64_t n, uint64_t k, HcclAmdScaleType scaleType, void *y, HcclDataType yType, uint64_t yStride, void *stream);

/* wGrad[e][n][k] = sum over the rows r of e's groups of yGrad[r][n] * x[r][k] (added to what is there with `accumulate`), from
 * both sides' 8-bit columns (HcclAmdBlockQuantColumns of the same rows, groups, offsets and columns, below 2^23).  offsets and
 * expertOfGroup as in HcclAmdBlockMatmul.  Experts without rows get zeros; all sums are in 32 bits.  wGrad: FP32, FP16 or BFP16.
 * Limit: ceil(n / 128) * ceil(k / 128), rounded up to a multiple of 8, times experts <= 2^22. */
extern HcclResult HcclAmdBlockMatmulGradWeight(const void *yGradT, const void *yGradScales, const void *xT, const void *xScales,
    uint64_t columns, uint64_t rows, uint64_t n, uint64_t k, HcclAmdScaleType scaleType, uint32_t groups, const int32_t *offsets,
    const int32_t *expertOfGroup, uint32_t experts, void *wGrad, HcclDataType gradType, uint32_t accumulate, void *stream);

/* s = x + residual (x alone if residual is NULL), y = s * gain / sqrt(mean of s^2 over the row + epsilon).
 *   x, residual[rows][...]        FP32, FP16 or BFP16, sum and y alike; widened, and s and y stay in 32 bits until they are rounded once for
 *                                 each output.  The squares are summed in 64 bits: no row overflows
 *   gain[width]                   gainType: FP32, or the rows' type; NULL: all 1
 *   sum[rows][sumStride]          s; NULL: not wanted; may be x or residual, of the same stride
 *   y[rows][yStride]              NULL: not wanted
 *   q[rows][qStride], scales      8-bit rows of y as it is in 32 bits (see above), ceil(width / 128) scales to a row; both NULL with
 *                                 HCCL_AMD_SCALE_NONE
 * epsilon: 0 or more; with 0 the factor of a row whose root mean square is below 2^-127 (zeros, and next to them) is infinite.
 * width <= HCCL_AMD_MAX_NORM_WIDTH, rows < 2^31. */
extern HcclResult HcclAmdNormRows(const void *x, HcclDataType type, uint64_t rows, uint64_t width, uint64_t xStride, const void *residual,
    uint64_t residualStride, const void *gain, HcclDataType gainType, float epsilon, void *sum, uint64_t sumStride, void *y, uint64_t yStride,
    HcclAmdScaleType scaleType, void *q, uint64_t qStride, void *scales, uint64_t scaleStride, void *stream);

/* Bytes of device workspace that HcclAmdNormRowsGrad needs for gainGrad (host pointer `bytes`). */
extern HcclResult HcclAmdNormRowsGradWorkspace(uint64_t rows, uint64_t width, uint64_t *bytes);

/* Gradients of HcclAmdNormRows from yGrad and from sumGrad (NULL: none), what reaches the sum from elsewhere; `sum` as the forward call
 * left it (x, if there was no residual).
 *   xGrad[rows][xGradStride]      of x and of residual alike; NULL: not wanted; may be yGrad or sumGrad, of the same stride
 *   gainGrad[width]               32 bits (added to what is there with `accumulate`); NULL: not wanted, no workspace then
 * workspace: 16-byte aligned, HcclAmdNormRowsGradWorkspace bytes, free for other use once the stream is past the call. */
extern HcclResult HcclAmdNormRowsGrad(const void *yGrad, uint64_t yGradStride, const void *sum, HcclDataType type, uint64_t rows, uint64_t width,
    uint64_t sumStride, const void *gain, HcclDataType gainType, float epsilon, const void *sumGrad, uint64_t sumGradStride, void *xGrad,
    uint64_t xGradStride, float *gainGrad, uint32_t accumulate, void *workspace, uint64_t workspaceBytes, void *stream);

/* a[r][i] = g / (1 + exp(-g)) * u with g = h[r][i], u = h[r][width + i]: what stands between an expert's two products.
 *   h[rows][hStride]              2 * width to a row; FP32, FP16 or BFP16
 *   used[1]                       how many rows there are, on the device (a receive buffer's offsets[groups], say), brought into [0, rows];
 *                                 NULL: all.  Rows behind them are left as they are, in every output
 *   scaleType NONE                out[rows][outStride] in h's type
 *   FP32, E8M0                    8-bit rows (see above) of a as it is in 32 bits, and scales[rows][scaleStride], ceil(width / 128) to a row */
extern HcclResult HcclAmdExpertGate(const void *h, HcclDataType type, uint64_t rows, uint64_t width, uint64_t hStride, const int32_t *used,
    HcclAmdScaleType scaleType, void *out, uint64_t outStride, void *scales, uint64_t scaleStride, void *stream);

/* Gradient of HcclAmdExpertGate, and a once more for the gradient of the weights behind it, for those who did not keep it.
 *   hGrad[rows][hGradStride]      2 * width to a row; NULL: not wanted; may be h, of the same stride
 *   a[rows][aStride]              in h's type; NULL: not wanted; may be aGrad, of the same stride */
extern HcclResult HcclAmdExpertGateGrad(const void *aGrad, uint64_t aGradStride, const void *h, HcclDataType type, uint64_t rows, uint64_t width,
    uint64_t hStride, const int32_t *used, void *hGrad, uint64_t hGradStride, void *a, uint64_t aStride, void *stream);

typedef enum HcclAmdScoreDef {
    HCCL_AMD_SCORE_SOFTMAX = 0,
    HCCL_AMD_SCORE_SIGMOID = 1
} HcclAmdScore;

/* Chooses topK experts for every token by their scores, s = softmax(logits) over all experts or 1 / (1 + exp(-logits)), and counts them.
 *   logits, tokenMask, expertOf, rowOf, counts, offsets    as in HcclAmdExpertRoute
 *   bias[experts]                 added to the scores for the choice alone, in 64 bits; NULL: none.  -inf or NaN: never chosen, and the way to
 *                                 switch an expert off: finite biases that are far apart (100 and more) do as well, but then more
 *                                 tokens take 64 bits; all of them where biases are 1e4 apart or 2^24
 *                                 from 0, which is five times as slow
 *   groups, groupsKept, groupTop  the experts are `groups` groups of as many neighbours each; a token's experts come from its groupsKept best groups,
 *                                 by the sum of a group's groupTop (1 or 2) largest s + bias.  groups = groupsKept = 1: from all of them
 *   weights[tokens][topK]         weightScale * s, with `renormalise` weightScale * s / (sum of the chosen s): without the bias; 0 where expertOf is -1
 * Largest s + bias first, worked out in 64 bits, ties to the lowest group and expert.  A logit of -inf or NaN is never chosen, and nor is a group
 * without any that can be; in a softmax a NaN or +inf logit makes the weights of its token's others NaN, as the formula has it.
 * topK <= groupsKept * (experts / groups).  workspace: 16-byte aligned, HcclAmdExpertRouteScoredWorkspace bytes, free for other use once the stream
 * is past the call. */
extern HcclResult HcclAmdExpertRouteScoredWorkspace(uint64_t tokens, uint32_t experts, uint64_t *bytes);
extern HcclResult HcclAmdExpertRouteScored(const void *logits, HcclDataType logitType, uint64_t tokens, uint32_t experts, uint64_t logitStride,
    HcclAmdScore score, const float *bias, uint32_t groups, uint32_t groupsKept, uint32_t groupTop, uint32_t topK, uint32_t renormalise,
    float weightScale, const uint8_t *tokenMask, int32_t *expertOf, float *weights, int32_t *rowOf, int32_t *counts, int32_t *offsets,
    void *workspace, uint64_t workspaceBytes, void *stream);

/* Gradient of the logits from weightGrad[tokens][topK]; expertOf as HcclAmdExpertRouteScored left it.  Every logit's gradient is written; those of
 * tokens that chose nothing are zero, and so are, but for a softmax that is not renormalised, those of experts that were not chosen.  (The bias
 * only chooses: it has no gradient.)  A NaN or +inf logit makes all gradients of its token NaN in a softmax that is not renormalised.  In one that is, only
 * the chosen logits are read: +inf among them makes their gradients NaN, and of a NaN or +inf among the others, which made the weights NaN, the gradients
 * have what weightGrad has. */
extern HcclResult HcclAmdExpertRouteScoredGrad(const void *logits, HcclDataType logitType, uint64_t tokens, uint32_t experts, uint64_t logitStride,
    HcclAmdScore score, uint32_t topK, uint32_t renormalise, float weightScale, const int32_t *expertOf, const float *weightGrad, void *logitGrad,
    uint64_t logitGradStride, void *stream);

/* newBias[e] = bias[e] + rate where counts[e] is below the mean of all experts' counts, - rate where it is above it.  counts[experts] may be one router's or
 * the sum of all ranks' (HcclAllReduce, INT32).  newBias may be bias. */
extern HcclResult HcclAmdExpertBias(const int32_t *counts, uint32_t experts, float rate, const float *bias, float *newBias, void *stream);

/* A tensor of gradients: `count` elements (2^36 at most) behind each other (FP32, FP16 or BFP16), aligned to one.  Lists of these, of 2^24 at most, are host
 * memory, read during the call. */
typedef struct HcclAmdGradTensorDef {
    const void *in;
    void *out;             /* HcclAmdGradClip writes here; may be `in` */
    uint64_t count;
    HcclDataType type;
    uint32_t reserved;     /* 0 */
} HcclAmdGradTensor;

/* Bytes of device workspace that HcclAmdGradSquares needs (host pointer `bytes`). */
extern HcclResult HcclAmdGradSquaresWorkspace(const HcclAmdGradTensor *tensors, uint32_t n, uint64_t *bytes);

/* squares[0] = the sum of the squares of all elements of all tensors (added to what is there with `accumulate`), in 64 bits throughout: neither
 * large nor small gradients leave its range.  Where each rank has part of the gradients, HcclAllReduce (FP64, sum) of the ranks' squares comes next.
 * workspace: 16-byte aligned, HcclAmdGradSquaresWorkspace bytes, free for other use once the stream is past the call. */
extern HcclResult HcclAmdGradSquares(const HcclAmdGradTensor *tensors, uint32_t n, uint32_t accumulate, double *squares, void *workspace,
    uint64_t workspaceBytes, void *stream);

/* With norm = sqrt(squares[0]): out = in * (maxNorm / norm) where norm > maxNorm, else out = in (nothing is read or written then where they are the
 * same).  maxNorm / norm is rounded to 32 bits once, each product once more to the tensor's type.  norm[1]: written, in 32 bits; NULL: not wanted.  As
 * the formula has it, a NaN among the gradients makes all of them NaN, an infinity the finite ones 0 and itself NaN: norm[0] says so. */
extern HcclResult HcclAmdGradClip(const HcclAmdGradTensor *tensors, uint32_t n, const double *squares, float maxNorm, float *norm, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* HCCL_AMD_EXPERTS_H_ */
