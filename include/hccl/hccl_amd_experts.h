/* Operators of an expert-parallel layer, next to HcclAlltoAllV.  Nothing here exists in the reference.
 *
 *   HcclAmdExpertRoute      logits -> experts, weights, per-expert counts, rows in expert order, balance loss
 *   HcclAmdExpertPack       tokens -> rows in expert order (an all-to-all-v's send buffer), copied or in 8 bits
 *   HcclAmdBlockMatmul      8-bit rows, group by group, times their experts' 8-bit weights
 *   HcclAmdExpertCombine    rows -> tokens, weighted and summed
 *   ...Grad, HcclAmdBlockMatmulGradWeight, HcclAmdBlockQuant...   their gradients and what these read
 *
 * All of them: device pointers unless said otherwise, of one GPU; no communicator; the work is queued on `stream` (a
 * hipStream_t, not null) and nothing is allocated, copied or waited for, so a call can be captured into a HIP graph.  An
 * output must not overlap an input or another output.  Same inputs, same bits: no atomics whose order matters.  Strides are
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

#ifdef __cplusplus
}
#endif
#endif /* HCCL_AMD_EXPERTS_H_ */
