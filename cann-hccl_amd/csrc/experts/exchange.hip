// Rows into expert order and back: HcclAmdExpertPack, HcclAmdExpertCombine and its gradient.  No arithmetic to speak of: bytes
// moved bound all three, so every row is read once and written once, 16 bytes to a lane, 512 values to a wave and step, and what
// a step needs is loaded before any of it is used, the token's row numbers and weights first.  A copy to all of a token's rows needs
// one reading of the token; a wave to a token and 512 values gives 131072 waves for 16384 x 4096, each with no more than it can
// hold in registers.
//
// Measured, where a large copy reaches 5.15 TB/s: 16384 tokens of 4096 values to eight rows each in 8 bits (0.68 GB) 122 us, 5.5 TB/s;
// back and weighted (1.2 GB) 246 us, 4.9 TB/s; the gradients of that (2.2 GB) 424 us, 5.2 TB/s.  2001 values to a row, off every
// boundary (8191 tokens, four rows each): 41 and 74 us, 4.0 TB/s.  64 tokens of 8192: 4 us.
#include <type_traits>

#include "common.h"

namespace hcclamd {
namespace experts {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kEach = 8;                 // consecutive values of a lane
constexpr int kPiece = 64 * kEach;       // of a wave

// Launches are at most this many workgroups wide (a grid holds fewer than 2^32 threads); their waves take several pieces beyond.
constexpr int64_t kMostBlocks = int64_t(1) << 22;

__device__ __forceinline__ int64_t FirstWave()
{
    return int64_t(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
}

// The rows of a token's choices, all loaded at once: choice j's is in lane j, -1 where there is none within [0, rows).
__device__ __forceinline__ int RowsOf(const int32_t *rowOf, int64_t token, int topK, int64_t rows)
{
    const int j = int(__lane_id());
    if (rowOf == nullptr) {
        return j == 0 && token < rows ? int(token) : -1;
    }
    const int r = j < topK ? rowOf[token * topK + j] : -1;
    return r >= 0 && r < rows ? r : -1;
}

struct PackArgs {
    const void *x;
    const int32_t *rowOf;
    void *out;
    void *scales;
    int64_t xStride, outStride, scaleStride;
    int64_t rows;
    int64_t waves;       // tokens * pieces
    int width, padded, topK, pieces;
};

// A wave to a token and a piece of its width: read once, written to all of the token's rows.  T: words of the elements' size (as numbers, some
// NaN would come out with other bits).
template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads) CopyKernel(PackArgs a)
{
    for (int64_t w = FirstWave(); w < a.waves; w += int64_t(gridDim.x) * kWaves) {
        const int64_t t = w / a.pieces;
        const int at = int(w % a.pieces) * kPiece + int(threadIdx.x % 64) * kEach;
        const int rows = RowsOf(a.rowOf, t, a.topK, a.rows);
        T v[kEach];
        LoadPart<kWide, kEach>(static_cast<const T *>(a.x) + t * a.xStride, at, a.width, v);
        for (int j = 0; j < a.topK; j++) {
            const int64_t r = __builtin_amdgcn_readlane(rows, j);
            if (r >= 0) {
                StorePart<kWide, kEach>(static_cast<T *>(a.out) + r * a.outStride, at, a.width, v);
            }
        }
    }
}

// The same with 8-bit rows: 16 lanes hold a block of 128 values and agree on its maximum.
template <typename T, HcclAmdScaleType kScale, bool kWide>
__global__ void __launch_bounds__(kThreads) QuantKernel(PackArgs a)
{
    for (int64_t w = FirstWave(); w < a.waves; w += int64_t(gridDim.x) * kWaves) {
        const int64_t t = w / a.pieces;
        const int at = int(w % a.pieces) * kPiece + int(threadIdx.x % 64) * kEach;
        const int rows = RowsOf(a.rowOf, t, a.topK, a.rows);
        float v[kEach];
        LoadPart<kWide, kEach>(static_cast<const T *>(a.x) + t * a.xStride, at, a.width, v);
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            top = __builtin_fmaxf(top, FiniteSize(v[i]));
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            top = __builtin_fmaxf(top, __shfl_xor(top, d, 64));
        }
        const BlockScale<kScale> scale(top);
        Word2 q;
        float s[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            s[i] = Scaled8(v[i], scale.times);
        }
        q.x = Quantise4(s[0], s[1], s[2], s[3]);
        q.y = Quantise4(s[4], s[5], s[6], s[7]);
        for (int j = 0; j < a.topK; j++) {
            const int64_t r = __builtin_amdgcn_readlane(rows, j);
            if (r >= 0 && at < a.padded) {
                *reinterpret_cast<Word2 *>(static_cast<uint8_t *>(a.out) + r * a.outStride + at) = q;
                if (threadIdx.x % 16 == 0) {
                    static_cast<typename BlockScale<kScale>::Stored *>(a.scales)[r * a.scaleStride + at / 128] = scale.stored;
                }
            }
        }
    }
}

struct CombineArgs {
    const void *x;
    const int32_t *rowOf;
    const float *weights;
    void *y;
    const void *yGrad;
    void *xGrad;
    float *weightGrad;
    int64_t xStride, yStride, xGradStride;
    int64_t rows;
    int64_t waves;
    int tokens, width, topK, pieces;
};

// A wave to a token and a piece of its width; the token's rows four at a time.
template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads) CombineKernel(CombineArgs a)
{
    for (int64_t w = FirstWave(); w < a.waves; w += int64_t(gridDim.x) * kWaves) {
        const int64_t t = w / a.pieces;
        const int at = int(w % a.pieces) * kPiece + int(threadIdx.x % 64) * kEach;
        const int rows = RowsOf(a.rowOf, t, a.topK, a.rows), lane = int(__lane_id());
        const float weight = rows >= 0 && a.weights != nullptr ? a.weights[t * a.topK + lane] : 1.0f;
        float sum[kEach] = {};
        for (int j0 = 0; j0 < a.topK; j0 += 4) {
            float v[4][kEach];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t r = __builtin_amdgcn_readlane(rows, j0 + j);     // (-1 from lanes beyond topK)
                if (r >= 0) {
                    LoadPart<kWide, kEach>(static_cast<const T *>(a.x) + r * a.xStride, at, a.width, v[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (__builtin_amdgcn_readlane(rows, j0 + j) >= 0) {
                    const float by = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), j0 + j));
#pragma unroll
                    for (int i = 0; i < kEach; i++) {
                        sum[i] = __builtin_fmaf(by, v[j][i], sum[i]);
                    }
                }
            }
        }
        StorePart<kWide, kEach>(static_cast<T *>(a.y) + t * a.yStride, at, a.width, sum);
    }
}

// A workgroup to a token: yGrad is read once, its rows' products with it are summed over the width.  kRows: topK at most.
template <typename T, int kRows, bool kWide>
__global__ void __launch_bounds__(kThreads) CombineGradKernel(CombineArgs a)
{
    __shared__ float part[kWaves][kRows];
    for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
        const T *dy = static_cast<const T *>(a.yGrad) + t * a.yStride;
        const int rows = RowsOf(a.rowOf, t, a.topK, a.rows), lane = int(__lane_id());
        const float weight = rows >= 0 && a.weights != nullptr ? a.weights[t * a.topK + lane] : 1.0f;
        int64_t r[kRows];
        float by[kRows], dot[kRows];
#pragma unroll
        for (int j = 0; j < kRows; j++) {
            r[j] = __builtin_amdgcn_readlane(rows, j);
            by[j] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), j));
            dot[j] = 0.0f;
        }
        for (int at = int(threadIdx.x) * kEach; at < a.width; at += kThreads * kEach) {
            float d[kEach];
            LoadPart<kWide, kEach>(dy, at, a.width, d);
#pragma unroll
            for (int j = 0; j < kRows; j++) {
                if (r[j] >= 0) {
                    if (a.weightGrad != nullptr) {
                        float v[kEach];
                        LoadPart<kWide, kEach>(static_cast<const T *>(a.x) + r[j] * a.xStride, at, a.width, v);
#pragma unroll
                        for (int i = 0; i < kEach; i++) {
                            dot[j] = __builtin_fmaf(d[i], v[i], dot[j]);
                        }
                    }
                    if (a.xGrad != nullptr) {
                        float g[kEach];
#pragma unroll
                        for (int i = 0; i < kEach; i++) {
                            g[i] = by[j] * d[i];
                        }
                        StorePart<kWide, kEach>(static_cast<T *>(a.xGrad) + r[j] * a.xGradStride, at, a.width, g);
                    }
                }
            }
        }
        if (a.weightGrad == nullptr) {
            continue;
        }
#pragma unroll
        for (int j = 0; j < kRows; j++) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                dot[j] += __shfl_xor(dot[j], d, 64);
            }
            if (threadIdx.x % 64 == 0) {
                part[threadIdx.x / 64][j] = dot[j];
            }
        }
        __syncthreads();
        if (int(threadIdx.x) < a.topK) {
            float sum = 0.0f;
            for (int i = 0; i < kWaves; i++) {
                sum += part[i][threadIdx.x];
            }
            a.weightGrad[t * a.topK + threadIdx.x] = sum;
        }
        __syncthreads();   // before the next token's sums
    }
}

template <typename F>
HcclResult ByType(HcclDataType type, F f)
{
    switch (type) {
        case HCCL_DATA_TYPE_FP32:
            return f(float{});
        case HCCL_DATA_TYPE_FP16:
            return f(_Float16{});
        default:
            return f(__bf16{});
    }
}

// Whether rows can be taken kEach values at a time, 16 bytes to a load (two for 32 bits).
bool Wide(HcclDataType type, uint64_t width, const void *p, int64_t stride)
{
    return width % kEach == 0 && Aligned(p, 16) && uint64_t(stride) * SizeOf(type) % 16 == 0;
}

uint32_t BlocksOf(int64_t waves)
{
    const int64_t blocks = (waves + kWaves - 1) / kWaves;
    return uint32_t(blocks < kMostBlocks ? blocks : kMostBlocks);
}

}  // namespace
}  // namespace experts
}  // namespace hcclamd

using namespace hcclamd::experts;

extern "C" {

HcclResult HcclAmdExpertPack(const void *x, HcclDataType type, uint64_t tokens, uint64_t width, uint64_t xStride, uint32_t topK,
    const int32_t *rowOf, HcclAmdScaleType scaleType, void *out, uint64_t rows, uint64_t outStride, void *scales, uint64_t scaleStride,
    void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK_TYPE(scaleType == HCCL_AMD_SCALE_NONE || Scaled(scaleType));
    EXPERTS_CHK(topK >= 1 && topK <= HCCL_AMD_MAX_TOPK);
    EXPERTS_CHK(tokens <= kMaxSize && rows <= kMaxSize && width <= kMaxSize - 4096);
    EXPERTS_CHK(rowOf != nullptr || topK == 1);
    if (tokens == 0 || rows == 0 || width == 0) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(x);
    EXPERTS_CHK_PTR(out);
    EXPERTS_CHK(Stride(xStride, width));
    EXPERTS_CHK(AlignedTo(type, x) && Aligned(rowOf, 4));
    PackArgs a{};
    a.x = x;
    a.rowOf = rowOf;
    a.out = out;
    a.scales = scales;
    a.xStride = int64_t(xStride == 0 ? width : xStride);
    a.rows = int64_t(rows);
    a.width = int(width);
    a.topK = int(topK);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    if (scaleType == HCCL_AMD_SCALE_NONE) {
        EXPERTS_CHK(Stride(outStride, width));
        EXPERTS_CHK(AlignedTo(type, out));
        a.outStride = int64_t(outStride == 0 ? width : outStride);
        a.pieces = int((width + kPiece - 1) / kPiece);
        a.waves = int64_t(tokens) * a.pieces;
        const bool wide = Wide(type, width, x, a.xStride) && Wide(type, width, out, a.outStride);
        return ByType(type, [&](auto of) {
            typedef std::conditional_t<sizeof(of) == 4, uint32_t, uint16_t> T;
            return Launch("HcclAmdExpertPack", wide ? CopyKernel<T, true> : CopyKernel<T, false>, BlocksOf(a.waves), kThreads, 0, on, a);
        });
    }
    EXPERTS_CHK_PTR(scales);
    EXPERTS_CHK(ScaleAligned(scaleType, scales));
    a.outStride = int64_t(outStride == 0 ? Up128(width) : outStride);
    a.scaleStride = int64_t(scaleStride == 0 ? Blocks(width) : scaleStride);
    EXPERTS_CHK(Stride(outStride, Up128(width)) && outStride % 16 == 0 && Aligned(out, 16));
    EXPERTS_CHK(Stride(scaleStride, Blocks(width)));
    a.padded = int(Up128(width));
    a.pieces = (a.padded + kPiece - 1) / kPiece;
    a.waves = int64_t(tokens) * a.pieces;
    const bool wide = Wide(type, width, x, a.xStride);
    return ByType(type, [&](auto of) {
        typedef decltype(of) T;
        const auto go = [&](auto kernel) { return Launch("HcclAmdExpertPack", kernel, BlocksOf(a.waves), kThreads, 0, on, a); };
        if (scaleType == HCCL_AMD_SCALE_FP32) {
            return wide ? go(QuantKernel<T, HCCL_AMD_SCALE_FP32, true>) : go(QuantKernel<T, HCCL_AMD_SCALE_FP32, false>);
        }
        return wide ? go(QuantKernel<T, HCCL_AMD_SCALE_E8M0, true>) : go(QuantKernel<T, HCCL_AMD_SCALE_E8M0, false>);
    });
}

HcclResult HcclAmdExpertCombine(const void *x, HcclDataType type, uint64_t rows, uint64_t width, uint64_t xStride, uint64_t tokens,
    uint32_t topK, const int32_t *rowOf, const float *weights, void *y, uint64_t yStride, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK(topK >= 1 && topK <= HCCL_AMD_MAX_TOPK);
    EXPERTS_CHK(tokens <= kMaxSize && rows <= kMaxSize && width <= kMaxSize - 4096);
    EXPERTS_CHK(rowOf != nullptr || topK == 1);
    if (tokens == 0 || width == 0) {
        return HCCL_SUCCESS;
    }
    if (rows != 0) {
        EXPERTS_CHK_PTR(x);
    }
    EXPERTS_CHK_PTR(y);
    EXPERTS_CHK(Stride(xStride, width));
    EXPERTS_CHK(Stride(yStride, width));
    EXPERTS_CHK(AlignedTo(type, x) && AlignedTo(type, y) && Aligned(rowOf, 4) && Aligned(weights, 4));
    CombineArgs a{};
    a.x = x;
    a.rowOf = rowOf;
    a.weights = weights;
    a.y = y;
    a.xStride = int64_t(xStride == 0 ? width : xStride);
    a.yStride = int64_t(yStride == 0 ? width : yStride);
    a.rows = int64_t(rows);
    a.tokens = int(tokens);
    a.width = int(width);
    a.topK = int(topK);
    a.pieces = int((width + kPiece - 1) / kPiece);
    a.waves = int64_t(tokens) * a.pieces;
    const bool wide = Wide(type, width, x, a.xStride) && Wide(type, width, y, a.yStride);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    return ByType(type, [&](auto of) {
        typedef decltype(of) T;
        return Launch("HcclAmdExpertCombine", wide ? CombineKernel<T, true> : CombineKernel<T, false>, BlocksOf(a.waves), kThreads, 0, on, a);
    });
}

HcclResult HcclAmdExpertCombineGrad(const void *yGrad, uint64_t yGradStride, const void *x, HcclDataType type, uint64_t rows,
    uint64_t width, uint64_t xStride, uint64_t tokens, uint32_t topK, const int32_t *rowOf, const float *weights, void *xGrad,
    uint64_t xGradStride, float *weightGrad, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK(topK >= 1 && topK <= HCCL_AMD_MAX_TOPK);
    EXPERTS_CHK(tokens <= kMaxSize && rows <= kMaxSize && width <= kMaxSize - 4096);
    EXPERTS_CHK(rowOf != nullptr || topK == 1);
    if (tokens == 0 || (xGrad == nullptr && weightGrad == nullptr)) {
        return HCCL_SUCCESS;
    }
    if (width != 0) {
        EXPERTS_CHK_PTR(yGrad);
        if (rows != 0 && weightGrad != nullptr) {
            EXPERTS_CHK_PTR(x);
        }
    }
    EXPERTS_CHK(Stride(xStride, width));
    EXPERTS_CHK(Stride(yGradStride, width));
    EXPERTS_CHK(Stride(xGradStride, width));
    EXPERTS_CHK(AlignedTo(type, x) && AlignedTo(type, yGrad) && AlignedTo(type, xGrad));
    EXPERTS_CHK(Aligned(rowOf, 4) && Aligned(weights, 4) && Aligned(weightGrad, 4));
    CombineArgs a{};
    a.x = x;
    a.rowOf = rowOf;
    a.weights = weights;
    a.yGrad = yGrad;
    a.xGrad = xGrad;
    a.weightGrad = weightGrad;
    a.xStride = int64_t(xStride == 0 ? width : xStride);
    a.yStride = int64_t(yGradStride == 0 ? width : yGradStride);
    a.xGradStride = int64_t(xGradStride == 0 ? width : xGradStride);
    a.rows = int64_t(rows);
    a.tokens = int(tokens);
    a.width = int(width);
    a.topK = int(topK);
    const bool wide = Wide(type, width, x, a.xStride) && Wide(type, width, yGrad, a.yStride) && Wide(type, width, xGrad, a.xGradStride);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    return ByType(type, [&](auto of) {
        typedef decltype(of) T;
        const auto go = [&](auto kernel) { return Launch("HcclAmdExpertCombineGrad", kernel, BlocksOf(int64_t(tokens) * kWaves), kThreads, 0, on, a); };
        if (topK <= 2) {
            return wide ? go(CombineGradKernel<T, 2, true>) : go(CombineGradKernel<T, 2, false>);
        }
        if (topK <= 8) {
            return wide ? go(CombineGradKernel<T, 8, true>) : go(CombineGradKernel<T, 8, false>);
        }
        return wide ? go(CombineGradKernel<T, 16, true>) : go(CombineGradKernel<T, 16, false>);
    });
}

}  // extern "C"
