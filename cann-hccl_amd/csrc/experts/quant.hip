// 8-bit operands of the experts' products that are not rows: columns (HcclAmdBlockQuantColumns, for the weights' gradient, whose
// sum runs over rows) and weights (HcclAmdBlockQuantWeights).  Both take tiles of 128 x 128, read once, 16 bytes to a lane; a
// thread holds eight values of each of eight rows that follow each other, so its part of a transposed row is eight bytes in one
// piece.  The transposed tile passes through LDS and leaves it in whole lines of 128 bytes.  Bytes moved bound it: 16411 rows of
// 4096 values (0.2 GB) take 48 us, 4.2 TB/s, where a large copy reaches 5.15.
#include <type_traits>

#include "common.h"

namespace hcclamd {
namespace experts {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 128;
constexpr int kPitch = kTile + 16;    // LDS bytes from one transposed row to the next

// Where the eight bytes of rows 8 * group + [0, 8) of column c lie in the transposed tile.  16-byte pieces change places by column / 16: with the
// pitch, which moves every other eight columns by half the banks, the 64 writes of a wave are spread over all banks evenly.
__device__ __forceinline__ int TransposedAt(int c, int group) { return c * kPitch + (group ^ c / 16 * 2) * 8; }

struct TileArgs {
    const void *x;
    const int32_t *offsets;
    void *q, *scales;      // rows as they are (weights)
    void *qT, *scalesT;    // transposed
    int64_t stride;        // of x
    int64_t pitchT;        // of qT, bytes
    int rows, width, groups;
};

// 8 x 8 values of the tile at (first, column): rows first + 8 * (thread / 16) + p, columns column + 8 * (thread % 16) + i.
template <bool kWide, typename T>
__device__ __forceinline__ void LoadTile(const T *x, int64_t stride, int first, int last, int column, int width, float (&v)[8][8])
{
    const int r0 = first + 8 * (int(threadIdx.x) / 16), c = column + 8 * (int(threadIdx.x) % 16);
#pragma unroll
    for (int p = 0; p < 8; p++) {
        // (rows behind the last one: no column is within their width)
        LoadPart<kWide, 8>(x + int64_t(r0 + p) * stride, c, r0 + p < last ? width : 0, v[p]);
    }
}

// Writes the transposed tile: to[(column + c) * pitch + at + ...] for the columns within the width.
__device__ __forceinline__ void StoreTransposed(const uint8_t *tile, uint8_t *to, int64_t pitch, int64_t at, int column, int width)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int piece = int(threadIdx.x) + i * kThreads, c = piece / 8, b = piece % 8 * 16;
        if (column + c < width) {
            *reinterpret_cast<Word4 *>(to + int64_t(column + c) * pitch + at + b) = *reinterpret_cast<const Word4 *>(tile + TransposedAt(c, b / 8));
        }
    }
}

// One unit of 128 rows by 128 columns: a scale for every column.
template <typename T, HcclAmdScaleType kScale, bool kWide>
__global__ void __launch_bounds__(kThreads) ColumnsKernel(TileArgs a)
{
    __shared__ __align__(16) uint8_t tile[kTile * kPitch];
    __shared__ float tops[16][kTile + 1];
    const int tiles = (a.width + kTile - 1) / kTile;
    const int unit = int(blockIdx.x) / tiles, column = int(blockIdx.x) % tiles * kTile;   // the tiles of a unit's rows lie next to each other
    const Unit u = FindUnit(a.offsets, a.groups, a.rows, unit, kTile);
    if (u.group < 0) {
        return;
    }
    float v[8][8];
    LoadTile<kWide>(static_cast<const T *>(a.x), a.stride, u.first, u.last, column, a.width, v);
    const int rg = int(threadIdx.x) / 16, cg = int(threadIdx.x) % 16 * 8;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float top = 0.0f;
#pragma unroll
        for (int p = 0; p < 8; p++) {
            top = __builtin_fmaxf(top, FiniteSize(v[p][i]));
        }
        tops[rg][cg + i] = top;
    }
    __syncthreads();
    if (threadIdx.x < kTile) {
        const int c = int(threadIdx.x);
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            top = __builtin_fmaxf(top, tops[i][c]);
        }
        const BlockScale<kScale> scale(top);
        tops[0][c] = scale.times;
        if (column + c < a.width) {
            static_cast<typename BlockScale<kScale>::Stored *>(a.scalesT)[int64_t(unit) * a.width + column + c] = scale.stored;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float times = tops[0][cg + i];
        float s[8];
#pragma unroll
        for (int p = 0; p < 8; p++) {
            s[p] = Scaled8(v[p][i], times);
        }
        *reinterpret_cast<Word2 *>(tile + TransposedAt(cg + i, rg)) = Word2{Quantise4(s[0], s[1], s[2], s[3]), Quantise4(s[4], s[5], s[6], s[7])};
    }
    __syncthreads();
    StoreTransposed(tile, static_cast<uint8_t *>(a.qT), a.pitchT, int64_t(unit) * kTile, column, a.width);
}

// One block of an expert's weights: a scale for all of it.
template <typename T, HcclAmdScaleType kScale, bool kWide>
__global__ void __launch_bounds__(kThreads) WeightsKernel(TileArgs a)
{
    typedef typename BlockScale<kScale>::Stored Stored;
    __shared__ __align__(16) uint8_t tile[kTile * kPitch];
    __shared__ float tops[kThreads / 64];
    const int nb = (a.rows + kTile - 1) / kTile, kb = (a.width + kTile - 1) / kTile;
    const int64_t block = blockIdx.x;
    const int b = int(block % kb), row = int(block / kb % nb);
    const int64_t expert = block / kb / nb;
    float v[8][8];
    LoadTile<kWide>(static_cast<const T *>(a.x) + expert * a.rows * a.stride, a.stride, row * kTile, a.rows, b * kTile, a.width, v);
    float top = 0.0f;
#pragma unroll
    for (int p = 0; p < 8; p++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            top = __builtin_fmaxf(top, FiniteSize(v[p][i]));
        }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        top = __builtin_fmaxf(top, __shfl_xor(top, d, 64));
    }
    if (threadIdx.x % 64 == 0) {
        tops[threadIdx.x / 64] = top;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; i++) {
        top = __builtin_fmaxf(top, tops[i]);
    }
    const BlockScale<kScale> scale(top);
    if (threadIdx.x == 0) {
        if (a.q != nullptr) {
            static_cast<Stored *>(a.scales)[(expert * nb + row) * kb + b] = scale.stored;
        }
        if (a.qT != nullptr) {
            static_cast<Stored *>(a.scalesT)[(expert * kb + b) * nb + row] = scale.stored;
        }
    }
    const int rg = int(threadIdx.x) / 16, cg = int(threadIdx.x) % 16 * 8;
#pragma unroll
    for (int p = 0; p < 8; p++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[p][i] = Scaled8(v[p][i], scale.times);
        }
        const int r = row * kTile + rg * 8 + p;
        if (a.q != nullptr && r < a.rows) {
            *reinterpret_cast<Word2 *>(static_cast<uint8_t *>(a.q) + (expert * a.rows + r) * (int64_t(kb) * kTile) + b * kTile + cg) =
                Word2{Quantise4(v[p][0], v[p][1], v[p][2], v[p][3]), Quantise4(v[p][4], v[p][5], v[p][6], v[p][7])};
        }
    }
    if (a.qT == nullptr) {
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        *reinterpret_cast<Word2 *>(tile + TransposedAt(cg + i, rg)) =
            Word2{Quantise4(v[0][i], v[1][i], v[2][i], v[3][i]), Quantise4(v[4][i], v[5][i], v[6][i], v[7][i])};
    }
    __syncthreads();
    StoreTransposed(tile, static_cast<uint8_t *>(a.qT) + expert * a.width * a.pitchT, a.pitchT, int64_t(row) * kTile, b * kTile, a.width);
}

// f(type, scale type, whether 16 bytes can be loaded at once), as constants
template <typename F>
HcclResult Choose(HcclDataType type, HcclAmdScaleType scaleType, bool wide, F f)
{
    const auto byWide = [&](auto of, auto scale) {
        return wide ? f(of, scale, std::true_type{}) : f(of, scale, std::false_type{});
    };
    const auto byScale = [&](auto of) {
        return scaleType == HCCL_AMD_SCALE_FP32 ? byWide(of, std::integral_constant<HcclAmdScaleType, HCCL_AMD_SCALE_FP32>{})
                                                : byWide(of, std::integral_constant<HcclAmdScaleType, HCCL_AMD_SCALE_E8M0>{});
    };
    switch (type) {
        case HCCL_DATA_TYPE_FP32:
            return byScale(float{});
        case HCCL_DATA_TYPE_FP16:
            return byScale(_Float16{});
        default:
            return byScale(__bf16{});
    }
}

}  // namespace
}  // namespace experts
}  // namespace hcclamd

using namespace hcclamd::experts;

extern "C" {

HcclResult HcclAmdBlockQuantWeights(const void *w, HcclDataType type, uint32_t experts, uint64_t n, uint64_t k, uint64_t wStride,
    HcclAmdScaleType scaleType, void *q, void *scales, void *qT, void *scalesT, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK_TYPE(Scaled(scaleType));
    EXPERTS_CHK(experts <= HCCL_AMD_MAX_GROUPS && n <= kMaxSize - 256 && k <= kMaxSize - 256);
    if (experts == 0 || n == 0 || k == 0 || (q == nullptr && qT == nullptr)) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(w);
    if (q != nullptr) {
        EXPERTS_CHK_PTR(scales);
    }
    if (qT != nullptr) {
        EXPERTS_CHK_PTR(scalesT);
    }
    EXPERTS_CHK(Stride(wStride, k));
    EXPERTS_CHK(AlignedTo(type, w) && Aligned(q, 16) && Aligned(qT, 16) && ScaleAligned(scaleType, scales) && ScaleAligned(scaleType, scalesT));
    EXPERTS_CHK(Blocks(n) * Blocks(k) * experts <= (uint64_t(1) << 23));   // workgroups of 256 below 2^32 threads
    TileArgs a{};
    a.x = w;
    a.q = q;
    a.scales = scales;
    a.qT = qT;
    a.scalesT = scalesT;
    a.stride = int64_t(wStride == 0 ? k : wStride);
    a.pitchT = int64_t(Up128(n));
    a.rows = int(n);
    a.width = int(k);
    const bool wide = k % 8 == 0 && Aligned(w, 16) && uint64_t(a.stride) * SizeOf(type) % 16 == 0;
    return Choose(type, scaleType, wide, [&](auto of, auto scale, auto is) {
        return Launch("HcclAmdBlockQuantWeights", WeightsKernel<decltype(of), decltype(scale)::value, decltype(is)::value>,
            uint32_t(Blocks(n) * Blocks(k) * experts), kThreads, 0, static_cast<hipStream_t>(stream), a);
    });
}

HcclResult HcclAmdBlockQuantColumns(const void *x, HcclDataType type, uint64_t rows, uint64_t width, uint64_t xStride,
    uint32_t groups, const int32_t *offsets, HcclAmdScaleType scaleType, void *qT, uint64_t columns, void *scales, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK_TYPE(Scaled(scaleType));
    EXPERTS_CHK(rows <= kMaxGroupedRows && width <= kMaxSize - 256);
    EXPERTS_CHK(groups >= 1 && groups <= HCCL_AMD_MAX_GROUPS);
    EXPERTS_CHK(offsets != nullptr || groups == 1);
    EXPERTS_CHK(columns % 128 == 0 && columns >= (rows / 128 + groups) * 128 && columns <= kMaxSize);
    if (rows == 0 || width == 0) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(x);
    EXPERTS_CHK_PTR(qT);
    EXPERTS_CHK_PTR(scales);
    EXPERTS_CHK(Stride(xStride, width));
    EXPERTS_CHK(AlignedTo(type, x) && Aligned(qT, 16) && ScaleAligned(scaleType, scales) && Aligned(offsets, 4));
    const uint64_t units = rows / 128 + groups;
    EXPERTS_CHK(Blocks(width) * units <= (uint64_t(1) << 23));
    TileArgs a{};
    a.x = x;
    a.offsets = offsets;
    a.qT = qT;
    a.scalesT = scales;
    a.stride = int64_t(xStride == 0 ? width : xStride);
    a.pitchT = int64_t(columns);
    a.rows = int(rows);
    a.width = int(width);
    a.groups = int(groups);
    const bool wide = width % 8 == 0 && Aligned(x, 16) && uint64_t(a.stride) * SizeOf(type) % 16 == 0;
    return Choose(type, scaleType, wide, [&](auto of, auto scale, auto is) {
        return Launch("HcclAmdBlockQuantColumns", ColumnsKernel<decltype(of), decltype(scale)::value, decltype(is)::value>,
            uint32_t(Blocks(width) * units), kThreads, 0, static_cast<hipStream_t>(stream), a);
    });
}

}  // extern "C"
