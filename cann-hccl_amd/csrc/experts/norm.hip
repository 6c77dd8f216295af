// Rows and their residual, normed by their root mean square (HcclAmdNormRows), in their type and as 8-bit rows, and the gradient.
//
// With r = (mean s^2 + epsilon)^-1/2, d = dy * gain and n = s r:
//   y = n * gain      dx = r (d - n mean(d n)) + dsum      dgain = sum over rows of dy * n
//
// Up to 8192 columns a row stays in registers between its sums and its results: read once, written once.  64 to 1024 threads to a row, each with eight neighbouring
// values (16 or 32 beyond 8192), so that a lane's accesses are 16 bytes and 16 lanes hold a block of an 8-bit row.  Sums are in 64 bits: a square of 32 bits is
// exact there, and no row overflows.
//
// Bytes moved bound them, where a large copy reaches 5.15 TB/s: 16384 rows of 8192 values with residual and sum (1.07 GB) 177 us, 6.0 TB/s, their gradient
// (1.07 GB) 199 us, 5.4 TB/s, the 5 us that add up the gain's included.  8192 rows of 4096 to 8 bits (0.24 GB) 50 us, 4.7 TB/s.  More values to a thread, fewer
// threads to a row were slower: 16 and 512 for rows of 8192 411 us in all instead of 383.  Rows of 2001 values, off every boundary (5003 of them):
// 13.7 us, 22 and 6; 16384 of them 102 us in all, of 2000 values 84.  One row of 8192: 4 us, the latency of loads, sums and a launch.
//
// Where something else bounds them (16 bits, residual and sum): rows that do not fill a wave's 512 columns, which pays for each of them whole: 262144 rows of 128 80 us, 3.4 TB/s, the
// gradient 133, 2.0, by vector instructions.  And rows that do not fit the registers: forward above 16384 columns (2 to 29 registers to scratch), gradient above 8192 (5 to 11 at 16384
// and 242 to 358 at 32768, 91 to 991 off boundaries), which then fetches no row ahead either: 2048 rows of 16384 49 us and 78 (5.5 and 3.5 TB/s), of 32768 105 and 381 (5.1 and
// 1.4), of 16383 61 and 143, of 32767 143 and 610.
#include <type_traits>

#include "sums.h"

namespace hcclamd {
namespace experts {
namespace {

constexpr int kEach = 8;     // neighbouring values of a lane

struct NormArgs {
    const void *x, *residual, *gain;
    void *sum, *y, *q, *scales;
    int64_t xStride, residualStride, sumStride, yStride, qStride, scaleStride;
    int64_t rows;
    int width, padded;
    float epsilon;
    bool gain32;               // gain is in 32 bits, else in the rows' type
    bool powers;               // the scales are powers of two
};

// A wave to a row: four rows to a workgroup.  More than one: a row to a workgroup, whose waves meet twice a row.
constexpr int BlockOf(int rowThreads) { return rowThreads == 64 ? 256 : rowThreads; }

// The sum of kWaves places, a power of two up to 16, on all lanes: each reads one, and they are added up as AddWave does.
template <int kWaves>
__device__ __forceinline__ double AddParts(const double *parts)
{
    double x = parts[threadIdx.x % kWaves];
    if constexpr (kWaves > 8) {
        x += Turned<8>(x);
    }
    if constexpr (kWaves > 4) {
        x += Turned<4>(x);
    }
    if constexpr (kWaves > 2) {
        x += Turned<2>(x);
    }
    return x + Turned<1>(x);
}

// The row's sum on all its threads.  `parts`: a place per wave, used by one call between two barriers.
template <int kRowThreads>
__device__ __forceinline__ double AddRow(double x, double *parts)
{
    x = AddWave(x);
    if constexpr (kRowThreads > 64) {
        if (threadIdx.x % 64 == 0) {
            parts[threadIdx.x / 64] = x;
        }
        __syncthreads();
        x = AddParts<kRowThreads / 64>(parts);
    }
    return x;
}

// gain[at ...], 1 where there is none.
template <int kHow, typename T>
__device__ __forceinline__ void LoadGain(const void *gain, bool gain32, int at, int width, float (&g)[kEach])
{
    if (gain == nullptr) {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            g[i] = 1.0f;
        }
    } else if (gain32) {
        float v[kEach];
        Fetch<kHow, kEach>(static_cast<const float *>(gain), at, width, v);
        Settle<kHow, kEach>(v, at, width, g);
    } else {
        T v[kEach];
        Fetch<kHow, kEach>(static_cast<const T *>(gain), at, width, v);
        Settle<kHow, kEach>(v, at, width, g);
    }
}

template <HcclAmdScaleType kScale>
__device__ __forceinline__ void StoreBlock(float (&v)[kEach], const NormArgs &a, int64_t row, int at)
{
    typename BlockScale<kScale>::Stored scale;
    const Word2 q = QuantiseBlock<kScale>(v, scale);
    if (at < a.padded) {
        *reinterpret_cast<Word2 *>(static_cast<uint8_t *>(a.q) + row * a.qStride + at) = q;
        if (threadIdx.x % 16 == 0) {
            static_cast<typename BlockScale<kScale>::Stored *>(a.scales)[row * a.scaleStride + at / 128] = scale;
        }
    }
}

// kRowThreads threads to a row, each with kChunks times eight values.
template <typename T, int kRowThreads, int kChunks, bool kEight, int kHow>
__global__ void __launch_bounds__(BlockOf(kRowThreads)) NormKernel(NormArgs a)
{
    constexpr int kRows = BlockOf(kRowThreads) / kRowThreads;
    __shared__ double parts[kRowThreads / 64];
    const int l = int(threadIdx.x) % kRowThreads;
    for (int64_t row = int64_t(blockIdx.x) * kRows + int(threadIdx.x) / kRowThreads; row < a.rows; row += int64_t(gridDim.x) * kRows) {
        float s[kChunks][kEach], g[kChunks][kEach];
        {
            T x[kChunks][kEach], r[kChunks][kEach];
#pragma unroll
            for (int c = 0; c < kChunks; c++) {
                Fetch<kHow, kEach>(static_cast<const T *>(a.x) + row * a.xStride, (c * kRowThreads + l) * kEach, a.width, x[c]);
            }
            if (a.residual != nullptr) {
#pragma unroll
                for (int c = 0; c < kChunks; c++) {
                    Fetch<kHow, kEach>(static_cast<const T *>(a.residual) + row * a.residualStride, (c * kRowThreads + l) * kEach, a.width, r[c]);
                }
            }
#pragma unroll
            for (int c = 0; c < kChunks; c++) {
                Settle<kHow, kEach>(x[c], (c * kRowThreads + l) * kEach, a.width, s[c]);
                if (a.residual != nullptr) {
                    float v[kEach];
                    Settle<kHow, kEach>(r[c], (c * kRowThreads + l) * kEach, a.width, v);
#pragma unroll
                    for (int i = 0; i < kEach; i++) {
                        s[c][i] += v[i];
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            LoadGain<kHow, T>(a.gain, a.gain32, (c * kRowThreads + l) * kEach, a.width, g[c]);
        }
        double squares[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            squares[c] = 0.0;
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                squares[c] = __builtin_fma(double(s[c][i]), double(s[c][i]), squares[c]);
            }
        }
        if (a.sum != nullptr) {
#pragma unroll
            for (int c = 0; c < kChunks; c++) {
                StorePart<kHow, kEach>(static_cast<T *>(a.sum) + row * a.sumStride, (c * kRowThreads + l) * kEach, a.width, s[c]);
            }
        }
        double all = squares[0];
#pragma unroll
        for (int c = 1; c < kChunks; c++) {
            all += squares[c];
        }
        all = AddRow<kRowThreads>(all, parts);
        const float by = float(1.0 / __builtin_sqrt(all / double(a.width) + double(a.epsilon)));
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            const int at = (c * kRowThreads + l) * kEach;
            float v[kEach];
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                v[i] = s[c][i] * by * g[c][i];
            }
            if (a.y != nullptr) {
                StorePart<kHow, kEach>(static_cast<T *>(a.y) + row * a.yStride, at, a.width, v);
            }
            if constexpr (kEight) {
#pragma unroll
                for (int i = 0; i < kEach; i++) {
                    // (behind the row's end a gain of 1 may meet an infinite factor)
                    v[i] = kHow == kAligned ? (at < a.width ? v[i] : 0.0f) : (at + i < a.width ? v[i] : 0.0f);
                }
                if (a.powers) {
                    StoreBlock<HCCL_AMD_SCALE_E8M0>(v, a, row, at);
                } else {
                    StoreBlock<HCCL_AMD_SCALE_FP32>(v, a, row, at);
                }
            }
        }
        if constexpr (kRowThreads > 64) {
            __syncthreads();     // before the next row's sums
        }
    }
}

struct NormGradArgs {
    const void *yGrad, *sum, *gain, *sumGrad;
    void *xGrad;
    float *partial;            // [workgroups][width]: sums over a workgroup's rows of dy * n; null: not wanted
    int64_t yGradStride, sumStride, sumGradStride, xGradStride;
    int64_t rows;
    int width;
    float epsilon;
    bool gain32;
};

// A workgroup goes through rows and keeps what they add to the gain's gradient in registers, in 64 bits where these have room (one chunk: 198 us for 16384 rows of
// 8192 instead of 195), rounds it to 32 bits once and leaves it for NormGainKernel: with all sums in 32 bits a gradient of terms of one sign was up to 7 * 2^-24 off and
// 2.0 on average, now 0.9 and 0.4, most of it the result's own rounding.
template <typename T, int kRowThreads, int kChunks, int kHow>
__global__ void __launch_bounds__(BlockOf(kRowThreads)) NormGradKernel(NormGradArgs a)
{
    constexpr int kRows = BlockOf(kRowThreads) / kRowThreads;
    __shared__ double parts[2][kRowThreads / 64];
    __shared__ float sums[kRows > 1 ? kRows : 1][kRows > 1 ? kRowThreads * kChunks * kEach : 1];
    const int l = int(threadIdx.x) % kRowThreads, slot = int(threadIdx.x) / kRowThreads;
    typedef std::conditional_t<kChunks == 1, double, float> Sum;
    float gain[kChunks][kEach];
    Sum more[kChunks][kEach];
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
        LoadGain<kHow, T>(a.gain, a.gain32, (c * kRowThreads + l) * kEach, a.width, gain[c]);
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            more[c][i] = 0;
        }
    }
    const int64_t step = int64_t(gridDim.x) * kRows;
    int64_t row = int64_t(blockIdx.x) * kRows + slot;
    T nextD[kChunks][kEach], nextS[kChunks][kEach];
    const auto load = [&]() {
        if (row < a.rows) {
#pragma unroll
            for (int c = 0; c < kChunks; c++) {
                Fetch<kHow, kEach>(static_cast<const T *>(a.yGrad) + row * a.yGradStride, (c * kRowThreads + l) * kEach, a.width, nextD[c]);
                Fetch<kHow, kEach>(static_cast<const T *>(a.sum) + row * a.sumStride, (c * kRowThreads + l) * kEach, a.width, nextS[c]);
            }
        }
    };
    load();
    while (row < a.rows) {
        float d[kChunks][kEach], s[kChunks][kEach];
        T arrived[kChunks][kEach];
        double squares = 0.0, dots = 0.0;
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            Settle<kHow, kEach>(nextD[c], (c * kRowThreads + l) * kEach, a.width, d[c]);
            Settle<kHow, kEach>(nextS[c], (c * kRowThreads + l) * kEach, a.width, s[c]);
        }
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            if (a.sumGrad != nullptr) {
                Fetch<kHow, kEach>(static_cast<const T *>(a.sumGrad) + row * a.sumGradStride, (c * kRowThreads + l) * kEach, a.width, arrived[c]);
            }
        }
        const int64_t here = row;
        row += step;
        if constexpr (kChunks == 1) {
            load();       // the next row is on its way while this one is summed up (more chunks leave no registers for that)
        }
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                squares = __builtin_fma(double(s[c][i]), double(s[c][i]), squares);
                dots = __builtin_fma(double(d[c][i] * gain[c][i]), double(s[c][i]), dots);
            }
        }
        squares = AddWave(squares);
        dots = AddWave(dots);
        if constexpr (kRowThreads > 64) {
            if (threadIdx.x % 64 == 0) {
                parts[0][threadIdx.x / 64] = squares;
                parts[1][threadIdx.x / 64] = dots;
            }
            __syncthreads();
            squares = AddParts<kRowThreads / 64>(parts[0]);
            dots = AddParts<kRowThreads / 64>(parts[1]);
        }
        const double length = 1.0 / __builtin_sqrt(squares / double(a.width) + double(a.epsilon));
        const float by = float(length), mean = float(dots * length / double(a.width));
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            const int at = (c * kRowThreads + l) * kEach;
            float out[kEach], other[kEach] = {};
            if (a.sumGrad != nullptr) {
                Settle<kHow, kEach>(arrived[c], at, a.width, other);
            }
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                const float n = s[c][i] * by;
                more[c][i] += Sum(d[c][i] * n);
                out[i] = by * (d[c][i] * gain[c][i] - n * mean) + other[i];
            }
            if (a.xGrad != nullptr) {
                StorePart<kHow, kEach>(static_cast<T *>(a.xGrad) + here * a.xGradStride, at, a.width, out);
            }
        }
        if constexpr (kRowThreads > 64) {
            __syncthreads();     // before the next row's sums
        }
        if constexpr (kChunks > 1) {
            load();
        }
    }
    if (a.partial == nullptr) {
        return;
    }
    if constexpr (kRows > 1) {
        // the waves' sums, one behind the other
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                sums[slot][(c * kRowThreads + l) * kEach + i] = float(more[c][i]);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.width; i += BlockOf(kRowThreads)) {
            float all = sums[0][i];
#pragma unroll
            for (int k = 1; k < kRows; k++) {
                all += sums[k][i];
            }
            a.partial[int64_t(blockIdx.x) * a.width + i] = all;
        }
    } else {
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            StorePart<kAnyhow, kEach>(a.partial + int64_t(blockIdx.x) * a.width, (c * kRowThreads + l) * kEach, a.width, more[c]);
        }
    }
}

constexpr int kGainCols = 16, kGainRuns = 64, kGainThreads = kGainCols * kGainRuns;

// gainGrad from the workgroups' sums, in 64 bits: 16 columns to a workgroup, 64 runs of workgroups to a column, then the runs in their order.
__global__ void __launch_bounds__(kGainThreads) NormGainKernel(const float *partial, int slots, int width, float *gainGrad, bool accumulate)
{
    __shared__ double parts[kGainRuns][kGainCols + 1];
    const int c = int(threadIdx.x) % kGainCols, run = int(threadIdx.x) / kGainCols, at = int(blockIdx.x) * kGainCols + c;
    double sum = 0.0;
    if (at < width) {
#pragma unroll 16
        for (int s = run; s < slots; s += kGainRuns) {
            sum += partial[int64_t(s) * width + at];
        }
    }
    parts[run][c] = sum;
    __syncthreads();
    if (run == 0 && at < width) {
        double all = accumulate ? double(gainGrad[at]) : 0.0;
#pragma unroll
        for (int i = 0; i < kGainRuns; i++) {
            all += parts[i][c];
        }
        gainGrad[at] = float(all);
    }
}

// f(threads to a row, times eight values of a thread), as constants
template <typename F>
HcclResult ByWidth(uint64_t width, F f)
{
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    typedef std::integral_constant<int, 4> Four;
    if (width <= 512) {
        return f(std::integral_constant<int, 64>{}, One{});
    }
    if (width <= 1024) {
        return f(std::integral_constant<int, 128>{}, One{});
    }
    if (width <= 2048) {
        return f(std::integral_constant<int, 256>{}, One{});
    }
    if (width <= 4096) {
        return f(std::integral_constant<int, 512>{}, One{});
    }
    if (width <= 8192) {
        return f(std::integral_constant<int, 1024>{}, One{});
    }
    return width <= 16384 ? f(std::integral_constant<int, 1024>{}, Two{}) : f(std::integral_constant<int, 1024>{}, Four{});
}

template <typename F>
HcclResult ByType(HcclDataType type, F f)
{
    return type == HCCL_DATA_TYPE_FP32 ? f(float{}) : type == HCCL_DATA_TYPE_FP16 ? f(_Float16{}) : f(__bf16{});
}

// Workgroups that go through rows: what makes 16 waves to a compute unit, each of which leaves sums of its own.  Twice as many took 126 us for the gradient of 262144 rows of 128
// (instead of 133), but 50 for 65536 of 512 (47), 64 for 32768 of 1024 (53), 56 for 16384 of 2048 (50), 108 of 4096 (105), 204 of 8192 (198); half as many 157, 51, 61, 59, 130, 350.
uint64_t GradBlocks(uint64_t rows, uint64_t width)
{
    const uint64_t each = width <= 512 ? 4 : 1, blocks = (rows + each - 1) / each;
    const uint64_t most = width <= 512 ? 1024 : width <= 1024 ? 2048 : width <= 2048 ? 1024 : width <= 4096 ? 512 : 256;
    return blocks < most ? blocks : most;
}

// Whether rows at p can be taken 16 bytes at a time.
bool Wide(HcclDataType type, const void *p, int64_t stride) { return p == nullptr || (Aligned(p, 16) && uint64_t(stride) * SizeOf(type) % 16 == 0); }

int64_t Between(uint64_t stride, uint64_t width) { return int64_t(stride == 0 ? width : stride); }

}  // namespace
}  // namespace experts
}  // namespace hcclamd

using namespace hcclamd::experts;

extern "C" {

HcclResult HcclAmdNormRows(const void *x, HcclDataType type, uint64_t rows, uint64_t width, uint64_t xStride, const void *residual,
    uint64_t residualStride, const void *gain, HcclDataType gainType, float epsilon, void *sum, uint64_t sumStride, void *y, uint64_t yStride,
    HcclAmdScaleType scaleType, void *q, uint64_t qStride, void *scales, uint64_t scaleStride, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK_TYPE(gain == nullptr || gainType == type || gainType == HCCL_DATA_TYPE_FP32);
    EXPERTS_CHK_TYPE(scaleType == HCCL_AMD_SCALE_NONE || Scaled(scaleType));
    EXPERTS_CHK(rows <= kMaxSize && width <= HCCL_AMD_MAX_NORM_WIDTH);
    EXPERTS_CHK(epsilon >= 0.0f);
    if (rows == 0 || width == 0 || (sum == nullptr && y == nullptr && scaleType == HCCL_AMD_SCALE_NONE)) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(x);
    EXPERTS_CHK(Stride(xStride, width) && Stride(residualStride, width) && Stride(sumStride, width) && Stride(yStride, width));
    EXPERTS_CHK(AlignedTo(type, x) && AlignedTo(type, residual) && AlignedTo(type, sum) && AlignedTo(type, y));
    EXPERTS_CHK(gain == nullptr || AlignedTo(gainType, gain));
    NormArgs a{};
    a.x = x;
    a.residual = residual;
    a.gain = gain;
    a.sum = sum;
    a.y = y;
    a.xStride = Between(xStride, width);
    a.residualStride = Between(residualStride, width);
    a.sumStride = Between(sumStride, width);
    a.yStride = Between(yStride, width);
    a.rows = int64_t(rows);
    a.width = int(width);
    a.padded = int(Up128(width));
    a.epsilon = epsilon;
    a.gain32 = gainType == HCCL_DATA_TYPE_FP32;
    EXPERTS_CHK(sum == nullptr || ((sum != x || a.sumStride == a.xStride) && (sum != residual || a.sumStride == a.residualStride)));
    const bool eight = scaleType != HCCL_AMD_SCALE_NONE;
    if (eight) {
        EXPERTS_CHK_PTR(q);
        EXPERTS_CHK_PTR(scales);
        EXPERTS_CHK(Stride(qStride, Up128(width)) && qStride % 16 == 0 && Aligned(q, 16));
        EXPERTS_CHK(Stride(scaleStride, Blocks(width)) && ScaleAligned(scaleType, scales));
        a.q = q;
        a.scales = scales;
        a.qStride = Between(qStride, Up128(width));
        a.scaleStride = Between(scaleStride, Blocks(width));
        a.powers = scaleType == HCCL_AMD_SCALE_E8M0;
    } else {
        EXPERTS_CHK(q == nullptr && scales == nullptr);
    }
    const bool wide = width % kEach == 0 && Wide(type, x, a.xStride) && Wide(type, residual, a.residualStride) && Wide(type, sum, a.sumStride) &&
        Wide(type, y, a.yStride) && Aligned(gain, 16);
    return ByType(type, [&](auto of) {
        return ByWidth(width, [&](auto threads, auto chunks) {
            typedef decltype(of) T;
            constexpr int kThreads = decltype(threads)::value, kChunks = decltype(chunks)::value, kBlock = BlockOf(kThreads), kRows = kBlock / kThreads;
            const int64_t blocks = (a.rows + kRows - 1) / kRows;
            const auto go = [&](auto kernel) {
                return Launch("HcclAmdNormRows", kernel, uint32_t(blocks < (1 << 20) ? blocks : 1 << 20), kBlock, 0, static_cast<hipStream_t>(stream), a);
            };
            return eight ? (wide ? go(NormKernel<T, kThreads, kChunks, true, kAligned>) : go(NormKernel<T, kThreads, kChunks, true, kAnyhow>))
                         : (wide ? go(NormKernel<T, kThreads, kChunks, false, kAligned>) : go(NormKernel<T, kThreads, kChunks, false, kAnyhow>));
        });
    });
}

HcclResult HcclAmdNormRowsGradWorkspace(uint64_t rows, uint64_t width, uint64_t *bytes)
{
    EXPERTS_CHK_PTR(bytes);
    EXPERTS_CHK(rows <= kMaxSize && width <= HCCL_AMD_MAX_NORM_WIDTH);
    *bytes = GradBlocks(rows, width) * width * sizeof(float);
    return HCCL_SUCCESS;
}

HcclResult HcclAmdNormRowsGrad(const void *yGrad, uint64_t yGradStride, const void *sum, HcclDataType type, uint64_t rows, uint64_t width,
    uint64_t sumStride, const void *gain, HcclDataType gainType, float epsilon, const void *sumGrad, uint64_t sumGradStride, void *xGrad,
    uint64_t xGradStride, float *gainGrad, uint32_t accumulate, void *workspace, uint64_t workspaceBytes, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK_TYPE(gain == nullptr || gainType == type || gainType == HCCL_DATA_TYPE_FP32);
    EXPERTS_CHK(rows <= kMaxSize && width <= HCCL_AMD_MAX_NORM_WIDTH);
    EXPERTS_CHK(epsilon >= 0.0f);
    if (width == 0 || (xGrad == nullptr && gainGrad == nullptr) || (rows == 0 && gainGrad == nullptr)) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK(Aligned(gainGrad, 4));
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const uint64_t blocks = GradBlocks(rows, width);
    if (rows != 0) {
        EXPERTS_CHK_PTR(yGrad);
        EXPERTS_CHK_PTR(sum);
        EXPERTS_CHK(Stride(yGradStride, width) && Stride(sumStride, width) && Stride(sumGradStride, width) && Stride(xGradStride, width));
        EXPERTS_CHK(AlignedTo(type, yGrad) && AlignedTo(type, sum) && AlignedTo(type, sumGrad) && AlignedTo(type, xGrad));
        EXPERTS_CHK(gain == nullptr || AlignedTo(gainType, gain));
        NormGradArgs a{};
        a.yGrad = yGrad;
        a.sum = sum;
        a.gain = gain;
        a.sumGrad = sumGrad;
        a.xGrad = xGrad;
        a.yGradStride = Between(yGradStride, width);
        a.sumStride = Between(sumStride, width);
        a.sumGradStride = Between(sumGradStride, width);
        a.xGradStride = Between(xGradStride, width);
        a.rows = int64_t(rows);
        a.width = int(width);
        a.epsilon = epsilon;
        a.gain32 = gainType == HCCL_DATA_TYPE_FP32;
        EXPERTS_CHK(xGrad == nullptr || ((xGrad != yGrad || a.xGradStride == a.yGradStride) && (xGrad != sumGrad || a.xGradStride == a.sumGradStride)));
        if (gainGrad != nullptr) {
            EXPERTS_CHK_PTR(workspace);
            EXPERTS_CHK(Aligned(workspace, 16));
            EXPERTS_CHK(workspaceBytes >= blocks * width * sizeof(float));
            a.partial = static_cast<float *>(workspace);
        }
        const bool wide = width % kEach == 0 && Wide(type, yGrad, a.yGradStride) && Wide(type, sum, a.sumStride) && Wide(type, sumGrad, a.sumGradStride) &&
            Wide(type, xGrad, a.xGradStride) && Aligned(gain, 16);
        const HcclResult r = ByType(type, [&](auto of) {
            return ByWidth(width, [&](auto threads, auto chunks) {
                typedef decltype(of) T;
                constexpr int kThreads = decltype(threads)::value, kChunks = decltype(chunks)::value;
                const auto go = [&](auto kernel) { return Launch("HcclAmdNormRowsGrad", kernel, uint32_t(blocks), BlockOf(kThreads), 0, on, a); };
                return wide ? go(NormGradKernel<T, kThreads, kChunks, kAligned>) : go(NormGradKernel<T, kThreads, kChunks, kAnyhow>);
            });
        });
        if (r != HCCL_SUCCESS || gainGrad == nullptr) {
            return r;
        }
    }
    return Launch("HcclAmdNormRowsGrad", NormGainKernel, uint32_t((width + kGainCols - 1) / kGainCols), kGainThreads, 0, on,
        static_cast<const float *>(workspace), int(blocks), int(width), gainGrad, accumulate != 0);
}

}  // extern "C"
