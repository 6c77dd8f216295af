// What stands between an expert's two products, and its gradient: HcclAmdExpertGate, HcclAmdExpertGateGrad.
//
// With t = 1 / (1 + exp(-g)):   a = g t u      dg = da u t (1 + g (1 - t))      du = da g t
//
// A wave takes a row's piece of 512 values, eight neighbouring ones to a lane: 16 lanes hold a block of an 8-bit row.  Every value is read once and
// written once, and bytes moved bound both kernels: 65536 rows of 2048 values to 8 bits (0.67 GB) 113 us, 5.9 TB/s, where a large copy reaches 5.15; 14769 rows of
// 4095, off every boundary, 70 us (4.3 TB/s), their gradient 127 us (5.7 TB/s).
#include <type_traits>

#include "sums.h"

namespace hcclamd {
namespace experts {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kEach = 8;
constexpr int kPiece = 64 * kEach;
constexpr int64_t kMostBlocks = int64_t(1) << 22;

struct GateArgs {
    const void *h, *aGrad;
    const int32_t *used;
    void *out, *scales;        // a, in its type or in 8 bits
    void *hGrad;
    int64_t hStride, aGradStride, outStride, scaleStride, hGradStride;
    int64_t rows;
    int width, padded, pieces;
};

__device__ __forceinline__ int64_t Rows(const GateArgs &a)
{
    return a.used == nullptr ? a.rows : min(int64_t(max(a.used[0], 0)), a.rows);
}

// t = 1 / (1 + exp(-g)) and 1 - t.  What rounding loses of the power's argument comes back as a factor; the power and the reciprocal are the hardware's, a unit
// each.  t is within 3.7 * 2^-24 of itself (16 million g from -80 to 8; 0.65 to 0.9 on average, with a library's power and a quotient 2.7 and 0.65; one more step
// for the reciprocal, and exp(-|g|) so that nothing overflows, do not get it closer where g is negative, and cost 6 % of 65536 rows).  Below g = -87, where t is less than
// 2^-126, it may be 0; beyond 10000 the power is infinite or 0 whatever its argument loses.
struct Sigmoid {
    float t, rest;
    __device__ __forceinline__ explicit Sigmoid(float g)
    {
        const float x = __builtin_amdgcn_fmed3f(g, -10000.0f, 10000.0f), y = x * -0x1.715476p+0f;
        const float lost = __builtin_fmaf(x, -0x1.4ae0cp-26f, __builtin_fmaf(x, -0x1.715476p+0f, -y));      // log2(e) in two parts
        const float p = __builtin_amdgcn_exp2f(y), factor = __builtin_fmaf(lost, 0x1.62e43p-1f, 1.0f);
        t = __builtin_amdgcn_rcpf(__builtin_fmaf(p, factor, 1.0f));
        rest = g > 0.0f ? p * factor * t : 1.0f - t;      // (next to t = 1 the difference has lost what g multiplies it by: 18 * 2^-24 of the gradient at g = 17)
    }
};

template <typename T, HcclAmdScaleType kScale, bool kWide>
__global__ void __launch_bounds__(kThreads) GateKernel(GateArgs a)
{
    const int64_t waves = Rows(a) * a.pieces;
    for (int64_t w = int64_t(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64); w < waves; w += int64_t(gridDim.x) * kWaves) {
        const int64_t row = w / a.pieces;
        const int at = int(w % a.pieces) * kPiece + int(threadIdx.x % 64) * kEach;
        const T *h = static_cast<const T *>(a.h) + row * a.hStride;
        T gates[kEach], ups[kEach];
        Fetch<kWide, kEach>(h, at, a.width, gates);
        Fetch<kWide, kEach>(h + a.width, at, a.width, ups);
        float g[kEach], u[kEach];
        Settle<kWide, kEach>(gates, at, a.width, g);
        Settle<kWide, kEach>(ups, at, a.width, u);
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            u[i] *= g[i] * Sigmoid(g[i]).t;
        }
        if constexpr (kScale == HCCL_AMD_SCALE_NONE) {
            StorePart<kWide, kEach>(static_cast<T *>(a.out) + row * a.outStride, at, a.width, u);
        } else {
            typename BlockScale<kScale>::Stored scale;
            const Word2 q = QuantiseBlock<kScale>(u, scale);
            if (at < a.padded) {
                *reinterpret_cast<Word2 *>(static_cast<uint8_t *>(a.out) + row * a.outStride + at) = q;
                if (threadIdx.x % 16 == 0) {
                    static_cast<typename BlockScale<kScale>::Stored *>(a.scales)[row * a.scaleStride + at / 128] = scale;
                }
            }
        }
    }
}

template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads) GateGradKernel(GateArgs a)
{
    const int64_t waves = Rows(a) * a.pieces;
    for (int64_t w = int64_t(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64); w < waves; w += int64_t(gridDim.x) * kWaves) {
        const int64_t row = w / a.pieces;
        const int at = int(w % a.pieces) * kPiece + int(threadIdx.x % 64) * kEach;
        const T *h = static_cast<const T *>(a.h) + row * a.hStride;
        T gates[kEach], ups[kEach], grads[kEach] = {};
        Fetch<kWide, kEach>(h, at, a.width, gates);
        Fetch<kWide, kEach>(h + a.width, at, a.width, ups);
        if (a.hGrad != nullptr) {
            Fetch<kWide, kEach>(static_cast<const T *>(a.aGrad) + row * a.aGradStride, at, a.width, grads);
        }
        float g[kEach], u[kEach], d[kEach];
        Settle<kWide, kEach>(gates, at, a.width, g);
        Settle<kWide, kEach>(ups, at, a.width, u);
        Settle<kWide, kEach>(grads, at, a.width, d);
        float v[kEach], dg[kEach], du[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const Sigmoid s(g[i]);
            const float gt = g[i] * s.t;
            v[i] = gt * u[i];
            dg[i] = d[i] * u[i] * (s.t * (1.0f + g[i] * s.rest));
            du[i] = d[i] * gt;
        }
        if (a.out != nullptr) {
            StorePart<kWide, kEach>(static_cast<T *>(a.out) + row * a.outStride, at, a.width, v);
        }
        if (a.hGrad != nullptr) {
            T *to = static_cast<T *>(a.hGrad) + row * a.hGradStride;
            StorePart<kWide, kEach>(to, at, a.width, dg);
            StorePart<kWide, kEach>(to + a.width, at, a.width, du);
        }
    }
}

template <typename F>
HcclResult ByType(HcclDataType type, F f)
{
    return type == HCCL_DATA_TYPE_FP32 ? f(float{}) : type == HCCL_DATA_TYPE_FP16 ? f(_Float16{}) : f(__bf16{});
}

// Whether rows at p can be taken 16 bytes at a time.
bool Wide(HcclDataType type, const void *p, int64_t stride) { return p == nullptr || (Aligned(p, 16) && uint64_t(stride) * SizeOf(type) % 16 == 0); }

int64_t Between(uint64_t stride, uint64_t width) { return int64_t(stride == 0 ? width : stride); }

uint32_t BlocksOf(int64_t rows, int pieces)
{
    const int64_t blocks = (rows * pieces + kWaves - 1) / kWaves;
    return uint32_t(blocks < kMostBlocks ? blocks : kMostBlocks);
}

constexpr uint64_t kMaxWidth = kMaxSize / 2 - 4096;   // both halves of a row's columns fit 32 bits

}  // namespace
}  // namespace experts
}  // namespace hcclamd

using namespace hcclamd::experts;

extern "C" {

HcclResult HcclAmdExpertGate(const void *h, HcclDataType type, uint64_t rows, uint64_t width, uint64_t hStride, const int32_t *used,
    HcclAmdScaleType scaleType, void *out, uint64_t outStride, void *scales, uint64_t scaleStride, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK_TYPE(scaleType == HCCL_AMD_SCALE_NONE || Scaled(scaleType));
    EXPERTS_CHK(rows <= kMaxSize && width <= kMaxWidth);
    if (rows == 0 || width == 0) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(h);
    EXPERTS_CHK_PTR(out);
    EXPERTS_CHK(Stride(hStride, 2 * width));
    EXPERTS_CHK(AlignedTo(type, h) && Aligned(used, 4));
    GateArgs a{};
    a.h = h;
    a.used = used;
    a.out = out;
    a.hStride = Between(hStride, 2 * width);
    a.rows = int64_t(rows);
    a.width = int(width);
    a.padded = int(Up128(width));
    a.pieces = (a.padded + kPiece - 1) / kPiece;
    bool wide = width % kEach == 0 && Wide(type, h, a.hStride);
    if (scaleType == HCCL_AMD_SCALE_NONE) {
        EXPERTS_CHK(Stride(outStride, width));
        EXPERTS_CHK(AlignedTo(type, out));
        a.outStride = Between(outStride, width);
        wide = wide && Wide(type, out, a.outStride);
    } else {
        EXPERTS_CHK_PTR(scales);
        EXPERTS_CHK(Stride(outStride, Up128(width)) && outStride % 16 == 0 && Aligned(out, 16));
        EXPERTS_CHK(Stride(scaleStride, Blocks(width)) && ScaleAligned(scaleType, scales));
        a.outStride = Between(outStride, Up128(width));
        a.scales = scales;
        a.scaleStride = Between(scaleStride, Blocks(width));
    }
    return ByType(type, [&](auto of) {
        typedef decltype(of) T;
        const auto go = [&](auto kernel) { return Launch("HcclAmdExpertGate", kernel, BlocksOf(a.rows, a.pieces), kThreads, 0, static_cast<hipStream_t>(stream), a); };
        switch (scaleType) {
            case HCCL_AMD_SCALE_FP32:
                return wide ? go(GateKernel<T, HCCL_AMD_SCALE_FP32, true>) : go(GateKernel<T, HCCL_AMD_SCALE_FP32, false>);
            case HCCL_AMD_SCALE_E8M0:
                return wide ? go(GateKernel<T, HCCL_AMD_SCALE_E8M0, true>) : go(GateKernel<T, HCCL_AMD_SCALE_E8M0, false>);
            default:
                return wide ? go(GateKernel<T, HCCL_AMD_SCALE_NONE, true>) : go(GateKernel<T, HCCL_AMD_SCALE_NONE, false>);
        }
    });
}

HcclResult HcclAmdExpertGateGrad(const void *aGrad, uint64_t aGradStride, const void *h, HcclDataType type, uint64_t rows, uint64_t width,
    uint64_t hStride, const int32_t *used, void *hGrad, uint64_t hGradStride, void *aOut, uint64_t aStride, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(type));
    EXPERTS_CHK(rows <= kMaxSize && width <= kMaxWidth);
    if (rows == 0 || width == 0 || (hGrad == nullptr && aOut == nullptr)) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(h);
    if (hGrad != nullptr) {
        EXPERTS_CHK_PTR(aGrad);
    }
    EXPERTS_CHK(Stride(hStride, 2 * width) && Stride(hGradStride, 2 * width) && Stride(aGradStride, width) && Stride(aStride, width));
    EXPERTS_CHK(AlignedTo(type, h) && AlignedTo(type, aGrad) && AlignedTo(type, hGrad) && AlignedTo(type, aOut) && Aligned(used, 4));
    GateArgs a{};
    a.h = h;
    a.aGrad = aGrad;
    a.used = used;
    a.out = aOut;
    a.hGrad = hGrad;
    a.hStride = Between(hStride, 2 * width);
    a.hGradStride = Between(hGradStride, 2 * width);
    a.aGradStride = Between(aGradStride, width);
    a.outStride = Between(aStride, width);
    EXPERTS_CHK((hGrad != h || a.hGradStride == a.hStride) && (aOut == nullptr || aOut != aGrad || a.outStride == a.aGradStride));
    a.rows = int64_t(rows);
    a.width = int(width);
    a.pieces = int((width + kPiece - 1) / kPiece);
    const bool wide = width % kEach == 0 && Wide(type, h, a.hStride) && Wide(type, aGrad, a.aGradStride) && Wide(type, hGrad, a.hGradStride) &&
        Wide(type, aOut, a.outStride);
    return ByType(type, [&](auto of) {
        typedef decltype(of) T;
        return Launch("HcclAmdExpertGateGrad", wide ? GateGradKernel<T, true> : GateGradKernel<T, false>, BlocksOf(a.rows, a.pieces), kThreads, 0,
            static_cast<hipStream_t>(stream), a);
    });
}

}  // extern "C"
