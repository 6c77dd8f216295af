// What the operators of an expert-parallel layer share: checks of arguments, element types, 8-bit blocks, the way from a
// workgroup's number to its group of rows.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "hccl/hccl_amd_experts.h"
#include "log.h"

namespace hcclamd {
namespace experts {

#define EXPERTS_CHK_PTR(p)                                      \
    do {                                                        \
        if ((p) == nullptr) {                                   \
            HCCL_LOG_ERROR("%s: %s is null", __func__, #p);     \
            return HCCL_E_PTR;                                  \
        }                                                       \
    } while (0)

#define EXPERTS_CHK(cond)                                       \
    do {                                                        \
        if (!(cond)) {                                          \
            HCCL_LOG_ERROR("%s: needs %s", __func__, #cond);    \
            return HCCL_E_PARA;                                 \
        }                                                       \
    } while (0)

#define EXPERTS_CHK_TYPE(cond)                                          \
    do {                                                                \
        if (!(cond)) {                                                  \
            HCCL_LOG_ERROR("%s: type not supported", __func__);         \
            return HCCL_E_NOT_SUPPORT;                                  \
        }                                                               \
    } while (0)

constexpr uint64_t kMaxSize = (uint64_t(1) << 31) - 1;    // tokens, rows, widths; products of them are held in 64 bits
constexpr uint64_t kMaxGroupedRows = uint64_t(1) << 28;   // rows that are cut into units group by group (FindUnit)

inline uint64_t Up128(uint64_t n) { return (n + 127) / 128 * 128; }
inline uint64_t Blocks(uint64_t n) { return (n + 127) / 128; }
inline bool Float(HcclDataType t) { return t == HCCL_DATA_TYPE_FP32 || t == HCCL_DATA_TYPE_FP16 || t == HCCL_DATA_TYPE_BFP16; }
inline uint64_t SizeOf(HcclDataType t) { return t == HCCL_DATA_TYPE_FP32 ? 4 : 2; }
// From one row to the next, in elements; 0: no gap.  Beyond 2^40 lies no memory, and a negative number taken for an unsigned one does.
inline bool Stride(uint64_t stride, uint64_t least) { return stride == 0 || (stride >= least && stride <= uint64_t(1) << 40); }
inline bool Scaled(HcclAmdScaleType s) { return s == HCCL_AMD_SCALE_FP32 || s == HCCL_AMD_SCALE_E8M0; }
inline bool Aligned(const void *p, uint64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
inline bool AlignedTo(HcclDataType t, const void *p) { return Aligned(p, SizeOf(t)); }
inline bool ScaleAligned(HcclAmdScaleType s, const void *p) { return s != HCCL_AMD_SCALE_FP32 || Aligned(p, 4); }

// The launch's own answer decides: the thread's last error may be of another call, which its caller has dealt with or has yet to see.
template <typename... P>
HcclResult Launch(const char *fn, void (*kernel)(P...), uint32_t blocks, int threads, size_t lds, hipStream_t stream, P... args)
{
    void *argv[] = {&args...};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3(blocks), dim3(uint32_t(threads)), argv, lds, stream);
    if (e == hipSuccess) {
        return HCCL_SUCCESS;
    }
    (void)hipGetLastError();   // reported here, not once more by whoever asks next
    HCCL_LOG_ERROR("%s: %s", fn, hipGetErrorString(e));
    return HCCL_E_RUNTIME;
}

// ---- element types ---------------------------------------------------------------------------------------

typedef float Float4 __attribute__((ext_vector_type(4)));
typedef int32_t Int4 __attribute__((ext_vector_type(4)));
typedef int32_t Int8 __attribute__((ext_vector_type(8)));
typedef uint32_t Word2 __attribute__((ext_vector_type(2)));
typedef uint32_t Word4 __attribute__((ext_vector_type(4)));

// N consecutive elements from p, in loads of 16 bytes (or one of all of them, if they are fewer).  kWide: p is aligned to that; else to
// an element, which the hardware takes too (a lane's load then touches one line more).  V: float, or T itself for bits as they are.
template <bool kWide, int N, typename T, typename V>
__device__ __forceinline__ void Load(const T *p, V (&v)[N])
{
    constexpr int kAlign = !kWide ? sizeof(T) : N * sizeof(T) < 16 ? N * sizeof(T) : 16;
    typedef T Vec __attribute__((ext_vector_type(N), aligned(kAlign)));
    const Vec x = *reinterpret_cast<const Vec *>(p);
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = V(x[i]);
    }
}

template <bool kWide, int N, typename T, typename V>
__device__ __forceinline__ void Store(T *p, const V (&v)[N])
{
    constexpr int kAlign = !kWide ? sizeof(T) : N * sizeof(T) < 16 ? N * sizeof(T) : 16;
    typedef T Vec __attribute__((ext_vector_type(N), aligned(kAlign)));
    Vec x;
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = T(v[i]);
    }
    *reinterpret_cast<Vec *>(p) = x;
}

// How a row can be taken, N elements at a time: anyhow, aligned and of a multiple of N elements, or such that the caller's lanes cover
// it exactly and no lane has to look.
constexpr int kAnyhow = 0, kAligned = 1, kExactly = 2;

// N elements from column `at` of a row of `width`, `fill` beyond it.
template <int kHow, int N, typename T, typename V>
__device__ __forceinline__ void LoadPart(const T *row, int at, int width, V (&v)[N], V fill = V(0))
{
    if constexpr (kHow == kExactly) {
        Load<true, N>(row + at, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = fill;
    }
    if (kHow == kAligned ? at < width : at + N <= width) {
        Load<kHow == kAligned, N>(row + at, v);
    } else if (kHow == kAnyhow && at < width) {
        for (int i = 0; i < N; i++) {
            if (at + i < width) {
                v[i] = V(row[at + i]);
            }
        }
    }
}

template <int kHow, int N, typename T, typename V>
__device__ __forceinline__ void StorePart(T *row, int at, int width, const V (&v)[N])
{
    if (kHow == kExactly) {
        Store<true, N>(row + at, v);
    } else if (kHow == kAligned ? at < width : at + N <= width) {
        Store<kHow == kAligned, N>(row + at, v);
    } else if (kHow == kAnyhow && at < width) {
        for (int i = 0; i < N; i++) {
            if (at + i < width) {
                row[at + i] = T(v[i]);
            }
        }
    }
}

// ---- 8-bit blocks --------------------------------------------------------------------------------------------

constexpr float kLeastMax = 0x1p-96f;
constexpr float kLargest = 448.0f;

// A value's part in its block's maximum: infinities and NaN have none.
__device__ __forceinline__ float FiniteSize(float v)
{
    const float a = __builtin_fabsf(v);
    return a < __builtin_inff() ? a : 0.0f;
}

// What a block's values are multiplied by, from its maximum, and its scale as it is stored.
template <HcclAmdScaleType kScale>
struct BlockScale;

template <>
struct BlockScale<HCCL_AMD_SCALE_FP32> {
    typedef float Stored;
    float times;
    float stored;
    __device__ __forceinline__ explicit BlockScale(float top)
    {
        top = top > kLeastMax ? top : kLeastMax;
        times = 1.0f / top * kLargest;
        stored = top * (1.0f / kLargest);
    }
};

template <>
struct BlockScale<HCCL_AMD_SCALE_E8M0> {
    typedef uint8_t Stored;
    float times;
    uint8_t stored;
    __device__ __forceinline__ explicit BlockScale(float top)
    {
        top = top > kLeastMax ? top : kLeastMax;
        // top = m * 2^p with m in [1, 2): 448 = 1.75 * 2^8, so the power is p - 8, one more where m > 1.75; the comparison
        // of the mantissa's bits rounds up by a carry
        const uint32_t bits = __float_as_uint(top) + 0x1fffffu;
        const int power = int(bits >> 23) - 127 - 8;
        times = __uint_as_float(uint32_t(127 - power) << 23);
        stored = uint8_t(power + 127);
    }
};

// Four values as four 8-bit ones, lowest byte first.  A scaled value is at most 448 * (1 + 2^-22), which rounds to 448.
__device__ __forceinline__ uint32_t Quantise4(float a, float b, float c, float d)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return uint32_t(w);
}

// Infinities must become NaN whatever the conversion's overflow mode does, and so must their product with `times`.
__device__ __forceinline__ float Scaled8(float v, float times)
{
    return __builtin_fabsf(v) < __builtin_inff() ? v * times : __builtin_nanf("");
}

// ---- groups of rows ----------------------------------------------------------------------------------------

// The rows [first, last) of unit `unit` of `per` rows: groups are cut into units one after the other, the last of a group
// may be shorter.  `before`: how many units lie in front of the group's.
struct Unit {
    int group;        // -1: there is no such unit
    int first, last;  // rows
    int groupFirst, groupLast;
    int before;
};

// Called by all 64 lanes of a wave.  Offsets that are not ascending or not within [0, rows] are brought there, so that
// whatever they hold no row outside is named.  per >= 16, rows <= 2^28.
__device__ __forceinline__ Unit FindUnit(const int32_t *__restrict__ offsets, int groups, int rows, int unit, int per)
{
    if (offsets == nullptr) {
        const int64_t first = int64_t(unit) * per;
        Unit u{first < rows ? 0 : -1, int(first), 0, 0, rows, 0};
        u.last = rows - first < per ? rows : int(first + per);
        return u;
    }
    const int lane = int(__lane_id());
    int64_t before = 0;   // (64 groups of at most 2^24 units fit 32 bits, all groups do not where their rows overlap)
    for (int g0 = 0; g0 < groups; g0 += 64) {
        const int g = g0 + lane;
        int lo = 0, hi = 0;
        if (g < groups) {
            lo = min(max(offsets[g], 0), rows);
            hi = min(max(offsets[g + 1], lo), rows);
        }
        const int mine = (hi - lo + per - 1) / per;
        int sum = mine;   // inclusive prefix over the lanes
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int other = __shfl_up(sum, d, 64);
            sum += lane >= d ? other : 0;
        }
        const int64_t start = before + sum - mine;
        const unsigned long long has = __ballot(unit >= start && unit < start + mine);
        if (has != 0) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll(has) - 1);
            Unit u;                       // (readlane: the compiler sees that all lanes have the same)
            u.group = g0 + at;
            u.groupFirst = __builtin_amdgcn_readlane(lo, at);
            u.groupLast = __builtin_amdgcn_readlane(hi, at);
            u.before = int(before) + __builtin_amdgcn_readlane(sum - mine, at);
            u.first = u.groupFirst + (unit - u.before) * per;
            u.last = min(u.first + per, u.groupLast);
            return u;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return Unit{-1, 0, 0, 0, 0, 0};
}

}  // namespace experts
}  // namespace hcclamd
