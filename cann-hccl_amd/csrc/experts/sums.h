// Sums and maxima over neighbouring lanes, the order of a wave's LDS operations, rows of any width.
#pragma once
#include "common.h"

namespace hcclamd {
namespace experts {

// Adds up over the lanes whose numbers agree above the lowest bits: kLanes neighbouring lanes, a power of two up to 64.
template <int kLanes>
__device__ __forceinline__ float AddNeighbours(float x)
{
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) {
        x += __shfl_xor(x, d, 64);
    }
    return x;
}

// A row of 16 lanes turned by kBy.
template <int kBy>
__device__ __forceinline__ float Turned(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 + kBy, 0xf, 0xf, true));
}

// The same over 16 lanes without LDS.
template <>
__device__ __forceinline__ float AddNeighbours<16>(float x)
{
    x += Turned<8>(x);
    x += Turned<4>(x);
    x += Turned<2>(x);
    x += Turned<1>(x);
    return x;
}

// The largest, NaN being less than everything.
__device__ __forceinline__ float Larger(float a, float b) { return b > a ? b : a; }

template <int kLanes>
__device__ __forceinline__ float LargestOfNeighbours(float x)
{
    if constexpr (kLanes == 16) {
        x = Larger(x, Turned<8>(x));
        x = Larger(x, Turned<4>(x));
        x = Larger(x, Turned<2>(x));
        x = Larger(x, Turned<1>(x));
    } else {
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) {
            x = Larger(x, __shfl_xor(x, d, 64));
        }
    }
    return x;
}

template <int kBy>
__device__ __forceinline__ double Turned(double x)
{
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    const uint32_t low = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(bits)), 0x120 + kBy, 0xf, 0xf, true));
    const uint32_t high = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(bits >> 32)), 0x120 + kBy, 0xf, 0xf, true));
    return __builtin_bit_cast(double, uint64_t(high) << 32 | low);
}

__device__ __forceinline__ double FromLane(double x, int lane)
{
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    const uint32_t low = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(bits)), lane));
    const uint32_t high = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(bits >> 32)), lane));
    return __builtin_bit_cast(double, uint64_t(high) << 32 | low);
}

// Over all lanes of a wave, which all have to be there: rows of 16 by turning them, then the four rows.
__device__ __forceinline__ double AddWave(double x)
{
    x += Turned<8>(x);
    x += Turned<4>(x);
    x += Turned<2>(x);
    x += Turned<1>(x);
    return (FromLane(x, 0) + FromLane(x, 16)) + (FromLane(x, 32) + FromLane(x, 48));
}

// A block of 128 values, eight to each of 16 lanes, in 8 bits, and its scale.  Where all of a wave's are finite, as they mostly are, nothing looks at each of
// them (four of 28 instructions a value in the gate, whose vector unit is busy most of the time).  Called by whole waves.
template <HcclAmdScaleType kScale>
__device__ __forceinline__ Word2 QuantiseBlock(float (&v)[8], typename BlockScale<kScale>::Stored &stored)
{
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        top = __builtin_fmaxf(top, __builtin_fabsf(v[i]));      // (leaves NaN out)
    }
    top = LargestOfNeighbours<16>(top);
    if (__ballot(!(top < __builtin_inff())) != 0) {
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            top = __builtin_fmaxf(top, FiniteSize(v[i]));
            v[i] = Scaled8(v[i], 1.0f);
        }
        top = LargestOfNeighbours<16>(top);
    }
    const BlockScale<kScale> scale(top);
    stored = scale.stored;
    return Word2{Quantise4(v[0] * scale.times, v[1] * scale.times, v[2] * scale.times, v[3] * scale.times),
        Quantise4(v[4] * scale.times, v[5] * scale.times, v[6] * scale.times, v[7] * scale.times)};
}

// a - b in two parts: what rounding takes from the first is the second.
struct Difference {
    float high, low;
    __device__ __forceinline__ Difference(float a, float b) : high(a - b), low(0.0f)
    {
        const float back = high - a;
        low = (a - (high - back)) - (b + back);
    }
};

// exp(x + more) for x <= 0, `more` being what rounding took from x: good to two units in the last place where it is 2^-126 or more, 0 below.  What rounding the
// power's argument loses (up to 2^-24 of it: 22 * 2^-24 of the power at x = -40) comes back with the power, which is the hardware's.  A NaN stays; -inf needs no `more`.
__device__ __forceinline__ float Power(float x, float more)
{
    more = x < -10000.0f ? 0.0f : more;
    x = x < -10000.0f ? -10000.0f : x;
    const float t = x * 0x1.715476p+0f, p = __builtin_amdgcn_exp2f(t);
    const float lost = __builtin_fmaf(x, 0x1.4ae0cp-26f, __builtin_fmaf(x, 0x1.715476p+0f, -t));      // log2(e) in two parts
    return __builtin_fmaf(p, __builtin_fmaf(lost, 0x1.62e43p-1f, more), p);
}

// Keeps the compiler from moving LDS operations of one wave's lanes past each other.
__device__ __forceinline__ void Ordered()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A lane's N elements of a row of `width`, from column `at` on, in two steps: all that a row needs is fetched, then each part settled.  Where neither rows nor
// widths are multiples of anything (kAnyhow) a lane whose part crosses the row's end fetches the row's last N elements, and moves them down when it
// settles: one load on its way for each part, not one behind the other for each element (norm and gradient of 16384 rows of 2001 values: 102 us instead of 124).
template <int kHow, int N, typename T>
__device__ __forceinline__ void Fetch(const T *row, int at, int width, T (&v)[N])
{
    if (kHow != kAnyhow || width < N) {
        LoadPart<kHow, N>(row, at, width, v, T(0.0f));
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = T(0.0f);
    }
    if (at < width) {
        Load<false, N>(row + min(at, width - N), v);
    }
}

// Zeros behind the row's end.
template <int kHow, int N, typename T>
__device__ __forceinline__ void Settle(const T (&v)[N], int at, int width, float (&to)[N])
{
#pragma unroll
    for (int i = 0; i < N; i++) {
        to[i] = float(v[i]);
    }
    const int by = at + N - width;
    if (kHow != kAnyhow || width < N || __ballot(by > 0 && by < N) == 0) {
        return;
    }
#pragma unroll
    for (int d = N / 2; d > 0; d >>= 1) {
        const bool move = by > 0 && by < N && (by & d) != 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            to[i] = move ? (i + d < N ? to[i + d < N ? i + d : 0] : 0.0f) : to[i];
        }
    }
}

}  // namespace experts
}  // namespace hcclamd
