// Router by scores (HcclAmdExpertRouteScored): softmax or sigmoid, a bias that only chooses, groups of experts, weights that are renormalised or not;
// its gradient, and the bias's step (HcclAmdExpertBias).
//
// With s the scores, w = c s or c s / (sum of the chosen s), and dw the gradient of the weights:
//   sigmoid                 dx_j = w_j (1 - s_j) dw_j                 renormalised: dx_j = w_j (1 - s_j) (dw_j - sum_i (w_i / c) dw_i)
//   softmax, renormalised   dx_j = w_j (dw_j - sum_i (w_i / c) dw_i)  over the chosen ones; the others' gradients are zero
//   softmax                 dx_e = s_e (c dw_e - sum_i c s_i dw_i)    over all experts, dw_e = 0 where e was not chosen
//
// 16 lanes to a token (64 beyond 256 experts), its logits in registers.  Scores next to each other decide which expert a token goes to, and the choice
// is that of 64 bits; but it is made in 32 wherever these are enough.  A score and its bias become a whole number of 22 bits, a word of that and
// the expert goes into sorted lists by one median of three per entry, and the lists of a token's lanes are merged.  What the 22 bits are off by at most
// is known, so that a choice is settled unless, at some place that matters, two of them are closer than that and not made from the same logit and
// bias (which tie in any precision).  Waves with an unsettled token choose again in 64 bits.
#include <type_traits>

#include "rows.h"

namespace hcclamd {
namespace experts {
namespace {

struct ScoredArgs : RowsArgs {
    const void *logits;
    const uint8_t *mask;
    const float *bias;
    float *weights;
    int64_t stride;
    float weightScale;
    bool softmax, renormalise;
    int groups, kept, size;     // groups, how many of them a token may use, experts of each
    uint32_t perSize;           // 2^20 / size, rounded up: e * perSize >> 20 is e / size for e < 2^10
    bool second;                // a group's score is the sum of its two largest
};

__device__ __forceinline__ float Exp(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }

constexpr double kNever = -__builtin_inf();

// No instruction.  The compiler forgets what it knows of a lane's number, and works out what follows from it where it is needed instead of keeping
// it in registers over all tiles (64 of them and more).
__device__ __forceinline__ int Anew(int lane)
{
    asm volatile("" : "+v"(lane));
    return lane;
}

// Expert number of element i of lane l: eight neighbours to a lane, then the next lane's.
template <int kLanes>
__device__ __forceinline__ int ExpertOf(int i, int l) { return (i / 8 * kLanes + l) * 8 + i % 8; }

// ---- the choice in 64 bits --------------------------------------------------------------------------------
// One token's, by a whole wave: its experts best first, -1 where there is none.  kEach: a lane's experts, 64 apart.  `of`: a place per group, in LDS.
template <int kEach, int K, typename T>
__device__ __forceinline__ void ChooseExactly(const ScoredArgs &a, const T *row, double *of, int (&chosen)[K])
{
    const int lane = Anew(int(__lane_id()));
    float x[kEach];
    double key[kEach];
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        x[i] = i * 64 + lane < a.experts ? float(row[i * 64 + lane]) : -__builtin_inff();
    }
    if (a.softmax) {
        // (a NaN is left out, +inf takes all)
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            top = Larger(top, x[i]);
        }
        top = LargestOfNeighbours<64>(top);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            key[i] = x[i] == top ? 1.0 : x[i] < top ? exp(double(x[i]) - double(top)) : 0.0;
            sum += key[i];
        }
        sum = AddWave(sum);
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            key[i] /= sum;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            key[i] = 1.0 / (1.0 + exp(-double(x[i])));
        }
    }
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        if (a.bias != nullptr) {
            key[i] += double(a.bias[min(i * 64 + lane, a.experts - 1)]);
        }
        key[i] = x[i] > -__builtin_inff() && key[i] > kNever ? key[i] : kNever;
    }
    if (a.groups > 1) {
        for (int g = 0; g < a.groups; g++) {
            double first = kNever, next = kNever;
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                const bool mine = int(uint32_t(i * 64 + lane) * a.perSize >> 20) == g;
                const double k = mine ? key[i] : kNever;
                next = k > first ? first : k > next ? k : next;
                first = k > first ? k : first;
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double f = __shfl_xor(first, d, 64), n = __shfl_xor(next, d, 64);
                const double low = first < f ? first : f, rest = next > n ? next : n;
                next = low > rest ? low : rest;
                first = first > f ? first : f;
            }
            if (lane == 0) {
                of[g] = a.second && next > kNever ? first + next : first;
            }
        }
        Ordered();
        const double mine = lane < a.groups ? of[lane] : kNever;
        int before = 0;
        for (int o = 0; o < a.groups; o++) {
            const double other = of[o];
            before += other > mine || (other == mine && o < lane) ? 1 : 0;
        }
        const unsigned long long keep = __ballot(lane < a.groups && before < a.kept);
        Ordered();
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const uint32_t g = uint32_t(i * 64 + lane) * a.perSize >> 20;
            key[i] = (keep >> (g & 63) & 1) != 0 ? key[i] : kNever;
        }
    }
#pragma unroll
    for (int j = 0; j < K; j++) {
        chosen[j] = -1;
        if (j < a.topK) {
            double best = kNever;
            int e = -1;
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                const bool take = key[i] > best;      // (a lane's experts ascend)
                best = take ? key[i] : best;
                e = take ? i * 64 + lane : e;
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double other = __shfl_xor(best, d, 64);
                const int oe = __shfl_xor(e, d, 64);
                const bool take = other > best || (other == best && oe < e);
                best = take ? other : best;
                e = take ? oe : e;
            }
            chosen[j] = e;
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                key[i] = i * 64 + lane == e ? kNever : key[i];
            }
        }
    }
}

// log of the sigmoid
__device__ __forceinline__ float LogSigmoid(float x) { return fminf(x, 0.0f) - log1pf(Exp(-__builtin_fabsf(x))); }

__device__ __forceinline__ float Sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + Exp(-x)); }

// ---- the choice in 32 bits --------------------------------------------------------------------------------
// A score and its bias as a whole number: 1 + (s + b - least b) * times, below 2^22.  One step is (1 + largest b - least b) / 2^22.  With U = 2^-24, the
// difference b - least b, the sum and the product are each off by at most 2^22 U = 1/4 step, cutting off takes up to 1.  A sigmoid is off by
//   s (1 - s) (2 U |x| + 2 U)   the power's argument and the power         (|x| s (1 - s) < 0.23)
//   s (U + 2 U)                 the sum and the reciprocal
// which is 4 U, 1 step at most: two numbers are off against each other by twice 2.75.  A softmax's power, quotient and product are off by 5 U, and its sum, of 16 to a
// lane over up to 64 lanes, by 36 U, the same for all of a token's: 46 U, 11.5 steps between two of them, and 3.5 for the rest.
constexpr uint32_t kSlackSigmoid = 8, kSlackSoftmax = 24;

// Three bytes of DPP: the other lane of a pair, the other pair of four, the other four of eight, the other eight of sixteen (mirrored, where the
// lanes of each part are alike).
constexpr int kOther[4] = {0xb1, 0x4e, 0x141, 0x140};

template <int kWhich>
__device__ __forceinline__ uint32_t Other(uint32_t x)
{
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), kOther[kWhich], 0xf, 0xf, true));
}

__device__ __forceinline__ uint32_t Max(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t Min(uint32_t a, uint32_t b) { return a < b ? a : b; }

// The i-th of a sorted list and a new word is the median of the (i - 1)-th, the i-th and the new one.
__device__ __forceinline__ uint32_t Median(uint32_t a, uint32_t b, uint32_t c)
{
    uint32_t m;
    asm("v_med3_u32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
    return m;
}

// The larger half of two sorted lists: element by element against the other one backwards, which leaves a sequence that rises and falls once, then
// sorted by halving.
template <int K>
__device__ __forceinline__ void MergeLists(uint32_t (&best)[K], const uint32_t (&other)[K])
{
#pragma unroll
    for (int i = 0; i < K; i++) {
        best[i] = Max(best[i], other[K - 1 - i]);
    }
#pragma unroll
    for (int d = K / 2; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            if ((i & d) == 0) {
                const uint32_t hi = Max(best[i], best[i + d]), lo = Min(best[i], best[i + d]);
                best[i] = hi;
                best[i + d] = lo;
            }
        }
    }
}

template <int kWhich, int K>
__device__ __forceinline__ void MergeOther(uint32_t (&best)[K])
{
    uint32_t other[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        other[i] = Other<kWhich>(best[i]);
    }
    MergeLists(best, other);
}

// The two largest of these and another lane's two largest.
template <int kWhich>
__device__ __forceinline__ void MergeTwo(uint32_t &first, uint32_t &next)
{
    const uint32_t f = Other<kWhich>(first), n = Other<kWhich>(next);
    next = Max(Min(first, f), Max(next, n));
    first = Max(first, f);
}

template <int kLanes>
__device__ __forceinline__ uint32_t AddAll(uint32_t x)
{
    x += Other<0>(x);
    x += Other<1>(x);
    x += Other<2>(x);
    x += Other<3>(x);
    if constexpr (kLanes == 64) {
        x += uint32_t(__shfl_xor(int(x), 16, 64));
        x += uint32_t(__shfl_xor(int(x), 32, 64));
    }
    return x;
}

// What a launch's biases make of whole numbers.
struct Steps {
    float least, times;
    uint32_t slack;      // two numbers this close or closer need not be in their order
    bool fine;           // false: a bias is infinite, everything is chosen in 64 bits
};

// A lane's biases above the least of all, and what becomes of them.  Called by whole waves, which find out the same.
template <int kLanes, int kEach>
__device__ __forceinline__ Steps StepsOf(const ScoredArgs &a, int l, float (&bias)[kEach])
{
    Steps s{0.0f, 0.0f, a.softmax ? kSlackSoftmax : kSlackSigmoid, true};
    float least = 0.0f, most = 0.0f;
    if (a.bias != nullptr) {
        bool infinite = false;
        least = __builtin_inff();
        most = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int e = ExpertOf<kLanes>(i, l);
            const float b = a.bias[min(e, a.experts - 1)];
            bias[i] = b > -__builtin_inff() && e < a.experts ? b : -__builtin_inff();
            infinite = infinite || b == __builtin_inff();
            most = Larger(most, bias[i]);
            least = bias[i] > -__builtin_inff() && bias[i] < least ? bias[i] : least;
        }
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) {
            most = Larger(most, __shfl_xor(most, d, 64));
            const float other = __shfl_xor(least, d, 64);
            least = other < least ? other : least;
        }
        s.fine = __ballot(infinite) == 0 && most - least < __builtin_inff();
        least = least <= most ? least : 0.0f;
        most = most > least ? most : least;
    } else {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            bias[i] = ExpertOf<kLanes>(i, l) < a.experts ? 0.0f : -__builtin_inff();
        }
    }
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        bias[i] -= least;
    }
    s.least = least;
    s.times = float((1 << 22) - 4) / (1.0f + (most - least));
    return s;
}

// Whether a group's experts are those of 1, 2, 4, 8 or 16 neighbouring lanes.
__host__ __device__ constexpr bool Evenly(int size) { return size % 8 == 0 && size <= 128 && (size & (size - 1)) == 0; }

// Takes out what is not in a token's best groups.  Returns false where 32 bits do not settle it.  `numbers`: a place per expert, `of`: one per group, the
// token's, in LDS.
template <int kLanes, int kEach>
__device__ __forceinline__ bool ChooseGroups(const ScoredArgs &a, uint32_t (&number)[kEach], uint32_t slack, int l, int lane, uint32_t *numbers, uint32_t *of)
{
    bool sure = true;
    constexpr int kChunks = kEach / 8;
    const int across = a.size / 8;        // lanes that share a group
    if (Evenly(a.size)) {
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            uint32_t first = number[c * 8], next = 0;
#pragma unroll
            for (int i = 1; i < 8; i++) {
                next = Median(first, next, number[c * 8 + i]);
                first = Max(first, number[c * 8 + i]);
            }
            if (across > 1) {
                MergeTwo<0>(first, next);
            }
            if (across > 2) {
                MergeTwo<1>(first, next);
            }
            if (across > 4) {
                MergeTwo<2>(first, next);
            }
            if (across > 8) {
                MergeTwo<3>(first, next);
            }
            const int e = (c * kLanes + l) * 8;
            if (l % across == 0 && e < a.experts) {
                // (a group with one choice or none left: its sum has another zero, or none)
                of[uint32_t(e) * a.perSize >> 20] = !a.second ? first : next != 0 ? first + next : first != 0 ? ~0u : 0;
            }
        }
        Ordered();
    } else {
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            const int e = (c * kLanes + l) * 8;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (e + i < a.experts) {
                    numbers[e + i] = number[c * 8 + i];
                }
            }
        }
        Ordered();
        for (int g = l; g < a.groups; g += kLanes) {
            uint32_t first = 0, next = 0;
            int at = l % a.size;           // (neighbouring lanes begin at different banks)
            for (int i = 0; i < a.size; i++) {
                const uint32_t n = numbers[g * a.size + at];
                next = Median(first, next, n);
                first = Max(first, n);
                at = at + 1 == a.size ? 0 : at + 1;
            }
            of[g] = !a.second ? first : next != 0 ? first + next : first != 0 ? ~0u : 0;
        }
        Ordered();
    }
    const uint32_t room = a.second ? 2 * slack : slack;
    uint32_t keep[2] = {0, 0};
    for (int g0 = 0; g0 < a.groups; g0 += kLanes) {
        const int g = g0 + l;
        const uint32_t mine = g < a.groups ? of[g] : 0;
        int before = 0, close = 0;         // groups in front of this one; those that might be
        for (int o = 0; o < a.groups; o++) {
            const uint32_t other = of[o];
            before += other > mine || (other == mine && o < g) ? 1 : 0;
            close += other + room >= mine && other <= mine + room ? 1 : 0;
        }
        // (a group is close to itself) settled where no group it is not sure of decides whether it is kept
        const bool kept = mine != 0 && before < a.kept;
        sure = sure && (mine == 0 || (mine != ~0u && (close == 1 || before + close <= a.kept || before - close >= a.kept)));
        const unsigned long long bits = __ballot(kept);
        if constexpr (kLanes == 64) {
            keep[0] = uint32_t(bits);
            keep[1] = uint32_t(bits >> 32);
        } else {
            const uint32_t part = uint32_t(bits >> (lane & 48)) & 0xffff;
            keep[0] |= g0 < 32 ? part << (g0 & 16) : 0;
            keep[1] |= g0 < 32 ? 0 : part << (g0 & 16);
        }
    }
    Ordered();
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const uint32_t g = uint32_t(ExpertOf<kLanes>(i, l)) * a.perSize >> 20;
        const uint32_t word = g < 32 ? keep[0] : keep[1];
        number[i] = (word >> (g & 31) & 1) != 0 ? number[i] : 0;
    }
    return sure;
}

// The choice in 32 bits.  Returns false where they do not settle it, on some of the token's lanes.
template <int kLanes, int kEach, int K, typename T>
__device__ __forceinline__ bool ChooseFast(const ScoredArgs &a, const Steps &steps, const float (&x)[kEach], const float (&bias)[kEach], const T *row, bool in, int l,
    int lane, uint32_t *numbers, uint32_t *of, int (&chosen)[K])
{
    uint32_t number[kEach];
    if (a.softmax) {
        float top = -__builtin_inff(), sum = 0.0f, s[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            top = Larger(top, x[i]);
        }
        top = LargestOfNeighbours<kLanes>(top);
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            s[i] = x[i] == top ? 1.0f : x[i] < top ? Exp(x[i] - top) : 0.0f;
            sum += s[i];
        }
        const float by = 1.0f / AddNeighbours<kLanes>(sum);
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            number[i] = 1 + uint32_t((s[i] * by + bias[i]) * steps.times);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            number[i] = 1 + uint32_t((Sigmoid(x[i]) + bias[i]) * steps.times);
        }
    }
    // (bias[i]: above the least one, -inf where the expert is never chosen)
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        number[i] = x[i] > -__builtin_inff() && bias[i] >= 0.0f ? number[i] : 0;
    }
    bool sure = true;
    if (a.groups > 1) {
        sure = ChooseGroups<kLanes, kEach>(a, number, steps.slack, l, lane, numbers, of);
    }
    uint32_t best[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        best[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        number[i] = number[i] != 0 ? number[i] << 10 | (1023u - uint32_t(ExpertOf<kLanes>(i, l))) : 0;
#pragma unroll
        for (int k = K - 1; k > 0; k--) {
            best[k] = Median(best[k - 1], best[k], number[i]);
        }
        best[0] = Max(best[0], number[i]);
    }
    MergeOther<0>(best);
    MergeOther<1>(best);
    MergeOther<2>(best);
    MergeOther<3>(best);
    if constexpr (kLanes == 64) {
#pragma unroll 1
        for (int d = 16; d < 64; d <<= 1) {
            uint32_t other[K];
#pragma unroll
            for (int i = 0; i < K; i++) {
                other[i] = uint32_t(__shfl_xor(int(best[i]), d, 64));
            }
            MergeLists(best, other);
        }
    }
    // places that are too close: among the chosen ones, and at the border
    const uint32_t room = (steps.slack + 1) << 10;
    uint32_t last = 0;
    bool close = false;
#pragma unroll
    for (int i = 0; i < K; i++) {
        last = i + 1 == a.topK ? best[i] : last;
        if (i + 1 < K) {
            close = close || (i + 1 < a.topK && best[i] - best[i + 1] <= room);
        }
    }
    const uint32_t border = last > room ? last - room : 1;
    uint32_t above = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        above += number[i] >= border ? 1 : 0;
    }
    above = AddAll<kLanes>(above);
    close = close || above != uint32_t(a.topK);
    if (__ballot(in && close) != 0) {
        // what is made from the same logit and bias ties in 64 bits too, and goes by its number; the others do not
        const bool has = l < a.topK;
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < K; i++) {
            mine = l == i ? best[i] : mine;
        }
        const int e = mine != 0 ? int(1023u - (mine & 1023u)) : 0;
        const float logit = mine != 0 ? float(row[e]) : 0.0f, b = mine != 0 && a.bias != nullptr ? a.bias[e] : 0.0f;
        const int from = lane - l + a.topK - 1;
        const float lastLogit = __shfl(logit, from, 64), lastBias = __shfl(b, from, 64);
        const uint32_t next = uint32_t(__shfl_down(int(mine), 1, 64));
        const float nextLogit = __shfl_down(logit, 1, 64), nextBias = __shfl_down(b, 1, 64);
        const bool pair = l + 1 < a.topK && mine - next <= room && !(logit == nextLogit && b == nextBias);
        const uint32_t listed = AddAll<kLanes>(has && !(logit == lastLogit && b == lastBias) ? 1 : 0);
        uint32_t others = 0;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            // (the biases themselves: two of them may be as far above the least, in 32 bits)
            const float own = a.bias != nullptr ? a.bias[min(ExpertOf<kLanes>(i, l), a.experts - 1)] : 0.0f;
            others += number[i] >= border && !(x[i] == lastLogit && own == lastBias) ? 1 : 0;
        }
        others = AddAll<kLanes>(others);
        sure = sure && !pair && last != 0 && others == listed;
    }
#pragma unroll
    for (int i = 0; i < K; i++) {
        chosen[i] = i < a.topK && in && best[i] != 0 ? int(1023u - (best[i] & 1023u)) : -1;
    }
    return sure || !in;
}

template <typename T, int K, int kLanes, int kEach, int kHow>
__global__ void __launch_bounds__(kThreads, kLanes == 64 ? 2 : 4) ScoredKernel(ScoredArgs a)
{
    constexpr int kWaveTokens = 64 / kLanes, kTile = kWaveTokens * kThreads / 64;
    extern __shared__ uint32_t lds[];
    const int E = a.experts;
    uint32_t *chose = lds;                                                // [experts]: one bit per token of the tile
    int *count = reinterpret_cast<int *>(chose + E);                      // [experts]: rows of the tiles so far
    int *part = count + E;                                                // [waves]
    int *routed = part + kThreads / 64;                                   // [1]
    __shared__ double groupScores[kThreads / 64][HCCL_AMD_MAX_EXPERT_GROUPS];
    __shared__ uint32_t groupNumbers[kTile][HCCL_AMD_MAX_EXPERT_GROUPS];
    uint32_t *numbers = reinterpret_cast<uint32_t *>(routed + 1);         // [tokens of the tile][experts], for groups that lanes do not share evenly

    const int wave = int(threadIdx.x) / 64;
    for (int e = threadIdx.x; e < E; e += kThreads) {
        chose[e] = 0;
        count[e] = 0;
    }
    if (threadIdx.x == 0) {
        *routed = 0;
    }
    float bias[kEach];
    const Steps steps = StepsOf<kLanes, kEach>(a, int(threadIdx.x) % kLanes, bias);
    __syncthreads();
    for (int tile = 0; tile < a.tiles; tile++) {
        const int lane = Anew(int(threadIdx.x) % 64), l = lane % kLanes, r = wave * kWaveTokens + lane / kLanes;
        const int token = (int(blockIdx.x) * a.tiles + tile) * kTile + r;
        const bool in = token < a.tokens && (a.mask == nullptr || a.mask[token] != 0);
        // (the row of a token that takes no part is read and forgotten)
        const T *row = static_cast<const T *>(a.logits) + int64_t(min(token, max(a.tokens - 1, 0))) * a.stride;
        float x[kEach];
#pragma unroll
        for (int c = 0; c < kEach / 8; c++) {
            float v[8];
            LoadPart<kHow, 8>(row, (c * kLanes + l) * 8, a.tokens > 0 ? E : 0, v, -__builtin_inff());
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c * 8 + i] = v[i];
            }
        }
        int chosen[K];
        const bool settled = ChooseFast<kLanes, kEach, K>(a, steps, x, bias, row, in, l, lane, numbers + r * E, groupNumbers[r], chosen);
        const bool sure = steps.fine && settled;
        const unsigned long long lanes = kLanes == 64 ? ~0ull : 0xffffull << (lane & 48);
        unsigned long long unsure = __ballot(in && !sure);
        while (unsure != 0) {
            const int which = (__ffsll(unsure) - 1) / kLanes, whose = (int(blockIdx.x) * a.tiles + tile) * kTile + wave * kWaveTokens + which;
            int exactly[K];
            ChooseExactly<kLanes * kEach / 64, K>(a, static_cast<const T *>(a.logits) + int64_t(whose) * a.stride, groupScores[wave], exactly);
#pragma unroll
            for (int i = 0; i < K; i++) {
                chosen[i] = lane / kLanes == which ? exactly[i] : chosen[i];
            }
            unsure &= ~(kLanes == 64 ? ~0ull : 0xffffull << which * 16);
        }
        // lane j of a token has its j-th choice
        int mine = -1;
#pragma unroll
        for (int i = 0; i < K; i++) {
            mine = l == i ? chosen[i] : mine;
        }
        const float logit = mine >= 0 ? float(row[mine]) : -__builtin_inff();
        float w;
        if (a.softmax) {
            float top = -__builtin_inff(), total = 0.0f;
            bool bad = false;
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                top = Larger(top, x[i]);
                bad = bad || !(x[i] < __builtin_inff());
            }
            top = LargestOfNeighbours<kLanes>(top);
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                total += Exp(x[i] - top);
            }
            total = AddNeighbours<kLanes>(total);
            if (a.renormalise) {
                top = LargestOfNeighbours<16>(logit);
            }
            w = mine >= 0 ? Exp(logit - top) : 0.0f;
            w /= a.renormalise ? AddNeighbours<16>(w) : total;
            // (a NaN or +inf in the row: the weights are NaN, chosen or not by these)
            const unsigned long long rows = __ballot(bad);
            w = (rows & lanes) != 0 ? __builtin_nanf("") : w;
        } else if (a.renormalise) {
            // by logarithms: the scores of very negative logits are 0 in 32 bits, their ratios are not
            const float s = mine >= 0 ? LogSigmoid(logit) : -__builtin_inff(), top = LargestOfNeighbours<16>(s);
            w = mine >= 0 ? Exp(s - top) : 0.0f;
            w /= AddNeighbours<16>(w);
        } else {
            w = Sigmoid(logit);
        }
        if (mine >= 0 && l == 0) {
            atomicAdd(routed, 1);   // a whole number: the order does not matter
        }
        const int64_t at = int64_t(token) * a.topK + l;
        const bool writes = token < a.tokens && l < a.topK;
        if (writes) {
            a.expertOf[at] = mine;
            a.weights[at] = mine >= 0 ? w * a.weightScale : 0.0f;
            if (mine >= 0) {
                atomicOr(&chose[mine], 1u << r);
            }
        }
        __syncthreads();
        // a choice's place among the workgroup's rows of its expert
        int place = -1;
        if (writes && mine >= 0) {
            place = count[mine] + __popc(chose[mine] & ((1u << r) - 1));
        }
        __syncthreads();
        for (int e = threadIdx.x; e < E; e += kThreads) {
            count[e] += __popc(chose[e]);
            chose[e] = 0;
        }
        __syncthreads();
        const bool last = a.blocks == 1 && tile + 1 == a.tiles;
        if (last) {
            // a single workgroup: its places become rows at once
            Finish<kThreads, false>(a, count, nullptr, *routed, part, nullptr, true);
        }
        if (writes) {
            a.rowOf[at] = place < 0 ? -1 : place + (last ? count[mine] : 0);
        }
    }
    if (a.blocks == 1) {
        for (int i = threadIdx.x; i < (a.tiles - 1) * kTile * a.topK; i += kThreads) {   // the tiles before the last one
            const int e = a.expertOf[i];
            if (e >= 0) {
                a.rowOf[i] += count[e];
            }
        }
        return;
    }
    for (int e = threadIdx.x; e < E; e += kThreads) {
        a.blockCounts[int64_t(blockIdx.x) * (E + 1) + e] = count[e];
    }
    if (threadIdx.x == 0) {
        a.blockCounts[int64_t(blockIdx.x) * (E + 1) + E] = *routed;
    }
}

struct ScoredGradArgs {
    const void *logits;
    const int32_t *expertOf;
    const float *weightGrad;
    void *logitGrad;
    int64_t stride, gradStride;
    int tokens, experts, topK;
    float weightScale;
    bool softmax, renormalise;
};

// kLanes lanes to a token.  Its row lies in LDS, zero but where the choices' lanes put their gradients, and goes out from there; a softmax that is
// not renormalised (kDense) puts all of it there.
template <typename T, int kLanes, int kEach, bool kDense, int kHow>
__global__ void __launch_bounds__(kThreads) ScoredGradKernel(ScoredGradArgs a)
{
    constexpr int kTokens = kThreads / kLanes, kStep = kLanes * 8;
    __shared__ __align__(16) float rows[kTokens][kLanes * kEach];
    const int l = int(threadIdx.x) % kLanes, slot = int(threadIdx.x) / kLanes, E = a.experts;
    float *mine = rows[slot];
#pragma unroll
    for (int c = 0; c < kEach; c++) {
        mine[c * kLanes + l] = 0.0f;
    }
    Ordered();
    for (int64_t t = int64_t(blockIdx.x) * kTokens + slot; t < a.tokens; t += int64_t(gridDim.x) * kTokens) {
        T *out = static_cast<T *>(a.logitGrad) + t * a.gradStride;
        const T *in = static_cast<const T *>(a.logits) + t * a.stride;
        int chosen = l < a.topK ? a.expertOf[t * a.topK + l] : -1;
        chosen = chosen < E ? chosen : -1;
        const float dw = chosen >= 0 ? a.weightGrad[t * a.topK + l] * a.weightScale : 0.0f;
        const float logit = chosen >= 0 ? float(in[chosen]) : -__builtin_inff();
        float more = 0.0f;
        if constexpr (kDense) {
            const bool none = a.expertOf[t * a.topK] < 0;
            float x[kEach], top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
            for (int c = 0; c < kEach / 8; c++) {
                float v[8];
                LoadPart<kHow, 8>(in, c * kStep + l * 8, E, v, -__builtin_inff());
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[c * 8 + i] = v[i];
                    top = Larger(top, v[i]);
                }
            }
            top = LargestOfNeighbours<kLanes>(top);
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                x[i] = Exp(x[i] - top);
                sum += x[i];
            }
            const float by = 1.0f / AddNeighbours<kLanes>(sum);
            more = chosen >= 0 ? Exp(logit - top) * by * dw : 0.0f;
            const float dot = AddNeighbours<kLanes>(more);
#pragma unroll
            for (int c = 0; c < kEach / 8; c++) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    mine[c * kStep + l * 8 + i] = none ? 0.0f : -(x[c * 8 + i] * by * dot);
                }
            }
            Ordered();
            if (chosen >= 0) {
                mine[chosen] += more;
            }
        } else {
            if (a.renormalise) {
                const float key = chosen < 0 ? -__builtin_inff() : a.softmax ? logit : LogSigmoid(logit);
                const float top = LargestOfNeighbours<16>(key);      // (what crosses lanes stands outside of what only some of them do)
                float w = chosen >= 0 ? Exp(key - top) : 0.0f;
                const float sum = AddNeighbours<16>(w);
                w = chosen >= 0 ? w / sum : 0.0f;
                const float mean = AddNeighbours<16>(w * dw);
                more = w * (dw - mean);
            } else {
                more = Sigmoid(logit) * dw;
            }
            // (1 - s is the sigmoid of -x)
            more = a.softmax ? more : more * Sigmoid(-logit);
            if (chosen >= 0) {
                mine[chosen] = more;
            }
        }
        Ordered();
#pragma unroll
        for (int c = 0; c < kEach / 8; c++) {
            const int e = c * kStep + l * 8;
            const Float4 f = *reinterpret_cast<const Float4 *>(mine + e), g = *reinterpret_cast<const Float4 *>(mine + e + 4);
            const float v[8] = {f[0], f[1], f[2], f[3], g[0], g[1], g[2], g[3]};
            StorePart<kHow, 8>(out, e, E, v);
        }
        Ordered();
        if (!kDense && chosen >= 0) {
            mine[chosen] = 0.0f;
        }
        Ordered();
    }
}

__global__ void __launch_bounds__(kThreads) BiasKernel(const int32_t *counts, int experts, float rate, const float *bias, float *newBias)
{
    __shared__ long long parts[kThreads / 64];
    long long sum = 0;
    for (int e = threadIdx.x; e < experts; e += kThreads) {
        sum += counts[e];
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        sum += __shfl_xor(sum, d, 64);
    }
    if (threadIdx.x % 64 == 0) {
        parts[threadIdx.x / 64] = sum;
    }
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) {
        sum += parts[w];
    }
    for (int e = threadIdx.x; e < experts; e += kThreads) {
        const long long all = static_cast<long long>(experts) * counts[e];    // against the mean, times the experts
        newBias[e] = bias[e] + (all < sum ? rate : all > sum ? -rate : 0.0f);
    }
}

// Tokens of a tile: four a wave with 16 lanes to each, one with 64.
int TileOf(uint32_t experts) { return experts <= 256 ? 16 : 4; }

template <typename T, int K, int kLanes, int kEach>
HcclResult LaunchScored(const ScoredArgs &a, bool wide, hipStream_t stream)
{
    const size_t lds = 4 * (2 * size_t(a.experts) + kThreads / 64 + 1 + (Evenly(a.size) ? 0 : kThreads / kLanes * size_t(a.experts)));
    const auto go = [&](auto kernel) { return Launch("HcclAmdExpertRouteScored", kernel, uint32_t(a.blocks), kThreads, lds, stream, a); };
    return wide ? go(ScoredKernel<T, K, kLanes, kEach, kAligned>) : go(ScoredKernel<T, K, kLanes, kEach, kAnyhow>);
}

template <typename T, int K>
HcclResult LaunchScoredShape(const ScoredArgs &a, bool wide, hipStream_t stream)
{
    return a.experts <= 128   ? LaunchScored<T, K, 16, 8>(a, wide, stream)
           : a.experts <= 256 ? LaunchScored<T, K, 16, 16>(a, wide, stream)
                              : LaunchScored<T, K, 64, 16>(a, wide, stream);
}

template <typename T>
HcclResult LaunchScoredType(const ScoredArgs &a, bool wide, hipStream_t stream)
{
    return a.topK <= 8 ? LaunchScoredShape<T, 8>(a, wide, stream) : LaunchScoredShape<T, 16>(a, wide, stream);
}

template <typename T, bool kDense, int kHow>
HcclResult LaunchScoredGrad(const ScoredGradArgs &a, hipStream_t stream)
{
    const auto go = [&](auto kernel, int lanes) {
        const int64_t blocks = (int64_t(a.tokens) * lanes + kThreads - 1) / kThreads;
        return Launch("HcclAmdExpertRouteScoredGrad", kernel, uint32_t(blocks < 2048 ? blocks : 2048), kThreads, 0, stream, a);
    };
    return a.experts <= 128   ? go(ScoredGradKernel<T, 16, 8, kDense, kHow>, 16)
           : a.experts <= 256 ? go(ScoredGradKernel<T, 16, 16, kDense, kHow>, 16)
                              : go(ScoredGradKernel<T, 64, 16, kDense, kHow>, 64);
}

}  // namespace
}  // namespace experts
}  // namespace hcclamd

using namespace hcclamd::experts;

extern "C" {

HcclResult HcclAmdExpertRouteScoredWorkspace(uint64_t tokens, uint32_t experts, uint64_t *bytes)
{
    EXPERTS_CHK_PTR(bytes);
    EXPERTS_CHK(experts >= 1 && experts <= HCCL_AMD_MAX_EXPERTS);
    EXPERTS_CHK(tokens <= kMaxTokens);
    const uint64_t blocks = uint64_t(BlocksOf(tokens, TileOf(experts)));
    *bytes = blocks == 1 ? 0 : 4 * blocks * (uint64_t(experts) + 1);
    return HCCL_SUCCESS;
}

HcclResult HcclAmdExpertRouteScored(const void *logits, HcclDataType logitType, uint64_t tokens, uint32_t experts, uint64_t logitStride,
    HcclAmdScore score, const float *bias, uint32_t groups, uint32_t groupsKept, uint32_t groupTop, uint32_t topK, uint32_t renormalise,
    float weightScale, const uint8_t *tokenMask, int32_t *expertOf, float *weights, int32_t *rowOf, int32_t *counts, int32_t *offsets,
    void *workspace, uint64_t workspaceBytes, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(logitType));
    EXPERTS_CHK_TYPE(score == HCCL_AMD_SCORE_SOFTMAX || score == HCCL_AMD_SCORE_SIGMOID);
    EXPERTS_CHK(experts >= 1 && experts <= HCCL_AMD_MAX_EXPERTS);
    EXPERTS_CHK(groups >= 1 && groups <= HCCL_AMD_MAX_EXPERT_GROUPS && experts % groups == 0);
    EXPERTS_CHK(groupsKept >= 1 && groupsKept <= groups);
    EXPERTS_CHK(groupTop == 1 || groupTop == 2);
    EXPERTS_CHK(topK >= 1 && topK <= HCCL_AMD_MAX_TOPK && topK <= groupsKept * (experts / groups));
    EXPERTS_CHK(tokens <= kMaxTokens);
    EXPERTS_CHK_PTR(counts);
    EXPERTS_CHK_PTR(offsets);
    EXPERTS_CHK(Aligned(counts, 4) && Aligned(offsets, 4) && Aligned(bias, 4));
    uint64_t needed = 0;
    HcclAmdExpertRouteScoredWorkspace(tokens, experts, &needed);
    if (tokens != 0) {
        EXPERTS_CHK_PTR(logits);
        EXPERTS_CHK_PTR(expertOf);
        EXPERTS_CHK_PTR(weights);
        EXPERTS_CHK_PTR(rowOf);
        EXPERTS_CHK(Stride(logitStride, experts));
        EXPERTS_CHK(AlignedTo(logitType, logits) && Aligned(expertOf, 4) && Aligned(weights, 4) && Aligned(rowOf, 4));
        if (needed != 0) {
            EXPERTS_CHK_PTR(workspace);
            EXPERTS_CHK(Aligned(workspace, 16));
            EXPERTS_CHK(workspaceBytes >= needed);
        }
    }
    const int tile = TileOf(experts);
    ScoredArgs a{};
    a.logits = logits;
    a.mask = tokenMask;
    a.bias = bias;
    a.expertOf = expertOf;
    a.weights = weights;
    a.rowOf = rowOf;
    a.counts = counts;
    a.offsets = offsets;
    a.stride = int64_t(logitStride == 0 ? experts : logitStride);
    a.weightScale = weightScale;
    a.softmax = score == HCCL_AMD_SCORE_SOFTMAX;
    a.renormalise = renormalise != 0;
    a.groups = int(groups);
    a.kept = int(groupsKept);
    a.size = int(experts / groups);
    a.perSize = uint32_t(((1 << 20) + a.size - 1) / a.size);
    a.second = groupTop == 2 && a.size > 1;
    a.tokens = int(tokens);
    a.experts = int(experts);
    a.topK = int(topK);
    a.tiles = TilesOf(tokens, tile);
    a.blocks = BlocksOf(tokens, tile);       // no token: the one workgroup writes the zeros
    a.blockCounts = static_cast<int32_t *>(workspace);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const bool wide = experts % 8 == 0 && Aligned(logits, 16) && uint64_t(a.stride) * SizeOf(logitType) % 16 == 0;
    HcclResult r = logitType == HCCL_DATA_TYPE_FP32   ? LaunchScoredType<float>(a, wide, on)
                   : logitType == HCCL_DATA_TYPE_FP16 ? LaunchScoredType<_Float16>(a, wide, on)
                                                      : LaunchScoredType<__bf16>(a, wide, on);
    if (r != HCCL_SUCCESS || a.blocks == 1) {
        return r;
    }
    const bool few = a.blocks <= 32;
    if (!few) {
        r = Launch("HcclAmdExpertRouteScored", ScanKernel<false>, experts / kScanCols + 1, kThreads, 0, on, RowsArgs(a));
        if (r != HCCL_SUCCESS) {
            return r;
        }
    }
    return Launch("HcclAmdExpertRouteScored", few ? RowsKernel<true, false> : RowsKernel<false, false>, uint32_t(a.blocks), kThreads, RowsLds(a.experts), on,
        RowsArgs(a), tile * a.tiles);
}

HcclResult HcclAmdExpertRouteScoredGrad(const void *logits, HcclDataType logitType, uint64_t tokens, uint32_t experts, uint64_t logitStride,
    HcclAmdScore score, uint32_t topK, uint32_t renormalise, float weightScale, const int32_t *expertOf, const float *weightGrad, void *logitGrad,
    uint64_t logitGradStride, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(logitType));
    EXPERTS_CHK_TYPE(score == HCCL_AMD_SCORE_SOFTMAX || score == HCCL_AMD_SCORE_SIGMOID);
    EXPERTS_CHK(experts >= 1 && experts <= HCCL_AMD_MAX_EXPERTS);
    EXPERTS_CHK(topK >= 1 && topK <= HCCL_AMD_MAX_TOPK && topK <= experts);
    EXPERTS_CHK(tokens <= kMaxTokens);
    if (tokens == 0) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(logits);
    EXPERTS_CHK_PTR(expertOf);
    EXPERTS_CHK_PTR(weightGrad);
    EXPERTS_CHK_PTR(logitGrad);
    EXPERTS_CHK(Stride(logitStride, experts) && Stride(logitGradStride, experts));
    EXPERTS_CHK(AlignedTo(logitType, logits) && AlignedTo(logitType, logitGrad) && Aligned(expertOf, 4) && Aligned(weightGrad, 4));
    ScoredGradArgs a{};
    a.logits = logits;
    a.expertOf = expertOf;
    a.weightGrad = weightGrad;
    a.logitGrad = logitGrad;
    a.stride = int64_t(logitStride == 0 ? experts : logitStride);
    a.gradStride = int64_t(logitGradStride == 0 ? experts : logitGradStride);
    a.tokens = int(tokens);
    a.experts = int(experts);
    a.topK = int(topK);
    a.weightScale = weightScale;
    a.softmax = score == HCCL_AMD_SCORE_SOFTMAX;
    a.renormalise = renormalise != 0;
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const uint64_t unit = SizeOf(logitType);
    const bool dense = a.softmax && !a.renormalise;
    const bool wide = experts % 8 == 0 && Aligned(logitGrad, 16) && uint64_t(a.gradStride) * unit % 16 == 0 &&
        (!dense || (Aligned(logits, 16) && uint64_t(a.stride) * unit % 16 == 0));
    const auto go = [&](auto of) {
        typedef decltype(of) T;
        return dense ? (wide ? LaunchScoredGrad<T, true, kAligned>(a, on) : LaunchScoredGrad<T, true, kAnyhow>(a, on))
                     : (wide ? LaunchScoredGrad<T, false, kAligned>(a, on) : LaunchScoredGrad<T, false, kAnyhow>(a, on));
    };
    return logitType == HCCL_DATA_TYPE_FP32 ? go(float{}) : logitType == HCCL_DATA_TYPE_FP16 ? go(_Float16{}) : go(__bf16{});
}

HcclResult HcclAmdExpertBias(const int32_t *counts, uint32_t experts, float rate, const float *bias, float *newBias, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK(experts >= 1 && experts <= HCCL_AMD_MAX_EXPERTS);
    EXPERTS_CHK_PTR(counts);
    EXPERTS_CHK_PTR(bias);
    EXPERTS_CHK_PTR(newBias);
    EXPERTS_CHK(Aligned(counts, 4) && Aligned(bias, 4) && Aligned(newBias, 4));
    return Launch("HcclAmdExpertBias", BiasKernel, 1, kThreads, 0, static_cast<hipStream_t>(stream), counts, int(experts), rate, bias, newBias);
}

}  // extern "C"
