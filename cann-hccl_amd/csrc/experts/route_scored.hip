// Router by scores (HcclAmdExpertRouteScored): softmax or sigmoid, a bias that only chooses, groups of experts, weights that are renormalised or not;
// its gradient, and the bias's step (HcclAmdExpertBias).
//
// With s the scores, w = c s or c s / (sum of the chosen s), and dw the gradient of the weights:
//   sigmoid                 dx_j = w_j (1 - s_j) dw_j                 renormalised: dx_j = w_j (1 - s_j) (dw_j - sum_i (w_i / c) dw_i)
//   softmax, renormalised   dx_j = w_j (dw_j - sum_i (w_i / c) dw_i)  over the chosen ones; the others' gradients are zero
//   softmax                 dx_e = s_e (c dw_e - sum_i c s_i dw_i)    over all experts, dw_e = 0 where e was not chosen
//
// 8, 16 or 64 lanes to a token, its logits in registers.  Scores next to each other decide which expert a token goes to, and the choice
// is that of 64 bits; but it is made in 32 wherever these are enough.  A score and its bias become a whole number of 22 bits, a word of that and
// the expert goes into sorted lists by one median of three per entry, and the lists of a token's lanes are merged.  What the 22 bits are off by at most
// is known, so that a choice is settled unless, at some place that matters, two of them are closer than that and not made from the same logit and
// bias (which tie in any precision).  Of an unsettled token the chosen ones and the next are put in order by their keys in 64 bits; where that does not
// settle it either -- its groups are too close, or several experts at the border -- a whole wave chooses for it in 64 bits.
//
// Measured: 65536 tokens of 256 experts in eight groups, eight chosen, 16-bit logits (33.5 MB): 34 us to choose, 6 to add up, 4 for the rows, 10 for the
// gradient, 2 for the bias.  Choosing spends about 35 vector instructions on each expert, of which eight are medians and eight what a power and a reciprocal take: they
// keep the vector units busy for 59 % of the time, and waves wait for 40 % of theirs, since a tile's logits are not fetched before the one in front is done.  One token in 300 has choices
// closer than 32 bits hold (3 us of the 34), one in 2000 groups that are (4 us, since the others wait); with everything in 64 bits it took 240 us, which is also what a finite bias
// 1e4 away from the others makes of it (64 us for all launches instead of 44 where it is 100 away, 105 at 1000).  Eight lanes to a token spend fewer instructions on merging than
// sixteen (43 us against 49 with all launches), sixteen are quicker where there are few tokens.  Above 256 experts there is one layout, a wave to a token with 16 experts to a lane, whatever
// share of them is there: 65536 tokens of 257, 384, 512 and 1024 experts 142, 135, 138 and 168 us with all launches, in eight groups of 40, 48, 64 and 128 231, 245, 167 and 437.
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
// it in registers over all tiles (64 of them and more): 43.0 us instead of 46.2 for 65536 tokens.
template <typename V>
__device__ __forceinline__ V Anew(V lane)
{
    asm volatile("" : "+v"(lane));
    return lane;
}

// The same of a number that all lanes have: masks made from it are two scalar registers each.
__device__ __forceinline__ int AnewForAll(int n)
{
    asm volatile("" : "+s"(n));
    return n;
}

// Expert number of element i of lane l: eight neighbours to a lane, then the next lane's.
template <int kLanes>
__device__ __forceinline__ int ExpertOf(int i, int l) { return (i / 8 * kLanes + l) * 8 + i % 8; }

// ---- the choice in 64 bits --------------------------------------------------------------------------------
// A key and its expert, and which of two is first: the larger, the lower expert of equal ones.
struct Choice {
    double key;
    int expert;
};

__device__ __forceinline__ bool Before(Choice a, Choice b) { return a.key > b.key || (a.key == b.key && a.expert < b.expert); }

__device__ __forceinline__ Choice First(Choice a, Choice b)
{
    const bool take = Before(b, a);
    return Choice{take ? b.key : a.key, take ? b.expert : a.expert};
}

template <int kBy>
__device__ __forceinline__ Choice TurnedChoice(Choice c)
{
    return Choice{Turned<kBy>(c.key), __builtin_amdgcn_update_dpp(0, c.expert, 0x120 + kBy, 0xf, 0xf, true)};
}

__device__ __forceinline__ Choice ChoiceFrom(Choice c, int lane) { return Choice{FromLane(c.key, lane), __builtin_amdgcn_readlane(c.expert, lane)}; }

// Over a whole wave.
__device__ __forceinline__ Choice FirstOfWave(Choice c)
{
    c = First(c, TurnedChoice<8>(c));
    c = First(c, TurnedChoice<4>(c));
    c = First(c, TurnedChoice<2>(c));
    c = First(c, TurnedChoice<1>(c));
    return First(First(ChoiceFrom(c, 0), ChoiceFrom(c, 16)), First(ChoiceFrom(c, 32), ChoiceFrom(c, 48)));
}

// What it takes of a launch's arguments: by value, since it is a function of its own, whose registers those that do not call it need not hold free.
struct ExactArgs {
    const float *bias;
    int experts, topK, groups, kept, size;
    uint32_t perSize;
    bool softmax, second;
};

// One token's, by a whole wave: lane j has the j-th expert, best first, -1 where there is none.  kEach: a lane's experts, 64 apart.  `keys`: a place per expert,
// `of`: one per group, in LDS.  Loops, not straight code: this is seldom called, and every instruction has to be fetched then.
template <int kEach, typename T>
__device__ __attribute__((noinline)) int ChooseExactly(ExactArgs a, const T *row, double *keys, double *of)
{
    const int lane = Anew(int(__lane_id()));
    float top = -__builtin_inff();
    double sum = 1.0;
    if (a.softmax) {
        // (a NaN is left out, +inf takes all)
        for (int e = lane; e < a.experts; e += 64) {
            top = Larger(top, float(row[e]));
        }
        top = LargestOfNeighbours<64>(top);
        sum = 0.0;
#pragma unroll 1
        for (int e = lane; e < a.experts; e += 64) {
            const float x = float(row[e]);
            sum += x == top ? 1.0 : x < top ? exp(double(x) - double(top)) : 0.0;
        }
        sum = AddWave(sum);
    }
#pragma unroll 1
    for (int e = lane; e < a.experts; e += 64) {
        const float x = float(row[e]);
        const double p = exp(a.softmax ? (x == top ? 0.0 : double(x) - double(top)) : -double(x));
        const double key = (a.softmax ? p / sum : 1.0 / (1.0 + p)) + (a.bias != nullptr ? double(a.bias[e]) : 0.0);
        keys[e] = x > -__builtin_inff() && key > kNever ? key : kNever;
    }
    Ordered();
    unsigned long long keep = ~0ull;
    if (a.groups > 1) {
        double mine = kNever;
        if (lane < a.groups) {
            double next = kNever;
            int at = lane % a.size;            // (neighbouring lanes begin at different banks)
#pragma unroll 4
            for (int i = 0; i < a.size; i++) {
                const double k = keys[lane * a.size + at];
                next = k > mine ? mine : k > next ? k : next;
                mine = k > mine ? k : mine;
                at = at + 1 == a.size ? 0 : at + 1;
            }
            mine = a.second && next > kNever ? mine + next : mine;
            of[lane] = mine;
        }
        Ordered();
        int before = 0;
#pragma unroll 4
        for (int o = 0; o < a.groups; o++) {
            const double other = of[o];
            before += other > mine || (other == mine && o < lane) ? 1 : 0;
        }
        keep = __ballot(lane < a.groups && before < a.kept);
    }
    double key[kEach];
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const int e = i * 64 + lane;
        const uint32_t g = a.groups > 1 ? uint32_t(e) * a.perSize >> 20 : 0;
        key[i] = e < a.experts && (keep >> (g & 63) & 1) != 0 ? keys[min(e, a.experts - 1)] : kNever;
    }
    Ordered();
    int taken = -1;                            // lane j: the j-th
#pragma unroll 1
    for (int j = 0; j < a.topK; j++) {
        Choice best{kNever, -1};
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const bool take = key[i] > best.key;      // (a lane's experts ascend)
            best = Choice{take ? key[i] : best.key, take ? i * 64 + lane : best.expert};
        }
        best = FirstOfWave(best);
        taken = lane == j ? best.expert : taken;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            key[i] = i * 64 + lane == best.expert ? kNever : key[i];
        }
    }
    return taken;
}

// For the choice in 32 bits, which knows what it is off by.
__device__ __forceinline__ float Sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + Exp(-x)); }

// ---- the choice in 32 bits --------------------------------------------------------------------------------
// A score and its bias as a whole number: 1 + (s + b - least b) * times, below 2^22; 0 for an expert that cannot be chosen.  One step is
// (1 + largest b - least b) / 2^22.  With U = 2^-24, the difference b - least b, its product and the sum with s are each off by at most 2^22 U = 1/4 step,
// cutting off takes up to 1.  A sigmoid is off by
//   s (1 - s) (2 U |x| + 2 U)   the power's argument and the power         (|x| s (1 - s) < 0.23)
//   s (U + 2 U)                 the sum and the reciprocal
// which is 4 U, 1 step at most: two numbers are off against each other by twice 2.75.  A softmax's power, quotient and product are off by 5 U, and its sum, of 32 to a
// lane over 8 lanes or 16 over 64, by 50 U, the same for all of a token's: 60 U, 15 steps between two of them, and 3.5 for the rest.
// (What 64 bits would change is within these, cut off to whole numbers; sums of two are off by twice as much.)  Two numbers further apart than that are of scores that
// are a step and a half apart at least.  In 64 bits a score next to a bias b loses up to 2^-53 |b|, which the difference of biases here does not: from |b| = 2^24
// times the biases' range on, a 128th of a step, nothing is settled here, since equal large biases make scores equal there that are not here.
constexpr uint32_t kSlackSigmoid = 5, kSlackSoftmax = 18;

// DPP of the other lane of a pair, the other pair of four, the other four of eight, the other eight of sixteen (mirrored, where the lanes of each
// part are alike).
constexpr int kOther[4] = {0xb1, 0x4e, 0x141, 0x140};

template <int kWhich>
__device__ __forceinline__ uint32_t Other(uint32_t x)
{
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), kOther[kWhich], 0xf, 0xf, true));
}

template <int kWhich>
__device__ __forceinline__ float Other(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kOther[kWhich], 0xf, 0xf, true));
}

// f(v, the other's) step by step until the kLanes lanes of a token have the same.
template <int kLanes, typename V, typename F>
__device__ __forceinline__ V OverLanes(V v, F f)
{
    v = f(v, Other<0>(v));
    v = f(v, Other<1>(v));
    v = f(v, Other<2>(v));
    if constexpr (kLanes > 8) {
        v = f(v, Other<3>(v));
    }
    if constexpr (kLanes == 64) {
        v = f(v, __shfl_xor(v, 16, 64));
        v = f(v, __shfl_xor(v, 32, 64));
    }
    return v;
}

template <int kLanes, typename V>
__device__ __forceinline__ V AddLanes(V v)
{
    return OverLanes<kLanes>(v, [](V a, V b) { return a + b; });
}

template <int kLanes>
__device__ __forceinline__ float LargestOfLanes(float v)
{
    return OverLanes<kLanes>(v, [](float a, float b) { return Larger(a, b); });
}

// For weights and gradients: t = 1 / (1 + exp(-|x|)) and exp(-|x|) t, the sigmoids of |x| and -|x|.
struct Sigmoids {
    float large, small;
    __device__ __forceinline__ explicit Sigmoids(float x)
    {
        const float e = Power(-__builtin_fabsf(x), 0.0f);
        large = 1.0f / (1.0f + e);
        small = e * large;
    }
};

// A lane's share of its token's chosen scores, all of the token's by one factor, which is such that the largest is neither 0 nor infinite however small
// the scores are: with m the largest chosen logit exp(x - m), of a sigmoid exp(min(x, 0) - min(m, 0)) / (1 + exp(-|x|)).  0 where nothing is `chosen`.
template <int kLanes>
__device__ __forceinline__ float Share(float logit, bool chosen, bool softmax)
{
    const float x = softmax ? logit : __builtin_fminf(logit, 0.0f);
    const Difference d(x, LargestOfLanes<kLanes>(chosen ? x : -__builtin_inff()));
    const float s = Power(d.high, d.low);
    return chosen ? softmax ? s : s * Sigmoids(logit).large : 0.0f;
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

// The hardware's conversion: what is below 1, -inf and NaN become 0.
__device__ __forceinline__ uint32_t Whole(float x)
{
    uint32_t n;
    asm("v_cvt_u32_f32 %0, %1" : "=v"(n) : "v"(x));
    return n;
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

// What a launch's biases make of whole numbers.
struct Steps {
    float times;
    uint32_t slack;      // two numbers this close or closer need not be in their order
    bool fine;           // false: a bias is infinite or too large, everything is chosen in 64 bits
};

// The part of the numbers that the biases make, -inf where the bias is -inf or NaN, into LDS.  Called by all waves, which find out the same.
template <int kMost>
__device__ __forceinline__ Steps StepsOf(const ScoredArgs &a, float *part)
{
    Steps s{float((1 << 22) - 4), a.softmax ? kSlackSoftmax : kSlackSigmoid, true};
    float least = __builtin_inff(), most = -__builtin_inff();
    if (a.bias != nullptr) {
        bool infinite = false;
        for (int e = int(threadIdx.x) % 64; e < a.experts; e += 64) {
            const float b = a.bias[e];
            infinite = infinite || b == __builtin_inff();
            most = Larger(most, b);
            least = b > -__builtin_inff() && b < least ? b : least;
        }
        most = LargestOfLanes<64>(most);
        least = -LargestOfLanes<64>(-least);
        const float size = __builtin_fmaxf(__builtin_fabsf(most), __builtin_fabsf(least)), range = most - least;
        s.fine = __ballot(infinite) == 0 && range < __builtin_inff() && !(least <= most && size > 0x1p24f * (1.0f + range));
    }
    least = least <= most ? least : 0.0f;
    s.times = s.times / (1.0f + (most > least ? most - least : 0.0f));
    for (int e = threadIdx.x; e < kMost; e += kThreads) {
        const float b = a.bias != nullptr && e < a.experts ? a.bias[e] : 0.0f;
        part[e] = b > -__builtin_inff() ? __builtin_fmaf(b - least, s.times, 1.0f) : -__builtin_inff();
    }
    return s;
}

// Whether a group's experts are those of 1, 2, 4 or 8 neighbouring lanes.
__host__ __device__ constexpr bool Evenly(int size) { return size % 8 == 0 && size <= 64 && (size & (size - 1)) == 0; }

// Takes out what is not in a token's best groups.  Returns false where 32 bits do not settle which these are.  In LDS, the token's own: `numbers`,
// a place per expert; `of`, 64 places for groups.
template <int kLanes, int kEach, bool kEvenly>
__device__ __forceinline__ bool ChooseGroups(const ScoredArgs &a, uint32_t (&number)[kEach], uint32_t slack, int l, uint32_t *numbers, uint32_t *of)
{
    constexpr int kChunks = kEach / 8;
    // a group's number: the sum of its two largest, or the largest; then its place among the groups, so that no two are alike.  A group with
    // one choice or none left: its sum has a zero in it, which has no number here.
    const auto leave = [&](uint32_t g, uint32_t first, uint32_t next) {
        const uint32_t sum = !a.second ? first : next != 0 ? first + next : first != 0 ? (1u << 24) - 1 : 0;
        of[g] = sum << 6 | (63 - g);
    };
    if constexpr (kEvenly) {
        const int across = a.size / 8;        // lanes that share a group
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
            const int e = (c * kLanes + l) * 8;
            if ((l & (across - 1)) == 0 && e < a.experts) {
                leave(uint32_t(e) * a.perSize >> 20, first, next);
            }
        }
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
            leave(uint32_t(g), first, next);
        }
    }
    Ordered();
    // the number of the last group that is kept: those that reach it are
    uint32_t least = ~0u, most = 0;      // of the kept ones' numbers, of the others'
#pragma unroll 1
    for (int g = l; g < a.groups; g += kLanes) {
        const uint32_t mine = of[g];
        int before = 0;
#pragma unroll 1
        for (int o = 0; o < a.groups; o += 4) {
            // (places behind the last group's hold 0)
            const Word4 four = *reinterpret_cast<const Word4 *>(of + o);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                before += four[i] > mine ? 1 : 0;
            }
        }
        const bool kept = mine >= 64 && before < a.kept;
        least = kept ? Min(least, mine) : least;
        most = kept ? most : Max(most, mine);
        // (one choice among the two that are summed: not settled)
        most = a.second && mine >> 6 == (1u << 24) - 1 ? ~0u : most;
    }
    least = OverLanes<kLanes>(least, [](uint32_t x, uint32_t y) { return Min(x, y); });
    most = OverLanes<kLanes>(most, [](uint32_t x, uint32_t y) { return Max(x, y); });
    const auto kept = [&](int e) { return e < a.experts && of[uint32_t(e) * a.perSize >> 20] >= least; };
#pragma unroll
    for (int c = 0; c < kChunks; c++) {
        if constexpr (kEvenly) {
            const bool use = kept((c * kLanes + l) * 8);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                number[c * 8 + i] = use ? number[c * 8 + i] : 0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                number[c * 8 + i] = kept((c * kLanes + l) * 8 + i) ? number[c * 8 + i] : 0;
            }
        }
    }
    Ordered();
    return most < 64 || least >> 6 > (most >> 6) + (a.second ? 2 * slack + 1 : slack);
}

// The keys in 64 bits of two experts of a lane's token.
template <int kLanes, typename T>
__device__ __forceinline__ void Keys(const ScoredArgs &a, const T *row, float top, int l, Choice &own, Choice &more)
{
    const int at = min(own.expert, a.experts - 1), next = min(more.expert, a.experts - 1);
    double x = double(float(row[at])), y = double(float(row[next])), total = 1.0;
    const double b = a.bias != nullptr ? double(a.bias[at]) : 0.0, c = a.bias != nullptr ? double(a.bias[next]) : 0.0;
    if (a.softmax) {
        total = 0.0;
#pragma unroll 1
        for (int i = l; i < a.experts; i += kLanes) {
            const float v = float(row[i]);
            total += v <= top ? exp(double(v) - double(top)) : 0.0;
        }
#pragma unroll 1
        for (int d = 1; d < kLanes; d <<= 1) {
            total += __shfl_xor(total, d, 64);
        }
        x = double(top) - x;
        y = double(top) - y;
    }
    const double p = exp(-x), q = exp(-y);
    own.key = (a.softmax ? p / total : 1.0 / (1.0 + p)) + b;
    more.key = (a.softmax ? q / total : 1.0 / (1.0 + q)) + c;
}

// Whether all that reach the border and are not the token's own are made from the same logit and bias as the last of its own, and none of its own that is close
// to its neighbour from others than that: such experts tie in 64 bits too, and go by their numbers.  `mine`: lane j has the j-th.
template <int kLanes, int kEach, typename T>
__device__ __forceinline__ bool Ties(const ScoredArgs &a, const T *row, const uint32_t (&number)[kEach], uint32_t mine, uint32_t border, uint32_t room, int l, int lane)
{
    const int e = min(int(1023u - (mine & 1023u)), a.experts - 1);
    const float logit = float(row[e]), b = a.bias != nullptr ? a.bias[e] : 0.0f;
    const int from = lane - l + a.topK - 1;
    const float lastLogit = __shfl(logit, from, 64), lastBias = __shfl(b, from, 64);
    const uint32_t next = uint32_t(__shfl_down(int(mine), 1, 64));
    const float nextLogit = __shfl_down(logit, 1, 64), nextBias = __shfl_down(b, 1, 64);
    const uint32_t pairs = AddLanes<kLanes>(l + 1 < a.topK && mine - next <= room && !(logit == nextLogit && b == nextBias) ? 1u : 0u);
    const uint32_t listed = AddLanes<kLanes>(l < a.topK && mine >= border && !(logit == lastLogit && b == lastBias) ? 1u : 0u);
    uint32_t others = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        if (number[i] >= border) {
            const int at = ExpertOf<kLanes>(i, l);
            others += !(float(row[at]) == lastLogit && (a.bias == nullptr || a.bias[at] == lastBias)) ? 1 : 0;
        }
    }
    others = AddLanes<kLanes>(others);
    return pairs == 0 && others == listed;
}

// The choice in 32 bits.  Returns false where they do not settle it, on some of the token's lanes.  Of a softmax also the row's largest logit and the sum of
// the powers, NaN where a logit is NaN or +inf.
template <int kLanes, int kEach, int K, bool kEvenly, typename T>
__device__ __forceinline__ bool ChooseFast(const ScoredArgs &a, const Steps &steps, const float (&x)[kEach], const float *part, const T *row, bool in, int l,
    int lane, uint32_t *numbers, uint32_t *of, int (&chosen)[K], float &top, float &sum)
{
    uint32_t number[kEach];
    float largest = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        largest = __builtin_fmaxf(largest, x[i]);      // (leaves NaN out)
    }
    // from eight scores, in units of `by`, NaN where the logit is infinite or NaN
    const auto make = [&](int c, const float (&s)[8], float by) {
        float p[8];
        Load<true, 8>(part + (c * kLanes + l) * 8, p);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            number[c * 8 + i] = Whole(__builtin_fmaf(s[i], by, p[i]));
        }
    };
    if (a.softmax) {
        float s[kEach];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            bad = bad || !(x[i] < __builtin_inff());
        }
        top = OverLanes<kLanes>(largest, [](float u, float v) { return __builtin_fmaxf(u, v); });
        // (+inf takes all, a NaN is left out)
        float sums[4] = {};
        if (a.renormalise) {
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                s[i] = Exp(x[i] == top ? 0.0f : x[i] - top);
            }
        } else {
            // (their sum divides the weights: powers that lose nothing of their arguments; where the largest is infinite, NaN, which says nothing then: -inf
            // leaves no choice, with +inf the weights are NaN and 64 bits choose)
            const float most = Anew(top);      // (the differences are not worked out in front of both branches, where registers would have to hold them)
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                const Difference d(x[i], most);
                s[i] = Power(d.high, d.low);
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            s[i] = x[i] <= top ? s[i] : 0.0f;
            sums[i % 4] += s[i];
            s[i] = __builtin_fmaf(x[i], 0.0f, s[i]);
        }
        sum = AddLanes<kLanes>((sums[0] + sums[1]) + (sums[2] + sums[3]));
        const float by = steps.times / sum;
        sum = AddLanes<kLanes>(bad ? 1.0f : 0.0f) > 0.0f ? __builtin_nanf("") : sum;
#pragma unroll
        for (int c = 0; c < kEach / 8; c++) {
            float eight[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                eight[i] = s[c * 8 + i];
            }
            make(c, eight, by);
        }
    } else {
#pragma unroll
        for (int c = 0; c < kEach / 8; c++) {
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                s[i] = __builtin_fmaf(x[c * 8 + i], 0.0f, Sigmoid(x[c * 8 + i]));
            }
            make(c, s, steps.times);
        }
    }
    bool sure = !(largest == __builtin_inff());       // (+inf can be chosen, but not like this)
    if (a.groups > 1) {
        const bool settled = ChooseGroups<kLanes, kEach, kEvenly>(a, number, steps.slack, l, numbers, of);
        sure = sure && settled;
    }
    // a word is a number and the expert, complemented; below kLeast there is no choice in it
    constexpr uint32_t kLeast = 1024;
    uint32_t best[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        best[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        number[i] = number[i] << 10 | (1023u - uint32_t(ExpertOf<kLanes>(i, l)));
#pragma unroll
        for (int k = K - 1; k > 0; k--) {
            if (k <= i) {      // (the first ones meet empty places)
                best[k] = k < i ? Median(best[k - 1], best[k], number[i]) : Min(best[k - 1], number[i]);
            }
        }
        best[0] = Max(best[0], number[i]);
    }
    MergeOther<0>(best);
    MergeOther<1>(best);
    MergeOther<2>(best);
    if constexpr (kLanes > 8) {
        MergeOther<3>(best);
    }
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
    uint32_t last = 0, gap = ~0u;
#pragma unroll
    for (int i = 0; i < K; i++) {
        last = i + 1 == a.topK ? best[i] : last;
        if (i + 1 < K) {
            gap = i + 1 < a.topK ? Min(gap, best[i] - best[i + 1]) : gap;
        }
    }
    uint32_t beyond = ~0u;        // how far below the last one the next of the others is (those above it wrap round)
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        beyond = Min(beyond, last - 1 - number[i]);
    }
    beyond = OverLanes<kLanes>(beyond, [](uint32_t u, uint32_t v) { return Min(u, v); });
    const bool close = in && sure && (gap <= room || beyond < room);
    sure = sure && last >= kLeast;
    if (__ballot(close) != 0) {
        // lane j has the j-th
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < K; i++) {
            mine = l == i ? best[i] : mine;
        }
        const uint32_t border = last >= kLeast + room ? last - room : kLeast, extra = last - 1 - beyond;      // the next of the others
        uint32_t above = 0;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            above += number[i] >= border ? 1 : 0;
        }
        above = AddLanes<kLanes>(above);
        const bool few = sure && above <= uint32_t(a.topK) + 1;
        if (__ballot(close && !few) != 0) {
            const bool ties = Ties<kLanes>(a, row, number, mine, border, room, l, lane);
            sure = sure && (!close || few || ties);
        }
        if (__ballot(close && few) != 0) {
            // between these and one more by their keys in 64 bits
            Choice own{kNever, int(1023u - (mine & 1023u))}, more{kNever, int(1023u - (extra & 1023u))};
            Keys<kLanes>(a, row, top, l, own, more);
            // (without another one within reach its key says nothing)
            more.key = above > uint32_t(a.topK) ? more.key : kNever;
            int place = 0;
            for (int i = 0; i < a.topK; i++) {
                const Choice other{__shfl(own.key, lane - l + i, 64), __shfl(own.expert, lane - l + i, 64)};
                place += Before(other, own) ? 1 : 0;
            }
            // the one more moves back what it goes before, and goes where they were
            const bool after = l < a.topK && Before(more, own);
            const int moved = int(AddLanes<kLanes>(after ? 1u : 0u));
            place += after ? 1 : 0;
#pragma unroll
            for (int i = 0; i < K; i++) {
                const uint32_t word = AddLanes<kLanes>(l < a.topK && place == i ? mine : 0u);
                best[i] = close && few && i < a.topK ? (moved > 0 && i == a.topK - moved ? extra : word) : best[i];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < K; i++) {
        chosen[i] = i < a.topK && in && best[i] >= kLeast ? int(1023u - (best[i] & 1023u)) : -1;
    }
    return sure || !in;
}

template <typename T, int K, int kLanes, int kEach, bool kEvenly>
__global__ void __launch_bounds__(kThreads, kLanes == 64 ? 2 : 4) ScoredKernel(ScoredArgs args)
{
    ScoredArgs a = args;
    constexpr int kWaveTokens = 64 / kLanes, kTile = kWaveTokens * kThreads / 64;
    extern __shared__ uint32_t lds[];
    const int E = a.experts;
    uint32_t *chose = lds;                                                // [experts]: one bit per token of the tile
    int *count = reinterpret_cast<int *>(chose + E);                      // [experts]: rows of the tiles so far
    int *parts = count + E;                                               // [waves]
    int *routed = parts + kThreads / 64;                                  // [1]
    __shared__ double groupKeys[kThreads / 64][HCCL_AMD_MAX_EXPERT_GROUPS];
    __shared__ double keys[kThreads / 64][kLanes * kEach];
    __shared__ __align__(16) uint32_t groupNumbers[kTile][HCCL_AMD_MAX_EXPERT_GROUPS];
    uint32_t *numbers = reinterpret_cast<uint32_t *>(routed + 1);         // [tokens of the tile][experts], for groups that lanes do not share evenly

    const int wave = int(threadIdx.x) / 64;
    for (int e = threadIdx.x; e < E; e += kThreads) {
        chose[e] = 0;
        count[e] = 0;
    }
    if (threadIdx.x == 0) {
        *routed = 0;
    }
    for (int i = threadIdx.x; i < kTile * int(HCCL_AMD_MAX_EXPERT_GROUPS); i += kThreads) {
        groupNumbers[0][i] = 0;
    }
    __shared__ __align__(16) float part[kLanes * kEach];
    const Steps steps = StepsOf<kLanes * kEach>(a, part);
    __syncthreads();
    int rank = -1, taken = -1;      // the last tile's
    for (int tile = 0; tile < a.tiles; tile++) {
        a.topK = AnewForAll(args.topK);
        const int lane = Anew(int(threadIdx.x) % 64), l = lane % kLanes, r = wave * kWaveTokens + lane / kLanes;
        const int token = (int(blockIdx.x) * a.tiles + tile) * kTile + r;
        const bool in = token < a.tokens && (a.mask == nullptr || a.mask[token] != 0);
        // (the row of a token that takes no part is read and forgotten)
        const T *row = static_cast<const T *>(a.logits) + int64_t(min(token, max(a.tokens - 1, 0))) * a.stride;
        float x[kEach];
#pragma unroll
        for (int c = 0; c < kEach / 8; c++) {
            float v[8];
            LoadPart<kAnyhow, 8>(row, (c * kLanes + l) * 8, a.tokens > 0 ? E : 0, v, -__builtin_inff());
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c * 8 + i] = v[i];
            }
        }
        int chosen[K];
        float top = 0.0f, total = 0.0f;
        const bool settled = ChooseFast<kLanes, kEach, K, kEvenly>(a, steps, x, part, row, in, l, lane, numbers + r * E, groupNumbers[r], chosen, top, total);
        const bool sure = steps.fine && settled;
        unsigned long long unsure = __ballot(in && !sure);
        while (unsure != 0) {
            const int which = (__ffsll(unsure) - 1) / kLanes, whose = (int(blockIdx.x) * a.tiles + tile) * kTile + wave * kWaveTokens + which;
            const int best = ChooseExactly<kLanes * kEach / 64, T>(ExactArgs{a.bias, a.experts, a.topK, a.groups, a.kept, a.size, a.perSize, a.softmax, a.second},
                static_cast<const T *>(a.logits) + int64_t(whose) * a.stride, keys[wave], groupKeys[wave]);
#pragma unroll
            for (int i = 0; i < K; i++) {
                const int exactly = __builtin_amdgcn_readlane(best, i);
                chosen[i] = lane / kLanes == which ? exactly : chosen[i];
            }
            unsure &= ~(kLanes == 64 ? ~0ull : ((1ull << kLanes % 64) - 1) << which * kLanes);
        }
        // lane j of a token has its j-th choice
        int mine = -1;
#pragma unroll
        for (int i = 0; i < K; i++) {
            mine = l == i ? chosen[i] : mine;
        }
        const float logit = mine >= 0 ? float(row[mine]) : -__builtin_inff();
        float w;
        constexpr int kHold = kLanes < 16 ? kLanes : 16;      // lanes that hold choices
        if (a.renormalise) {
            w = Share<kHold>(logit, mine >= 0, a.softmax);
            w /= AddLanes<kHold>(w);
        } else if (a.softmax) {
            const Difference d(logit, top);
            w = Power(d.high, d.low) / total;
        } else {
            const Sigmoids s(logit);
            w = logit < 0.0f ? s.small : s.large;
        }
        // (a NaN or +inf in a softmax's row: the weights are NaN, chosen or not by these)
        w = !a.softmax || total > 0.0f ? w : __builtin_nanf("");
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
        if (writes) {
            a.rowOf[at] = place;
        }
        rank = writes ? place : -1;
        taken = mine;
    }
    if (a.blocks == 1) {
        // a single workgroup, which has a single tile: its places become rows at once
        Finish<kThreads, false>(a, count, nullptr, *routed, parts, nullptr, true);
        if (rank >= 0) {
            const int lane = int(threadIdx.x) % 64;
            a.rowOf[(wave * kWaveTokens + lane / kLanes) * a.topK + lane % kLanes] = rank + count[taken];
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
                const Difference d(x[i], top);
                x[i] = Power(d.high, d.low);
                sum += x[i];
            }
            const float by = 1.0f / AddNeighbours<kLanes>(sum);
            const Difference d(logit, top);
            more = chosen >= 0 ? Power(d.high, d.low) * by * dw : 0.0f;
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
            // (what crosses lanes stands outside of what only some of them do; 1 - s is the sigmoid of -x)
            const Sigmoids of(logit);
            if (a.renormalise) {
                const float share = Share<16>(logit, chosen >= 0, a.softmax), w = share / AddNeighbours<16>(share);
                const float mean = AddNeighbours<16>(chosen >= 0 ? w * dw : 0.0f);
                more = w * (dw - mean);
                more = a.softmax ? more : more * (logit < 0.0f ? of.large : of.small);
            } else {
                more = of.large * of.small * dw;
            }
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

// Lanes to a token.  All launches, with eight lanes and with sixteen, 60 experts (fp32, softmax) and 256 (16 bits, sigmoid): 2048 tokens 18.1 and 17.2 us, 18.3 and 17.2; 4097 18.4
// and 17.5, 20.0 and 19.1; 6500 18.5 and 18.1, 21.7 and 21.9; 8192 18.6 and 18.2, 22.0 and 22.3; 16384 19.6 and 21.6, 24.4 and 26.0; 32768 22.8 and 30.0, 31.1 and 34.1.  (Between 4097 tokens and about 7000
// sixteen would be up to 5 % quicker.)
int LanesOf(uint64_t tokens, uint32_t experts, uint32_t topK) { return experts > 256 ? 64 : topK > 8 || tokens <= 4096 ? 16 : 8; }

int TileOf(uint64_t tokens, uint32_t experts, uint32_t topK) { return kThreads / LanesOf(tokens, experts, topK); }

// Tiles to a workgroup: one, until there are as many workgroups as the launches behind take.  (64 tokens by four workgroups and a launch that joins them take
// 11 us; by one workgroup and no such launch they took 18 when four took 13.)
int TilesEach(uint64_t tokens, int tile)
{
    const uint64_t tiles = (tokens + uint64_t(tile) - 1) / uint64_t(tile);
    return tiles == 0 ? 1 : int((tiles + kMostBlocks - 1) / kMostBlocks);
}

int Workgroups(uint64_t tokens, int tile)
{
    const uint64_t each = uint64_t(tile) * uint64_t(TilesEach(tokens, tile));
    return tokens == 0 ? 1 : int((tokens + each - 1) / each);
}

template <typename T, int K, int kLanes, int kEach>
HcclResult LaunchScored(const ScoredArgs &a, hipStream_t stream)
{
    const size_t lds = 4 * (2 * size_t(a.experts) + kThreads / 64 + 1 + (a.groups == 1 || Evenly(a.size) ? 0 : kThreads / kLanes * size_t(a.experts)));
    const auto go = [&](auto kernel) { return Launch("HcclAmdExpertRouteScored", kernel, uint32_t(a.blocks), kThreads, lds, stream, a); };
    return a.groups == 1 || Evenly(a.size) ? go(ScoredKernel<T, K, kLanes, kEach, true>) : go(ScoredKernel<T, K, kLanes, kEach, false>);
}

template <typename T>
HcclResult LaunchScoredType(const ScoredArgs &a, int lanes, hipStream_t stream)
{
    if (lanes == 8) {
        return a.experts <= 64    ? LaunchScored<T, 8, 8, 8>(a, stream)
               : a.experts <= 128 ? LaunchScored<T, 8, 8, 16>(a, stream)
                                  : LaunchScored<T, 8, 8, 32>(a, stream);
    }
    if (lanes == 64) {
        return a.topK <= 8 ? LaunchScored<T, 8, 64, 16>(a, stream) : LaunchScored<T, 16, 64, 16>(a, stream);
    }
    if (a.topK <= 8) {
        return a.experts <= 128 ? LaunchScored<T, 8, 16, 8>(a, stream) : LaunchScored<T, 8, 16, 16>(a, stream);
    }
    return a.experts <= 128 ? LaunchScored<T, 16, 16, 8>(a, stream) : LaunchScored<T, 16, 16, 16>(a, stream);
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
    // (whatever topK will be)
    const uint64_t few = uint64_t(Workgroups(tokens, TileOf(tokens, experts, 1))), many = uint64_t(Workgroups(tokens, TileOf(tokens, experts, HCCL_AMD_MAX_TOPK)));
    const uint64_t blocks = few > many ? few : many;
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
    const int tile = TileOf(tokens, experts, topK);
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
    a.tiles = TilesEach(tokens, tile);
    a.blocks = Workgroups(tokens, tile);       // no token: the one workgroup writes the zeros
    a.blockCounts = static_cast<int32_t *>(workspace);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    HcclResult r = logitType == HCCL_DATA_TYPE_FP32   ? LaunchScoredType<float>(a, kThreads / tile, on)
                   : logitType == HCCL_DATA_TYPE_FP16 ? LaunchScoredType<_Float16>(a, kThreads / tile, on)
                                                      : LaunchScoredType<__bf16>(a, kThreads / tile, on);
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
