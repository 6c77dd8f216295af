// Router of an expert-parallel layer: the topK largest logits of every token, their weights, rows in expert order, per-expert
// counts and the balance loss; and the gradient of all that.
//
// With p = softmax(x) over a token's experts, n_e the tokens that chose e, A their sum, T the tokens that chose any:
//   loss = c E sum_e (n_e / A) (sum_t p_te / T)       d loss / d p_te = c E n_e / (A T)
//   w_j = p_j, or p_j / sum of the chosen p           dx = p (g - sum p g), and for the quotient w_j (dw_j - sum_i w_i dw_i)
//
// The logits are read once, into registers, a token's by several lanes.  Every lane keeps the topK largest of its experts as a
// sorted list: a new one is put in without exchanges between lanes -- for 16-bit logits value and expert share a word, and one
// median of three per entry does it -- and the lists of a token's lanes are merged at the end.  Which tokens of a tile of 64 chose an
// expert is a mask of one bit per token: set with LDS atomics whose order cannot matter, its bits counted in front of a token give the
// token's place, so that counts and rows are the same in every run.  A workgroup goes through several tiles and leaves its counts and
// probability sums in the workspace; a second launch adds up what lies in front of every workgroup's, a third adds that to the
// rows (up to 512 tokens the third does both).  Up to 64 tokens (a decoding step) one launch does it all.
//
// Measured: 65536 tokens of 256 experts, eight chosen, 16-bit logits (33.5 MB): 21 us to choose, 7 to add up, 5 for the rows, 20 for the
// gradient (67 MB); 32-bit logits 49 us in all and 26 for the gradient.  Choosing is bound by vector instructions (their unit is busy 88 % of the
// time), not by the 7 us its bytes take: 64 logits a lane, 35 instructions each, of which the eight medians are less than a quarter; the others map
// values, take exponentials and add up.  The gradient keeps that unit busy 56 % of the time and waits on one chain of dependent steps a token; the
// rest is the latency of few dependent accesses.  One token: 7 us, the latency of one wave's way through the code.
#include <type_traits>

#include "common.h"

namespace hcclamd {
namespace experts {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kNone = 0xffffffffu;
constexpr uint64_t kMaxTokens = uint64_t(1) << 25;

struct RouteArgs {
    const void *logits;
    const uint8_t *mask;
    int32_t *expertOf;
    float *weights;
    int32_t *rowOf;
    int32_t *counts;
    int32_t *offsets;
    float *loss;
    int32_t *blockCounts;  // [blocks][experts + 1]: rows per expert; last column: tokens that chose
    float *blockSums;      // [blocks][experts]: sum of probabilities
    float *sums;           // [experts]
    int64_t stride;
    int tokens, experts, topK;
    int blocks, tiles;     // workgroups; tiles of each
    float lossScale;
    bool renormalise;
};

// exp of a difference to the row's maximum.  Its argument, at most 0, is rounded twice, which moves a probability by 2^-24 of
// the difference; the hardware's power of two is good to one unit.
__device__ __forceinline__ float Exp(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }

// ---- sorted lists of the K largest ------------------------------------------------------------------------
// Ordered by value, then by lower expert.  An empty place precedes nothing; -inf and NaN are never put in.

// 16-bit logits: a word of the value, mapped to an unsigned number of the same order, and the expert, complemented.  0: empty.
template <int K>
struct WordList {
    uint32_t best[K];

    __device__ __forceinline__ WordList()
    {
#pragma unroll
        for (int i = 0; i < K; i++) {
            best[i] = 0;
        }
    }
    template <typename T>
    __device__ __forceinline__ void Put(float v, uint32_t expert)
    {
        // (v + 0: both zeros are one value)
        uint32_t bits;     // of the logit, in the upper half
        if constexpr (std::is_same_v<T, __bf16>) {
            bits = __float_as_uint(v + 0.0f);
        } else {
            bits = uint32_t(__builtin_bit_cast(uint16_t, T(v + 0.0f))) << 16;
        }
        const uint32_t order = bits ^ (uint32_t(int32_t(bits) >> 31) | 0x80000000u);
        const uint32_t word = v > -__builtin_inff() ? (order & 0xffff0000u) | (0xffffu - expert) : 0;
        // of a sorted list and a new word the i-th is the median of the (i - 1)-th, the i-th and the new one
#pragma unroll
        for (int i = K - 1; i > 0; i--) {
            asm("v_med3_u32 %0, %1, %2, %3" : "=v"(best[i]) : "v"(best[i - 1]), "v"(best[i]), "v"(word));
        }
        best[0] = best[0] > word ? best[0] : word;
    }
    __device__ __forceinline__ void Clear()
    {
#pragma unroll
        for (int i = 0; i < K; i++) {
            best[i] = 0;
        }
    }
    // The larger half of two lists: element by element against the other one backwards, which leaves a sequence that rises and falls
    // once, then sorted by halving.
    __device__ __forceinline__ void Merge(int lanes)
    {
        uint32_t other[K];
#pragma unroll
        for (int i = 0; i < K; i++) {
            other[i] = __shfl_xor(best[i], lanes, 64);
        }
#pragma unroll
        for (int i = 0; i < K; i++) {
            best[i] = best[i] > other[K - 1 - i] ? best[i] : other[K - 1 - i];
        }
#pragma unroll
        for (int d = K / 2; d > 0; d >>= 1) {
#pragma unroll
            for (int i = 0; i < K; i++) {
                if ((i & d) == 0) {
                    const uint32_t hi = best[i] > best[i + d] ? best[i] : best[i + d], lo = best[i] > best[i + d] ? best[i + d] : best[i];
                    best[i] = hi;
                    best[i + d] = lo;
                }
            }
        }
    }
    template <typename T>
    __device__ __forceinline__ float Value(int i) const
    {
        const uint32_t order = best[i] >> 16;
        return float(__builtin_bit_cast(T, uint16_t(order ^ ((order & 0x8000u) != 0 ? 0x8000u : 0xffffu))));
    }
    __device__ __forceinline__ uint32_t Expert(int i) const { return best[i] == 0 ? kNone : 0xffffu - (best[i] & 0xffffu); }
};

// 32-bit logits: value and expert apart.
template <int K>
struct PairList {
    float v[K];
    uint32_t e[K];

    __device__ __forceinline__ PairList()
    {
#pragma unroll
        for (int i = 0; i < K; i++) {
            v[i] = -__builtin_inff();
            e[i] = kNone;
        }
    }
    __device__ __forceinline__ void Clear() { *this = PairList(); }
    // No instruction.  Without it the compiler reasons about chains of dozens of selects as one, for hours.
    __device__ __forceinline__ void Settle(int i) { asm("" : "+v"(v[i]), "+v"(e[i])); }

    // x goes behind the last entry that is not less, those after it move on.  A lane's experts come in ascending order: of
    // equal values the one that is there stays in front (and NaN, greater than nothing, is never put in).
    template <typename T>
    __device__ __forceinline__ void Put(float x, uint32_t expert)
    {
        bool ahead = x > v[K - 1];
#pragma unroll
        for (int i = K - 1; i > 0; i--) {
            const bool further = x > v[i - 1];
            v[i] = further ? v[i - 1] : ahead ? x : v[i];
            e[i] = further ? e[i - 1] : ahead ? expert : e[i];
            ahead = further;
        }
        v[0] = ahead ? x : v[0];
        e[0] = ahead ? expert : e[0];
    }
    __device__ __forceinline__ void Merge(int lanes)
    {
        float ov[K];
        uint32_t oe[K];
#pragma unroll
        for (int i = 0; i < K; i++) {
            ov[i] = __shfl_xor(v[i], lanes, 64);
            oe[i] = __shfl_xor(e[i], lanes, 64);
        }
#pragma unroll
        for (int i = 0; i < K; i++) {
            const int j = K - 1 - i;
            const bool take = ov[j] > v[i] || (ov[j] == v[i] && oe[j] < e[i]);
            v[i] = take ? ov[j] : v[i];
            e[i] = take ? oe[j] : e[i];
            Settle(i);
        }
#pragma unroll
        for (int d = K / 2; d > 0; d >>= 1) {
#pragma unroll
            for (int i = 0; i < K; i++) {
                if ((i & d) == 0) {
                    const bool swap = v[i + d] > v[i] || (v[i + d] == v[i] && e[i + d] < e[i]);
                    const float hv = swap ? v[i + d] : v[i], lv = swap ? v[i] : v[i + d];
                    const uint32_t he = swap ? e[i + d] : e[i], le = swap ? e[i] : e[i + d];
                    v[i] = hv;
                    e[i] = he;
                    v[i + d] = lv;
                    e[i + d] = le;
                    Settle(i);
                    Settle(i + d);
                }
            }
        }
    }
    template <typename T>
    __device__ __forceinline__ float Value(int i) const { return v[i]; }
    __device__ __forceinline__ uint32_t Expert(int i) const { return e[i]; }
};

template <typename T, int K>
using List = std::conditional_t<sizeof(T) == 2, WordList<K>, PairList<K>>;

// ---- sums ------------------------------------------------------------------------------------------------

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

// Exclusive prefix sums of n <= 1024 values in LDS, in place, by kThreads threads; returns the total.  `part`: a word per wave.
template <int kThreads>
__device__ __forceinline__ int Scan(int *values, int n, int *part)
{
    const int per = (n + kThreads - 1) / kThreads, from = min(n, int(threadIdx.x) * per), to = min(n, from + per);
    int mine = 0;
    for (int i = from; i < to; i++) {
        mine += values[i];
    }
    const int lane = int(threadIdx.x) % 64;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int other = __shfl_up(sum, d, 64);
        sum += lane >= d ? other : 0;
    }
    if (lane == 63) {
        part[threadIdx.x / 64] = sum;
    }
    __syncthreads();
    int at = sum - mine, total = 0;
    for (int w = 0; w < kThreads / 64; w++) {
        at += w < int(threadIdx.x) / 64 ? part[w] : 0;
        total += part[w];
    }
    for (int i = from; i < to; i++) {
        const int v = values[i];
        values[i] = at;
        at += v;
    }
    __syncthreads();
    return total;
}

// counts[experts + 1], offsets and the loss (`write`) from per-expert counts and sums in LDS; afterwards `count` holds the offsets.
template <int kThreads>
__device__ __forceinline__ void Finish(const RouteArgs &a, int *count, const float *sum, int tokens, int *part, float *partSum, bool write)
{
    float load = 0.0f;
    for (int e = threadIdx.x; e < a.experts && write; e += kThreads) {
        load += float(count[e]) * sum[e];
        a.counts[e] = count[e];
    }
    load = AddNeighbours<64>(load);
    if (threadIdx.x % 64 == 0) {
        partSum[threadIdx.x / 64] = load;
    }
    __syncthreads();
    const int rows = Scan<kThreads>(count, a.experts, part);
    if (!write) {
        return;
    }
    for (int e = threadIdx.x; e < a.experts; e += kThreads) {
        a.offsets[e] = count[e];
    }
    if (threadIdx.x == 0) {
        float all = 0.0f;
        for (int w = 0; w < kThreads / 64; w++) {
            all += partSum[w];
        }
        a.counts[a.experts] = tokens;
        a.offsets[a.experts] = rows;
        a.loss[0] = rows == 0 ? 0.0f : a.lossScale * float(a.experts) * (all / float(rows) / float(tokens));
    }
}

// One step of adding up over lanes and sharing out the sums: of 2 kHalf values a lane keeps the half that its bit names, and adds what
// its partner, whose bit is the other one, has of it.  kDpp: how lanes are exchanged.
template <int kDpp, int kHalf, int kEach>
__device__ __forceinline__ void AddAndShare(float (&v)[kEach], bool upper)
{
#pragma unroll
    for (int i = 0; i < kHalf; i++) {
        const float keep = upper ? v[i + kHalf] : v[i], give = upper ? v[i] : v[i + kHalf];
        v[i] = keep + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(give), kDpp, 0xf, 0xf, true));
    }
}

// A tile's probabilities, added up over a wave's tokens, into the wave's own sums in LDS.  Partners' numbers differ in the bits 15, 7, 3
// and 1 (mirrored rows and halves of rows, quads turned round), which reach all 16 lanes.
template <int kWaveTokens, int kLanes, int kEach>
__device__ __forceinline__ void Columns(float (&p)[kEach], float *sum, int experts, int lane, int wave, int l)
{
    constexpr int kQuarter = kWaveTokens == 16 ? kEach / 4 : kEach, kMine = kEach / kWaveTokens;
    static_assert(kMine >= 1, "a sum to a lane at least");
    if constexpr (kWaveTokens == 16) {
        AddAndShare<0x140, kEach / 2>(p, (lane & 8) != 0);
        AddAndShare<0x141, kEach / 4>(p, (lane & 4) != 0);
    }
    AddAndShare<0x1b, kQuarter / 2>(p, (lane & 2) != 0);
    AddAndShare<0xb1, kQuarter / 4>(p, (lane & 1) != 0);
    const int first = lane % kWaveTokens * kMine;     // (the highest bit has chosen between the halves of all)
#pragma unroll
    for (int i = 0; i < kMine; i++) {
        const int at = first + i, e = (at / 8 * kLanes + l) * 8 + at % 8;
        if (e < experts) {
            sum[wave * experts + e] += p[i];
        }
    }
}

// The waves' sums into the first one's.
__device__ __forceinline__ void AddWaves(float *sum, int experts)
{
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kThreads) {
        float s = sum[e];
        for (int w = 1; w < kThreads / 64; w++) {
            s += sum[w * experts + e];
        }
        sum[e] = s;
    }
    __syncthreads();
}

// kLanes lanes to a token, each with kChunks times eight neighbouring experts; lists of K.  Token t of a wave's 64 / kLanes is in
// the lanes whose number leaves t.
template <typename T, int K, int kLanes, int kChunks, int kHow>
__global__ void __launch_bounds__(kThreads) RouteKernel(RouteArgs a)
{
    constexpr int kWaveTokens = 64 / kLanes, kTile = kWaveTokens * kThreads / 64, kEach = 8 * kChunks;
    extern __shared__ uint32_t lds[];
    const int E = a.experts;
    uint32_t *chose = lds;                                                // [experts][2]: one bit per token of the tile
    int *count = reinterpret_cast<int *>(chose + 2 * E);                  // [experts]: rows of the tiles so far
    float *sum = reinterpret_cast<float *>(count + E);                    // [waves][experts]
    int *part = reinterpret_cast<int *>(sum + kThreads / 64 * E);         // [waves]
    float *partSum = reinterpret_cast<float *>(part + kThreads / 64);     // [waves]
    int *routed = reinterpret_cast<int *>(partSum + kThreads / 64);       // [1]

    const int lane = int(threadIdx.x) % 64, wave = int(threadIdx.x) / 64, l = lane / kWaveTokens, r = wave * kWaveTokens + lane % kWaveTokens;
    for (int e = threadIdx.x; e < E; e += kThreads) {
        chose[2 * e] = chose[2 * e + 1] = 0;
        count[e] = 0;
        for (int w = 0; w < kThreads / 64; w++) {
            sum[w * E + e] = 0.0f;
        }
    }
    if (threadIdx.x == 0) {
        *routed = 0;
    }
    __syncthreads();
    for (int tile = 0; tile < a.tiles; tile++) {
        const int token = (int(blockIdx.x) * a.tiles + tile) * kTile + r;
        const bool in = token < a.tokens && (a.mask == nullptr || a.mask[token] != 0);
        // (the row of a token that takes no part is read and forgotten)
        const T *row = static_cast<const T *>(a.logits) + int64_t(min(token, max(a.tokens - 1, 0))) * a.stride;
        float x[kEach];
        List<T, K> best;
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
            float v[8];
            LoadPart<kHow, 8>(row, (c * kLanes + l) * 8, a.tokens > 0 ? E : 0, v, -__builtin_inff());
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[c * 8 + i] = v[i];
            }
        }
#pragma unroll
        for (int c = 0; c < kChunks; c++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                best.template Put<T>(x[c * 8 + i], uint32_t((c * kLanes + l) * 8 + i));
            }
        }
#pragma unroll 1
        for (int d = kWaveTokens; d < 64; d <<= 1) {
            best.Merge(d);
        }
        if (!in) {
            best.Clear();
        }
        const bool any = best.Expert(0) != kNone;
        const float top = any ? best.template Value<T>(0) : 0.0f;
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            x[i] = Exp(x[i] - top);
            total += x[i];
        }
#pragma unroll
        for (int d = kWaveTokens; d < 64; d <<= 1) {
            total += __shfl_xor(total, d, 64);
        }
        // (a token that chose nothing adds nothing to the sums, whatever its row holds)
        const float times = 1.0f / total;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            x[i] = any ? x[i] * times : 0.0f;
        }
        Columns<kWaveTokens, kLanes>(x, sum, E, lane, wave, l);
        float inside = 0.0f, weight[K];
#pragma unroll
        for (int i = 0; i < K; i++) {
            weight[i] = i < a.topK && best.Expert(i) != kNone ? Exp(best.template Value<T>(i) - top) : 0.0f;
            inside += weight[i];
        }
        const bool bad = !(total < __builtin_inff());   // a NaN or +inf in the row: its weights are NaN, chosen or not by these
        const float by = bad ? __builtin_nanf("") : a.renormalise ? 1.0f / inside : times;
        if (any && l == 0) {
            atomicAdd(routed, 1);   // a whole number: the order does not matter
        }
        if (token < a.tokens) {
#pragma unroll
            for (int i = 0; i < K; i++) {
                if (i < a.topK && i % kLanes == l) {
                    const int64_t at = int64_t(token) * a.topK + i;
                    const uint32_t e = best.Expert(i);
                    a.expertOf[at] = int32_t(e);      // (kNone is -1)
                    a.weights[at] = e != kNone ? weight[i] * by : 0.0f;
                    if (e != kNone) {
                        atomicOr(&chose[2 * e + (r >> 5)], 1u << (r & 31));
                    }
                }
            }
        }
        __syncthreads();
        // a choice's place among the workgroup's rows of its expert
        int32_t place[K];
#pragma unroll
        for (int i = 0; i < K; i++) {
            place[i] = -1;
            const uint32_t e = best.Expert(i);
            if (i < a.topK && i % kLanes == l && e != kNone && token < a.tokens) {
                const uint32_t low = chose[2 * e], high = chose[2 * e + 1];
                place[i] = count[e] + (r < 32 ? __popc(low & ((1u << r) - 1)) : __popc(low) + __popc(high & ((1u << (r - 32)) - 1)));
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < E; e += kThreads) {
            count[e] += __popc(chose[2 * e]) + __popc(chose[2 * e + 1]);
            chose[2 * e] = chose[2 * e + 1] = 0;
        }
        __syncthreads();
        if (a.blocks == 1 && tile + 1 == a.tiles) {
            // a single workgroup: its places become rows at once
            AddWaves(sum, E);
            Finish<kThreads>(a, count, sum, *routed, part, partSum, true);
        }
        if (token < a.tokens) {
#pragma unroll
            for (int i = 0; i < K; i++) {
                if (i < a.topK && i % kLanes == l) {
                    const bool last = a.blocks == 1 && tile + 1 == a.tiles;
                    a.rowOf[int64_t(token) * a.topK + i] = place[i] < 0 ? -1 : place[i] + (last ? count[best.Expert(i)] : 0);
                }
            }
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
    AddWaves(sum, E);
    for (int e = threadIdx.x; e < E; e += kThreads) {
        a.blockCounts[int64_t(blockIdx.x) * (E + 1) + e] = count[e];
        a.blockSums[int64_t(blockIdx.x) * E + e] = sum[e];
    }
    if (threadIdx.x == 0) {
        a.blockCounts[int64_t(blockIdx.x) * (E + 1) + E] = *routed;
    }
}

constexpr int kMostBlocks = 1024, kScanCols = 8, kScanRuns = kThreads / kScanCols, kScanEach = kMostBlocks / kScanRuns;

// Adds up the workgroups' counts and probabilities, eight experts (columns) to a workgroup and 32 runs of rows to an expert, all of a run
// on its way at once, and leaves in blockCounts what lies in front of every workgroup.  Column `experts` holds the tokens that chose.
__global__ void __launch_bounds__(kThreads) ScanKernel(RouteArgs a)
{
    __shared__ int parts[kScanRuns][kScanCols + 1];
    __shared__ float partSums[kScanRuns][kScanCols + 1];
    const int c = int(threadIdx.x) % kScanCols, run = int(threadIdx.x) / kScanCols, e = int(blockIdx.x) * kScanCols + c;
    const int64_t width = a.experts + 1;
    const int per = (a.blocks + kScanRuns - 1) / kScanRuns, from = run * per;
    int n[kScanEach], all = 0;
    float p[kScanEach], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kScanEach; i++) {
        const bool in = i < per && from + i < a.blocks;
        n[i] = in && e <= a.experts ? a.blockCounts[(from + i) * width + e] : 0;
        p[i] = in && e < a.experts ? a.blockSums[int64_t(from + i) * a.experts + e] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kScanEach; i++) {
        all += n[i];
        sum += p[i];
    }
    parts[run][c] = all;
    partSums[run][c] = sum;
    __syncthreads();
    int before = 0;
    all = 0;
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kScanRuns; i++) {
        before += i < run ? parts[i][c] : 0;
        all += parts[i][c];
        sum += partSums[i][c];
    }
    if (e > a.experts) {
        return;
    }
#pragma unroll
    for (int i = 0; i < kScanEach; i++) {
        if (i < per && from + i < a.blocks) {
            a.blockCounts[(from + i) * width + e] = before;
            before += n[i];
        }
    }
    if (run == 0) {
        a.counts[e] = all;
        if (e < a.experts) {
            a.sums[e] = sum;
        }
    }
}

// Every choice's row: its expert's first row, the rows of the workgroups before its own, its place in its own.  kAll: every workgroup adds up
// the table of counts itself, and no launch has done so before.
template <bool kAll>
__global__ void __launch_bounds__(kThreads) RowsKernel(RouteArgs a, int tokensEach)
{
    extern __shared__ uint32_t lds[];
    const int E = a.experts, block = int(blockIdx.x);
    int *count = reinterpret_cast<int *>(lds);                           // [experts + 1]
    float *sum = reinterpret_cast<float *>(count + E + 1);               // [experts]
    int *before = reinterpret_cast<int *>(sum + E);                      // [experts]
    int *part = before + E;                                              // [waves]
    float *partSum = reinterpret_cast<float *>(part + kThreads / 64);    // [waves]
    for (int e = threadIdx.x; e <= E; e += kThreads) {
        int all = 0, front = 0;
        float p = 0.0f;
        if constexpr (kAll) {
#pragma unroll 8
            for (int b = 0; b < a.blocks; b++) {
                const int n = a.blockCounts[int64_t(b) * (E + 1) + e];
                all += n;
                front += b < block ? n : 0;
            }
            if (block == 0 && e < E) {
#pragma unroll 8
                for (int b = 0; b < a.blocks; b++) {
                    p += a.blockSums[int64_t(b) * E + e];
                }
            }
        } else {
            all = a.counts[e];
            front = a.blockCounts[int64_t(block) * (E + 1) + e];
            p = block == 0 && e < E ? a.sums[e] : 0.0f;
        }
        count[e] = all;
        if (e < E) {
            sum[e] = p;
            before[e] = front;
        }
    }
    __syncthreads();
    const int tokens = count[E];
    Finish<kThreads>(a, count, sum, tokens, part, partSum, block == 0);
    const int64_t first = int64_t(block) * tokensEach * a.topK;
    const int64_t last = min(first + int64_t(tokensEach) * a.topK, int64_t(a.tokens) * a.topK);
    for (int64_t i = first + threadIdx.x; i < last; i += kThreads) {
        const int e = a.expertOf[i];
        if (e >= 0) {
            a.rowOf[i] += count[e] + before[e];
        }
    }
}

struct RouteGradArgs {
    const void *logits;
    const uint8_t *mask;
    const int32_t *expertOf;
    const int32_t *counts;
    const float *weightGrad;
    const float *lossGrad;
    void *logitGrad;
    int64_t stride, gradStride;
    int tokens, experts, topK;
    float lossScale;
    bool renormalise;
};

// Keeps the compiler from moving LDS operations of one wave's lanes past each other.
__device__ __forceinline__ void Ordered()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// kLanes lanes to a token (at least as many as it has choices), kEach experts to a lane, in vectors of four that the lanes of a token
// take in turn.  A workgroup goes through tokens, what it knows of the experts stays in registers.  What the weights' gradients add at
// the chosen experts is worked out by one lane for each and put in on the way out through LDS.
template <typename T, int kLanes, int kEach, int kHow>
__global__ void __launch_bounds__(kThreads) RouteGradKernel(RouteGradArgs a)
{
    constexpr int kTokens = kThreads / kLanes;
    __shared__ __align__(16) float rows[kTokens][kLanes * kEach];
    __shared__ int parts[kThreads / 64];
    const int l = int(threadIdx.x) % kLanes, slot = int(threadIdx.x) / kLanes, E = a.experts;
    // the balance loss's gradient of p_te is c E n_e / (A T) * lossGrad
    float load[kEach];
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        load[i] = 0.0f;
    }
    if (a.lossGrad != nullptr) {
        int n = 0;
        for (int e = threadIdx.x; e < E; e += kThreads) {
            n += a.counts[e];
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            n += __shfl_xor(n, d, 64);
        }
        if (threadIdx.x % 64 == 0) {
            parts[threadIdx.x / 64] = n;
        }
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 64; w++) {
            all += parts[w];
        }
        const float by = all > 0 ? a.lossGrad[0] * a.lossScale * float(E) / float(all) / float(a.counts[E]) : 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int e = (i / 4 * kLanes + l) * 4 + i % 4;
            load[i] = e < E ? by * float(a.counts[e]) : 0.0f;
        }
    }
    for (int64_t t = int64_t(blockIdx.x) * kTokens + slot; t < a.tokens; t += int64_t(gridDim.x) * kTokens) {
        T *out = static_cast<T *>(a.logitGrad) + t * a.gradStride;
        const T *in = static_cast<const T *>(a.logits) + t * a.stride;
        const int chosen = l < a.topK ? a.expertOf[t * a.topK + l] : -1;
        const float dw = chosen >= 0 && a.weightGrad != nullptr ? a.weightGrad[t * a.topK + l] : 0.0f;
        const bool none = (a.mask != nullptr && a.mask[t] == 0) || a.expertOf[t * a.topK] < 0;
        float x[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
            float v[4];
            LoadPart<kHow, 4>(in, (i / 4 * kLanes + l) * 4, E, v, -__builtin_inff());
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[i + j] = v[j];
            }
        }
        // the chosen logits, from other lanes, through LDS (a token's lanes are in one wave, whose LDS operations keep their order)
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
            *reinterpret_cast<Float4 *>(&rows[slot][(i / 4 * kLanes + l) * 4]) = Float4{x[i], x[i + 1], x[i + 2], x[i + 3]};
        }
        Ordered();
        const float logit = chosen >= 0 && chosen < E ? rows[slot][chosen] : -__builtin_inff();
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            top = Larger(top, x[i]);
        }
        top = LargestOfNeighbours<kLanes>(top);
        float sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            x[i] = Exp(x[i] - top);
            sum += x[i];
            dot = __builtin_fmaf(x[i], load[i], dot);
        }
        const float w = chosen >= 0 ? Exp(logit - top) : 0.0f;
        sum = AddNeighbours<kLanes>(sum);
        const float by = 1.0f / sum;
        float more;     // what this lane's choice adds
        if (a.renormalise) {
            const float inside = AddNeighbours<kLanes>(w), mean = AddNeighbours<kLanes>(w * dw) / inside;
            more = w / inside * (dw - mean);
        } else {
            dot = __builtin_fmaf(w, dw, dot);
            more = w * by * dw;
        }
        dot = AddNeighbours<kLanes>(dot) * by;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            x[i] = x[i] * by * (load[i] - dot);
        }
        if (__ballot(none) != 0) {
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                x[i] = none ? 0.0f : x[i];
            }
        }
        Ordered();
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
            const Float4 v{x[i], x[i + 1], x[i + 2], x[i + 3]};
            *reinterpret_cast<Float4 *>(&rows[slot][(i / 4 * kLanes + l) * 4]) = v;
        }
        Ordered();
        if (a.weightGrad != nullptr && chosen >= 0 && chosen < E && !none) {
            rows[slot][chosen] += more;
        }
        Ordered();
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
            const int e = (i / 4 * kLanes + l) * 4;
            const Float4 f = *reinterpret_cast<const Float4 *>(&rows[slot][e]);
            const float v[4] = {f[0], f[1], f[2], f[3]};
            StorePart<kHow, 4>(out, e, E, v);
        }
        Ordered();
    }
}

// Tokens of a tile: 64 with four lanes to a token, 16 with sixteen.  Sixteen lanes where a lane would have more than 64 experts,
// and for few tokens, where the time is one lane's.
int TileOf(uint64_t tokens, uint32_t experts) { return experts > 256 || tokens <= 64 * 64 ? 16 : 64; }

// Workgroups: at most 1024, four to a compute unit, each with as many tiles as that takes.
int TilesOf(uint64_t tokens, int tile)
{
    const uint64_t tiles = (tokens + uint64_t(tile) - 1) / uint64_t(tile);
    return tiles == 0 ? 1 : tiles <= 4 ? int(tiles) : int((tiles + kMostBlocks - 1) / kMostBlocks);
}

int BlocksOf(uint64_t tokens, int tile)
{
    const uint64_t each = uint64_t(tile) * uint64_t(TilesOf(tokens, tile));
    return tokens == 0 ? 1 : int((tokens + each - 1) / each);
}

template <typename T, int K, int kLanes, int kChunks>
HcclResult LaunchRoute(const RouteArgs &a, bool wide, hipStream_t stream)
{
    const size_t lds = 4 * ((3 + kThreads / 64) * size_t(a.experts) + 2 * (kThreads / 64) + 1);
    const auto go = [&](auto kernel) { return Launch("HcclAmdExpertRoute", kernel, uint32_t(a.blocks), kThreads, lds, stream, a); };
    return wide && a.experts == 8 * kLanes * kChunks && a.tokens > 0 ? go(RouteKernel<T, K, kLanes, kChunks, kExactly>)
           : wide                                                    ? go(RouteKernel<T, K, kLanes, kChunks, kAligned>)
                                                                     : go(RouteKernel<T, K, kLanes, kChunks, kAnyhow>);
}

template <typename T, int K>
HcclResult LaunchRouteShape(const RouteArgs &a, int tile, bool wide, hipStream_t stream)
{
    if (tile == 64) {
        return a.experts <= 64 ? LaunchRoute<T, K, 4, 2>(a, wide, stream) : LaunchRoute<T, K, 4, 8>(a, wide, stream);
    }
    return a.experts <= 256 ? LaunchRoute<T, K, 16, 2>(a, wide, stream) : LaunchRoute<T, K, 16, 8>(a, wide, stream);
}

template <typename T>
HcclResult LaunchRouteType(const RouteArgs &a, int tile, bool wide, hipStream_t stream)
{
    return a.topK <= 2   ? LaunchRouteShape<T, 2>(a, tile, wide, stream)
           : a.topK <= 4 ? LaunchRouteShape<T, 4>(a, tile, wide, stream)
           : a.topK <= 8 ? LaunchRouteShape<T, 8>(a, tile, wide, stream)
                         : LaunchRouteShape<T, 16>(a, tile, wide, stream);
}

template <typename T, int kHow>
HcclResult LaunchRouteGrad(const RouteGradArgs &a, hipStream_t stream)
{
    const auto go = [&](auto kernel, int lanes) {
        const int64_t blocks = (int64_t(a.tokens) * lanes + kThreads - 1) / kThreads;
        return Launch("HcclAmdExpertRouteGrad", kernel, uint32_t(blocks < 1024 ? blocks : 1024), kThreads, 0, stream, a);
    };
    if (a.experts <= 64) {
        return go(RouteGradKernel<T, 16, 4, kHow>, 16);
    }
    if (a.experts <= 128) {
        return go(RouteGradKernel<T, 16, 8, kHow>, 16);
    }
    if (a.experts <= 256) {
        return go(RouteGradKernel<T, 16, 16, kHow>, 16);
    }
    return go(RouteGradKernel<T, 64, 16, kHow>, 64);
}

}  // namespace
}  // namespace experts
}  // namespace hcclamd

using namespace hcclamd::experts;

extern "C" {

HcclResult HcclAmdExpertRouteWorkspace(uint64_t tokens, uint32_t experts, uint64_t *bytes)
{
    EXPERTS_CHK_PTR(bytes);
    EXPERTS_CHK(experts >= 1 && experts <= HCCL_AMD_MAX_EXPERTS);
    EXPERTS_CHK(tokens <= kMaxTokens);
    const uint64_t blocks = uint64_t(BlocksOf(tokens, TileOf(tokens, experts)));
    *bytes = blocks == 1 ? 0 : 4 * (blocks * (2 * uint64_t(experts) + 1) + experts);
    return HCCL_SUCCESS;
}

HcclResult HcclAmdExpertRoute(const void *logits, HcclDataType logitType, uint64_t tokens, uint32_t experts, uint64_t logitStride,
    uint32_t topK, uint32_t renormalise, const uint8_t *tokenMask, float lossScale, int32_t *expertOf, float *weights, int32_t *rowOf,
    int32_t *counts, int32_t *offsets, float *loss, void *workspace, uint64_t workspaceBytes, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(logitType));
    EXPERTS_CHK(experts >= 1 && experts <= HCCL_AMD_MAX_EXPERTS);
    EXPERTS_CHK(topK >= 1 && topK <= HCCL_AMD_MAX_TOPK && topK <= experts);
    EXPERTS_CHK(tokens <= kMaxTokens);
    EXPERTS_CHK_PTR(counts);
    EXPERTS_CHK_PTR(offsets);
    EXPERTS_CHK_PTR(loss);
    EXPERTS_CHK(Aligned(counts, 4) && Aligned(offsets, 4) && Aligned(loss, 4));
    uint64_t needed = 0;
    HcclAmdExpertRouteWorkspace(tokens, experts, &needed);
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
    const int tile = TileOf(tokens, experts);
    RouteArgs a{};
    a.logits = logits;
    a.mask = tokenMask;
    a.expertOf = expertOf;
    a.weights = weights;
    a.rowOf = rowOf;
    a.counts = counts;
    a.offsets = offsets;
    a.loss = loss;
    a.stride = int64_t(logitStride == 0 ? experts : logitStride);
    a.tokens = int(tokens);
    a.experts = int(experts);
    a.topK = int(topK);
    a.tiles = TilesOf(tokens, tile);
    a.blocks = BlocksOf(tokens, tile);       // no token: the one workgroup writes the zeros
    a.blockCounts = static_cast<int32_t *>(workspace);
    a.blockSums = reinterpret_cast<float *>(a.blockCounts + int64_t(a.blocks) * (a.experts + 1));
    a.lossScale = lossScale;
    a.renormalise = renormalise != 0;
    const hipStream_t on = static_cast<hipStream_t>(stream);
    a.sums = a.blockSums + int64_t(a.blocks) * a.experts;
    const bool wide = experts % 8 == 0 && Aligned(logits, 16) && uint64_t(a.stride) * SizeOf(logitType) % 16 == 0;
    HcclResult r = logitType == HCCL_DATA_TYPE_FP32   ? LaunchRouteType<float>(a, tile, wide, on)
                   : logitType == HCCL_DATA_TYPE_FP16 ? LaunchRouteType<_Float16>(a, tile, wide, on)
                                                      : LaunchRouteType<__bf16>(a, tile, wide, on);
    if (r != HCCL_SUCCESS || a.blocks == 1) {
        return r;
    }
    // Up to 32 workgroups (512 tokens) each adds up the others' counts: a call of 300 tokens of 64 experts takes 12 us instead of 15, of
    // 256 experts 13 instead of 15; with more of them that reading takes as long as a launch of its own.
    const bool few = a.blocks <= 32;
    if (!few) {
        r = Launch("HcclAmdExpertRoute", ScanKernel, experts / kScanCols + 1, kThreads, 0, on, a);
        if (r != HCCL_SUCCESS) {
            return r;
        }
    }
    return Launch("HcclAmdExpertRoute", few ? RowsKernel<true> : RowsKernel<false>, uint32_t(a.blocks), kThreads,
        4 * (3 * size_t(experts) + 1 + 2 * (kThreads / 64)), on, a, tile * a.tiles);
}

HcclResult HcclAmdExpertRouteGrad(const void *logits, HcclDataType logitType, uint64_t tokens, uint32_t experts, uint64_t logitStride,
    uint32_t topK, uint32_t renormalise, const uint8_t *tokenMask, float lossScale, const int32_t *expertOf, const int32_t *counts,
    const float *weightGrad, const float *lossGrad, void *logitGrad, uint64_t logitGradStride, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(logitType));
    EXPERTS_CHK(experts >= 1 && experts <= HCCL_AMD_MAX_EXPERTS);
    EXPERTS_CHK(topK >= 1 && topK <= HCCL_AMD_MAX_TOPK && topK <= experts);
    EXPERTS_CHK(tokens <= kMaxTokens);
    if (tokens == 0) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(logits);
    EXPERTS_CHK_PTR(expertOf);
    EXPERTS_CHK_PTR(counts);
    EXPERTS_CHK_PTR(logitGrad);
    EXPERTS_CHK(Stride(logitStride, experts));
    EXPERTS_CHK(Stride(logitGradStride, experts));
    EXPERTS_CHK(AlignedTo(logitType, logits) && AlignedTo(logitType, logitGrad) && Aligned(expertOf, 4) && Aligned(counts, 4));
    EXPERTS_CHK(Aligned(weightGrad, 4) && Aligned(lossGrad, 4));
    RouteGradArgs a{};
    a.logits = logits;
    a.mask = tokenMask;
    a.expertOf = expertOf;
    a.counts = counts;
    a.weightGrad = weightGrad;
    a.lossGrad = lossGrad;
    a.logitGrad = logitGrad;
    a.stride = int64_t(logitStride == 0 ? experts : logitStride);
    a.gradStride = int64_t(logitGradStride == 0 ? experts : logitGradStride);
    a.tokens = int(tokens);
    a.experts = int(experts);
    a.topK = int(topK);
    a.lossScale = lossScale;
    a.renormalise = renormalise != 0;
    const uint64_t four = 4 * SizeOf(logitType);
    const bool wide = experts % 4 == 0 && a.stride % 4 == 0 && a.gradStride % 4 == 0 && Aligned(logits, four) && Aligned(logitGrad, four);
    const hipStream_t on = static_cast<hipStream_t>(stream);
    const bool exactly = wide && (experts == 64 || experts == 128 || experts == 256 || experts == 1024);
    const auto go = [&](auto of) {
        typedef decltype(of) T;
        return exactly ? LaunchRouteGrad<T, kExactly>(a, on) : wide ? LaunchRouteGrad<T, kAligned>(a, on) : LaunchRouteGrad<T, kAnyhow>(a, on);
    };
    return logitType == HCCL_DATA_TYPE_FP32 ? go(float{}) : logitType == HCCL_DATA_TYPE_FP16 ? go(_Float16{}) : go(__bf16{});
}

}  // extern "C"
