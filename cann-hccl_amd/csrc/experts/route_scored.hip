// Router by scores (HcclAmdExpertRouteScored): softmax or sigmoid, a bias that only chooses, groups of experts, weights that are renormalised or not;
// its gradient, and the bias's step (HcclAmdExpertBias).
//
// With s the scores, w = c s or c s / (sum of the chosen s), and dw the gradient of the weights:
//   sigmoid                 dx_j = w_j (1 - s_j) dw_j                 renormalised: dx_j = w_j (1 - s_j) (dw_j - sum_i (w_i / c) dw_i)
//   softmax, renormalised   dx_j = w_j (dw_j - sum_i (w_i / c) dw_i)  over the chosen ones; the others' gradients are zero
//   softmax                 dx_e = s_e (c dw_e - sum_i c s_i dw_i)    over all experts, dw_e = 0 where e was not chosen
//
// 16 lanes to a token (64 beyond 256 experts), its experts' scores in registers.  Scores next to each other decide which expert a token goes to, so
// that the choice is made in 64 bits.
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

__device__ __forceinline__ double FromOther(double x, int lanes)
{
    return __shfl_xor(x, lanes, 64);
}

// Expert number of element i of lane l: eight neighbours to a lane, then the next lane's.
template <int kLanes>
__device__ __forceinline__ int ExpertOf(int i, int l) { return (i / 8 * kLanes + l) * 8 + i % 8; }

// The choice in 64 bits.  All lanes of a token know its experts afterwards, best first, -1 where there is none.  `of`: a place per group, the token's.
template <int kLanes, int kEach, int K>
__device__ __forceinline__ void Choose(const ScoredArgs &a, const float (&x)[kEach], bool in, int l, double *of, int (&chosen)[K])
{
    double key[kEach];
    if (a.softmax) {
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            top = Larger(top, x[i]);
        }
        top = LargestOfNeighbours<kLanes>(top);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            key[i] = x[i] == top ? 1.0 : x[i] < top ? exp(double(x[i]) - double(top)) : 0.0;
            sum += key[i];
        }
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) {
            sum += FromOther(sum, d);
        }
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
        const int e = ExpertOf<kLanes>(i, l);
        if (a.bias != nullptr && e < a.experts) {
            key[i] += double(a.bias[e]);
        }
        key[i] = in && x[i] > -__builtin_inff() && key[i] > kNever ? key[i] : kNever;
    }
    if (a.groups > 1) {
        for (int g = 0; g < a.groups; g++) {
            double first = kNever, next = kNever;
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                const bool mine = int(uint32_t(ExpertOf<kLanes>(i, l)) * a.perSize >> 20) == g;
                const double k = mine ? key[i] : kNever;
                next = k > first ? first : k > next ? k : next;
                first = k > first ? k : first;
            }
#pragma unroll
            for (int d = 1; d < kLanes; d <<= 1) {
                const double f = FromOther(first, d), n = FromOther(next, d);
                const double low = first < f ? first : f, rest = next > n ? next : n;
                next = low > rest ? low : rest;
                first = first > f ? first : f;
            }
            if (l == 0) {
                of[g] = a.second && next > kNever ? first + next : first;
            }
        }
        Ordered();
        uint32_t keep[2] = {0, 0};
        for (int g = l; g < a.groups; g += kLanes) {
            const double mine = of[g];
            int before = 0;
            for (int o = 0; o < a.groups; o++) {
                const double other = of[o];
                before += other > mine || (other == mine && o < g) ? 1 : 0;
            }
            if (before < a.kept) {
                keep[g / 32] |= 1u << g % 32;
            }
        }
        Ordered();
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) {
            keep[0] |= uint32_t(__shfl_xor(int(keep[0]), d, 64));
            keep[1] |= uint32_t(__shfl_xor(int(keep[1]), d, 64));
        }
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const uint32_t g = uint32_t(ExpertOf<kLanes>(i, l)) * a.perSize >> 20;
            const bool kept = g < 64 && (keep[g / 32 % 2] >> g % 32 & 1) != 0;
            key[i] = kept ? key[i] : kNever;
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
                e = take ? ExpertOf<kLanes>(i, l) : e;
            }
#pragma unroll
            for (int d = 1; d < kLanes; d <<= 1) {
                const double other = FromOther(best, d);
                const int oe = __shfl_xor(e, d, 64);
                const bool take = other > best || (other == best && oe < e);
                best = take ? other : best;
                e = take ? oe : e;
            }
            chosen[j] = best > kNever ? e : -1;
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                key[i] = ExpertOf<kLanes>(i, l) == e ? kNever : key[i];
            }
        }
    }
}

// log of the sigmoid
__device__ __forceinline__ float LogSigmoid(float x) { return fminf(x, 0.0f) - log1pf(Exp(-__builtin_fabsf(x))); }

__device__ __forceinline__ float Sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + Exp(-x)); }

template <typename T, int K, int kLanes, int kEach, int kHow>
__global__ void __launch_bounds__(kThreads) ScoredKernel(ScoredArgs a)
{
    constexpr int kWaveTokens = 64 / kLanes, kTile = kWaveTokens * kThreads / 64;
    extern __shared__ uint32_t lds[];
    const int E = a.experts;
    uint32_t *chose = lds;                                                // [experts]: one bit per token of the tile
    int *count = reinterpret_cast<int *>(chose + E);                      // [experts]: rows of the tiles so far
    int *part = count + E;                                                // [waves]
    int *routed = part + kThreads / 64;                                   // [1]
    __shared__ double groupScores[kTile][HCCL_AMD_MAX_EXPERT_GROUPS];

    const int lane = int(threadIdx.x) % 64, wave = int(threadIdx.x) / 64, l = lane % kLanes, r = wave * kWaveTokens + lane / kLanes;
    for (int e = threadIdx.x; e < E; e += kThreads) {
        chose[e] = 0;
        count[e] = 0;
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
        Choose<kLanes, kEach, K>(a, x, in, l, groupScores[r], chosen);
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
            const unsigned long long rows = __ballot(bad), lanes = kLanes == 64 ? ~0ull : 0xffffull << (lane & 48);
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
    const size_t lds = 4 * (2 * size_t(a.experts) + kThreads / 64 + 1);
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
    return a.topK <= 4 ? LaunchScoredShape<T, 4>(a, wide, stream) : a.topK <= 8 ? LaunchScoredShape<T, 8>(a, wide, stream) : LaunchScoredShape<T, 16>(a, wide, stream);
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
    a.second = groupTop == 2;
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
