// What the routers share behind the choice: from choices and counts of workgroups to counts, offsets and rows in expert order.
//
// A router's workgroup goes through tiles of tokens and leaves in rowOf a choice's place among the workgroup's own rows of its expert, and in
// blockCounts how many it has of each.  One launch adds up what lies in front of every workgroup's, another adds that to the rows; up to 32
// workgroups the second does both.
#pragma once
#include "sums.h"

namespace hcclamd {
namespace experts {
namespace {

constexpr int kThreads = 256;
constexpr uint64_t kMaxTokens = uint64_t(1) << 25;
constexpr int kMostBlocks = 1024;

struct RowsArgs {
    int32_t *expertOf;
    int32_t *rowOf;
    int32_t *counts;
    int32_t *offsets;
    float *loss;
    int32_t *blockCounts;  // [blocks][experts + 1]: rows per expert; last column: tokens that chose
    float *blockSums;      // [blocks][experts]: sum of probabilities (of a router with a loss)
    float *sums;           // [experts]
    int tokens, experts, topK;
    int blocks, tiles;     // workgroups; tiles of each
    float lossScale;
};

// Workgroups: at most 1024, four to a compute unit, each with as many tiles as that takes.
inline int TilesOf(uint64_t tokens, int tile)
{
    const uint64_t tiles = (tokens + uint64_t(tile) - 1) / uint64_t(tile);
    return tiles == 0 ? 1 : tiles <= 4 ? int(tiles) : int((tiles + kMostBlocks - 1) / kMostBlocks);
}

inline int BlocksOf(uint64_t tokens, int tile)
{
    const uint64_t each = uint64_t(tile) * uint64_t(TilesOf(tokens, tile));
    return tokens == 0 ? 1 : int((tokens + each - 1) / each);
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

// counts[experts + 1], offsets and (kLoss) the loss from per-expert counts and sums in LDS, if `write`; afterwards `count` holds the offsets.
template <int kThreads, bool kLoss>
__device__ __forceinline__ void Finish(const RowsArgs &a, int *count, const float *sum, int tokens, int *part, float *partSum, bool write)
{
    float load = 0.0f;
    for (int e = threadIdx.x; e < a.experts && write; e += kThreads) {
        if constexpr (kLoss) {
            load += float(count[e]) * sum[e];
        }
        a.counts[e] = count[e];
    }
    if constexpr (kLoss) {
        load = AddNeighbours<64>(load);
        if (threadIdx.x % 64 == 0) {
            partSum[threadIdx.x / 64] = load;
        }
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
        a.counts[a.experts] = tokens;
        a.offsets[a.experts] = rows;
        if constexpr (kLoss) {
            float all = 0.0f;
            for (int w = 0; w < kThreads / 64; w++) {
                all += partSum[w];
            }
            a.loss[0] = rows == 0 ? 0.0f : a.lossScale * float(a.experts) * (all / float(rows) / float(tokens));
        }
    }
}

constexpr int kScanCols = 8, kScanRuns = kThreads / kScanCols, kScanEach = kMostBlocks / kScanRuns;

// Adds up the workgroups' counts and probabilities, eight experts (columns) to a workgroup and 32 runs of rows to an expert, all of a run
// on its way at once, and leaves in blockCounts what lies in front of every workgroup.  Column `experts` holds the tokens that chose.
template <bool kLoss>
__global__ void __launch_bounds__(kThreads) ScanKernel(RowsArgs a)
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
        p[i] = kLoss && in && e < a.experts ? a.blockSums[int64_t(from + i) * a.experts + e] : 0.0f;
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
        if (kLoss && e < a.experts) {
            a.sums[e] = sum;
        }
    }
}

// Every choice's row: its expert's first row, the rows of the workgroups before its own, its place in its own.  kAll: every workgroup adds up
// the table of counts itself, and no launch has done so before.
template <bool kAll, bool kLoss>
__global__ void __launch_bounds__(kThreads) RowsKernel(RowsArgs a, int tokensEach)
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
            if (kLoss && block == 0 && e < E) {
#pragma unroll 8
                for (int b = 0; b < a.blocks; b++) {
                    p += a.blockSums[int64_t(b) * E + e];
                }
            }
        } else {
            all = a.counts[e];
            front = a.blockCounts[int64_t(block) * (E + 1) + e];
            p = kLoss && block == 0 && e < E ? a.sums[e] : 0.0f;
        }
        count[e] = all;
        if (e < E) {
            sum[e] = p;
            before[e] = front;
        }
    }
    __syncthreads();
    const int tokens = count[E];
    Finish<kThreads, kLoss>(a, count, sum, tokens, part, partSum, block == 0);
    const int64_t first = int64_t(block) * tokensEach * a.topK;
    const int64_t last = min(first + int64_t(tokensEach) * a.topK, int64_t(a.tokens) * a.topK);
    for (int64_t i = first + threadIdx.x; i < last; i += kThreads) {
        const int e = a.expertOf[i];
        if (e >= 0) {
            a.rowOf[i] += count[e] + before[e];
        }
    }
}

inline size_t RowsLds(int experts) { return 4 * (3 * size_t(experts) + 1 + 2 * (kThreads / 64)); }

}  // namespace
}  // namespace experts
}  // namespace hcclamd
