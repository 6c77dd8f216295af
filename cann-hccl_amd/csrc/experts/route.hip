// Router of an expert-parallel layer: the topK largest logits of every token, their weights, rows in expert order, per-expert
// counts and the balance loss; and the gradient of all that.
//
// With p = softmax(x) over a token's experts, n_e the tokens that chose e, A their sum, T the tokens that chose any:
//   loss = c E sum_e (n_e / A) (sum_t p_te / T)       d loss / d p_te = c E n_e / (A T)
//   w_j = p_j, or p_j / sum of the chosen p           dx = p (g - sum p g), and for the quotient w_j (dw_j - sum_i w_i dw_i)
//
// The logits are read once.  A workgroup holds a tile of tokens in LDS; several lanes share a token.  Every lane keeps the
// topK largest of its experts in registers as a sorted list -- inserting costs five instructions per entry and no exchange
// between lanes, whereas finding one maximum after the other over a whole wave costs six exchanges for each -- and the lists of a
// token's lanes are merged at the end.  Which tokens of the tile chose an expert is a mask of one bit per token: set with
// LDS atomics whose order cannot matter, its bits counted in front of a token give the token's place, and counts and rows are the
// same in every run.  Tiles leave counts and probability sums in the workspace, a second launch sums them expert by expert in
// tile order, a third adds up the rows' places.  Up to one tile (single tokens of a decoding step, small batches) one launch does it all.
#include "common.h"

namespace hcclamd {
namespace experts {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kNone = 0xffffffffu;
constexpr uint64_t kMaxTokens = uint64_t(1) << 25;   // 64 lanes each stay below the 2^32 threads of a grid

struct RouteArgs {
    const void *logits;
    const uint8_t *mask;
    int32_t *expertOf;
    float *weights;
    int32_t *rowOf;
    int32_t *counts;
    int32_t *offsets;
    float *loss;
    int32_t *tileCounts;   // [tiles][experts + 1]: rows per expert, then first row per expert within the expert's; last column: tokens that chose
    float *tileSums;       // [tiles][experts]: sum of probabilities
    float *sums;           // [experts]
    int64_t stride;
    int tokens, experts, topK, tiles;
    int rowWords;          // LDS words from one token to the next
    float lossScale;
    bool renormalise;
};

// (value, expert) pairs ordered by value, then by lower expert.  Lists are sorted, largest first; an empty place is
// (-inf, kNone), which every logit that may be chosen precedes.
struct Entry {
    float v;
    uint32_t e;
};

__device__ __forceinline__ bool Before(const Entry &a, const Entry &b) { return a.v > b.v || (a.v == b.v && a.e < b.e); }

// No instruction.  Without it the compiler reasons about chains of dozens of selects as one, for hours.
__device__ __forceinline__ void Settle(Entry &x) { asm("" : "+v"(x.v), "+v"(x.e)); }

// The larger half of two sorted lists: element by element against the other one backwards, which leaves a sequence that
// rises and falls once, then sorted by halving.
template <int K>
__device__ __forceinline__ void Merge(Entry (&a)[K], int lanes)
{
    Entry b[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        b[i].v = __shfl_xor(a[i].v, lanes, 64);
        b[i].e = __shfl_xor(a[i].e, lanes, 64);
    }
#pragma unroll
    for (int i = 0; i < K; i++) {
        const bool take = Before(b[K - 1 - i], a[i]);
        a[i].v = take ? b[K - 1 - i].v : a[i].v;
        a[i].e = take ? b[K - 1 - i].e : a[i].e;
        Settle(a[i]);
    }
#pragma unroll
    for (int d = K / 2; d > 0; d >>= 1) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            if ((i & d) == 0) {
                const bool swap = Before(a[i + d], a[i]);
                const Entry lo = a[i], hi = a[i + d];
                a[i].v = swap ? hi.v : lo.v;
                a[i].e = swap ? hi.e : lo.e;
                a[i + d].v = swap ? lo.v : hi.v;
                a[i + d].e = swap ? lo.e : hi.e;
                Settle(a[i]);
                Settle(a[i + d]);
            }
        }
    }
}

// Exclusive prefix sums of n <= 1024 values in LDS by one workgroup, and the total; `part`: kThreads words.
__device__ __forceinline__ int Scan(int *values, int n, int *part)
{
    const int per = (n + kThreads - 1) / kThreads, from = min(n, int(threadIdx.x) * per), to = min(n, from + per);
    int mine = 0;
    for (int i = from; i < to; i++) {
        mine += values[i];
    }
    part[threadIdx.x] = mine;
    __syncthreads();
    for (int d = 1; d < kThreads; d <<= 1) {
        const int other = int(threadIdx.x) >= d ? part[threadIdx.x - d] : 0;
        __syncthreads();
        part[threadIdx.x] += other;
        __syncthreads();
    }
    int at = part[threadIdx.x] - mine;
    const int total = part[kThreads - 1];
    for (int i = from; i < to; i++) {
        const int v = values[i];
        values[i] = at;
        at += v;
    }
    __syncthreads();
    return total;
}

// counts[experts + 1], offsets and the loss from per-expert counts and sums in LDS; afterwards `count` holds the offsets.
__device__ __forceinline__ void Finish(const RouteArgs &a, int *count, const float *sum, int tokens, int *part, float *partSum, bool write)
{
    float load = 0.0f;
    for (int e = threadIdx.x; e < a.experts; e += kThreads) {
        load += float(count[e]) * sum[e];
        if (write) {
            a.counts[e] = count[e];
        }
    }
    __syncthreads();
    const int rows = Scan(count, a.experts, part);
    if (!write) {
        return;
    }
    for (int e = threadIdx.x; e < a.experts; e += kThreads) {
        a.offsets[e] = count[e];
    }
    partSum[threadIdx.x] = load;
    for (int d = kThreads / 2; d > 0; d >>= 1) {
        __syncthreads();
        if (int(threadIdx.x) < d) {
            partSum[threadIdx.x] += partSum[threadIdx.x + d];
        }
    }
    if (threadIdx.x == 0) {
        a.counts[a.experts] = tokens;
        a.offsets[a.experts] = rows;
        a.loss[0] = rows == 0 ? 0.0f : a.lossScale * float(a.experts) * (partSum[0] / float(rows) / float(tokens));
    }
    __syncthreads();
}

// kLanes lanes to a token, kThreads / kLanes tokens to a tile; lists of K.
template <typename T, int K, int kLanes>
__global__ void __launch_bounds__(kThreads) RouteKernel(RouteArgs a)
{
    constexpr int kTile = kThreads / kLanes;
    extern __shared__ float lds[];
    float *tile = lds;                                                               // [kTile][rowWords]
    float *share = tile + kTile * a.rowWords;                                        // [kTile]: 1 / sum of a token's exponentials, 0 without
    uint32_t *chose = reinterpret_cast<uint32_t *>(share + kTile);                   // [experts][2]: one bit per token
    int *count = reinterpret_cast<int *>(chose + 2 * a.experts);                     // [experts]
    float *sum = reinterpret_cast<float *>(count + a.experts);                       // [experts]
    int *part = reinterpret_cast<int *>(sum + a.experts);                            // [kThreads]
    float *partSum = reinterpret_cast<float *>(part + kThreads);                     // [kThreads]
    uint32_t *routed = reinterpret_cast<uint32_t *>(partSum + kThreads);             // [1]

    const int first = int(blockIdx.x) * kTile, here = min(kTile, a.tokens - first);
    const int E = a.experts;
    for (int e = threadIdx.x; e < 2 * E; e += kThreads) {
        chose[e] = 0;
    }
    if (threadIdx.x == 0) {
        *routed = 0;
    }
    const T *logits = static_cast<const T *>(a.logits) + int64_t(first) * a.stride;
    for (int r = threadIdx.x / kLanes, l = threadIdx.x % kLanes; r < here; r += kTile) {
        const bool in = a.mask == nullptr || a.mask[first + r] != 0;
        for (int e = l; e < E; e += kLanes) {
            tile[r * a.rowWords + e] = in ? float(logits[int64_t(r) * a.stride + e]) : -__builtin_inff();
        }
    }
    __syncthreads();

    const int r = threadIdx.x / kLanes, l = threadIdx.x % kLanes;
    float *row = tile + r * a.rowWords;
    Entry best[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        best[i] = Entry{-__builtin_inff(), kNone};
    }
    if (r < here) {
        for (int e = l; e < E; e += kLanes) {
            const float x = row[e];
            // x goes behind the last entry that is not less, those after it move on.  Experts come in ascending order: of
            // equal values the one that is there stays in front (and NaN, greater than nothing, is never put in)
            bool ahead = x > best[K - 1].v;
#pragma unroll
            for (int i = K - 1; i > 0; i--) {
                const bool further = x > best[i - 1].v;
                best[i].v = further ? best[i - 1].v : ahead ? x : best[i].v;
                best[i].e = further ? best[i - 1].e : ahead ? uint32_t(e) : best[i].e;
                ahead = further;
            }
            best[0].v = ahead ? x : best[0].v;
            best[0].e = ahead ? uint32_t(e) : best[0].e;
        }
    }
#pragma unroll 1
    for (int d = 1; d < kLanes; d <<= 1) {
        Merge<K>(best, d);
    }
    const float top = best[0].v;
    const bool any = best[0].e != kNone;
    float total = 0.0f;
    if (r < here && any) {
        for (int e = l; e < E; e += kLanes) {
            const float x = expf(row[e] - top);
            row[e] = x;
            total += x;
        }
    }
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) {
        total += __shfl_xor(total, d, 64);
    }
    // (a row that chose nothing adds nothing to the sums, whatever it holds)
    const float times = any ? 1.0f / total : 0.0f;
    if (r < here && l == 0) {
        share[r] = times;
        if (any) {
            atomicAdd(routed, 1u);   // a whole number: the order does not matter
        }
    }
    float inside = 0.0f, weight[K];
#pragma unroll
    for (int i = 0; i < K; i++) {
        weight[i] = i < a.topK && best[i].e != kNone ? expf(best[i].v - top) : 0.0f;
        inside += weight[i];
    }
    const bool bad = any && !(total < __builtin_inff());   // a NaN or +inf in the row: its weights are NaN, chosen or not by these
    const float by = bad ? __builtin_nanf("") : a.renormalise ? (any ? 1.0f / inside : 0.0f) : times;
    if (r < here) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            if (i < a.topK && i % kLanes == l) {
                const int64_t at = int64_t(first + r) * a.topK + i;
                const bool is = best[i].e != kNone;
                a.expertOf[at] = is ? int32_t(best[i].e) : -1;
                a.weights[at] = is ? weight[i] * by : 0.0f;
                if (is) {
                    atomicOr(&chose[2 * best[i].e + (r >> 5)], 1u << (r & 31));
                }
            }
        }
    }
    __syncthreads();
    // sums of probabilities: the experts over the threads, the tile's tokens cut among the threads of one expert
    const int perExpert = E >= kThreads ? 1 : kThreads / E;
    for (int e0 = 0; e0 < E; e0 += kThreads) {
        const int e = e0 + int(threadIdx.x) % (E >= kThreads ? kThreads : E), piece = E >= kThreads ? 0 : int(threadIdx.x) / E;
        const int step = (here + perExpert - 1) / perExpert;
        float s = 0.0f;
        if (e < E && piece < perExpert) {
            for (int t = piece * step; t < min(here, piece * step + step); t++) {
                if (share[t] != 0.0f) {
                    s += tile[t * a.rowWords + e] * share[t];
                }
            }
        }
        partSum[threadIdx.x] = s;
        __syncthreads();
        if (e < E && piece == 0) {
            for (int i = 1; i < perExpert; i++) {
                s += partSum[int(threadIdx.x) + i * E];
            }
            sum[e] = s;
            count[e] = __popc(chose[2 * e]) + __popc(chose[2 * e + 1]);
        }
        __syncthreads();
    }
    const bool alone = a.tiles == 1;
    if (!alone) {
        for (int e = threadIdx.x; e < E; e += kThreads) {
            a.tileCounts[int64_t(blockIdx.x) * (E + 1) + e] = count[e];
            a.tileSums[int64_t(blockIdx.x) * E + e] = sum[e];
        }
        if (threadIdx.x == 0) {
            a.tileCounts[int64_t(blockIdx.x) * (E + 1) + E] = int(*routed);
        }
    } else {
        Finish(a, count, sum, int(*routed), part, partSum, true);
    }
    // a token's place among the tile's rows of its expert; with a single tile that is all
    if (r < here) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            if (i < a.topK && i % kLanes == l) {
                int32_t place = -1;
                if (best[i].e != kNone) {
                    const uint32_t low = chose[2 * best[i].e], high = chose[2 * best[i].e + 1];
                    place = r < 32 ? __popc(low & ((1u << r) - 1)) : __popc(low) + __popc(high & ((1u << (r - 32)) - 1));
                    place += alone ? count[best[i].e] : 0;
                }
                a.rowOf[int64_t(first + r) * a.topK + i] = place;
            }
        }
    }
}

// Sums the tiles' counts and probabilities, 16 experts (columns) to a workgroup and 16 runs of tiles to an expert, and leaves in
// tileCounts what lies in front of every tile.  Column `experts` holds the tokens that chose.
__global__ void __launch_bounds__(kThreads) TileScanKernel(RouteArgs a)
{
    __shared__ int parts[16][17];
    __shared__ float partSums[16][17];
    const int c = threadIdx.x % 16, run = threadIdx.x / 16, e = int(blockIdx.x) * 16 + c;
    const int per = (a.tiles + 15) / 16, from = min(a.tiles, run * per), to = min(a.tiles, from + per);
    const int64_t width = a.experts + 1;
    int n = 0;
    float s = 0.0f;
    if (e <= a.experts) {
        for (int t = from; t < to; t++) {
            n += a.tileCounts[t * width + e];
            s += e < a.experts ? a.tileSums[int64_t(t) * a.experts + e] : 0.0f;
        }
    }
    parts[run][c] = n;
    partSums[run][c] = s;
    __syncthreads();
    int before = 0, all = 0;
    float sum = 0.0f;
    for (int i = 0; i < 16; i++) {
        before += i < run ? parts[i][c] : 0;
        all += parts[i][c];
        sum += partSums[i][c];
    }
    if (e > a.experts) {
        return;
    }
    for (int t = from; t < to; t++) {
        const int here = a.tileCounts[t * width + e];
        a.tileCounts[t * width + e] = before;
        before += here;
    }
    if (run == 0) {
        a.counts[e] = all;
        if (e < a.experts) {
            a.sums[e] = sum;
        }
    }
}

// Every choice's row: its expert's first row, the rows of the tiles before its own, its place in its tile.
__global__ void __launch_bounds__(kThreads) RowsKernel(RouteArgs a, int tile)
{
    extern __shared__ float lds[];
    int *count = reinterpret_cast<int *>(lds);                       // [experts]
    float *sum = reinterpret_cast<float *>(count + a.experts);       // [experts]
    int *part = reinterpret_cast<int *>(sum + a.experts);            // [kThreads]
    float *partSum = reinterpret_cast<float *>(part + kThreads);     // [kThreads]
    for (int e = threadIdx.x; e < a.experts; e += kThreads) {
        count[e] = a.counts[e];
        sum[e] = a.sums[e];
    }
    const int tokens = a.counts[a.experts];
    __syncthreads();
    Finish(a, count, sum, tokens, part, partSum, blockIdx.x == 0);
    const int64_t all = int64_t(a.tokens) * a.topK;
    for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < all; i += int64_t(gridDim.x) * kThreads) {
        const int e = a.expertOf[i];
        if (e >= 0) {
            const int64_t t = i / a.topK / tile;
            a.rowOf[i] += count[e] + a.tileCounts[t * (a.experts + 1) + e];
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

// kLanes lanes to a token, kEach experts to a lane, in vectors of four that the lanes of a token take in turn.
template <typename T, int kLanes, int kEach, bool kWide>
__global__ void __launch_bounds__(kThreads) RouteGradKernel(RouteGradArgs a)
{
    const int l = threadIdx.x % kLanes;
    const int64_t t = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
    const int E = a.experts;
    __shared__ int total;
    if (a.lossGrad != nullptr) {   // rows in all
        if (threadIdx.x == 0) {
            total = 0;
        }
        __syncthreads();
        int n = 0;
        for (int e = threadIdx.x; e < E; e += kThreads) {
            n += a.counts[e];
        }
        atomicAdd(&total, n);      // whole numbers: the order does not matter
        __syncthreads();
    }
    if (t >= a.tokens) {
        return;
    }
    const int32_t *chosen = a.expertOf + t * a.topK;
    T *out = static_cast<T *>(a.logitGrad) + t * a.gradStride;
    const T *in = static_cast<const T *>(a.logits) + t * a.stride;
    float x[kEach];
    if ((a.mask != nullptr && a.mask[t] == 0) || chosen[0] < 0) {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            x[i] = 0.0f;
        }
    } else {
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
            const int e = (i / 4 * kLanes + l) * 4;
            float v[4];
            if (kWide) {
                if (e < E) {
                    Load<true, 4>(in + e, v);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[i + j] = e < E ? v[j] : -__builtin_inff();
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[i + j] = e + j < E ? float(in[e + j]) : -__builtin_inff();
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            top = x[i] > top ? x[i] : top;
        }
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) {
            const float other = __shfl_xor(top, d, 64);
            top = other > top ? other : top;
        }
        // the balance loss's gradient of p_te is c E n_e / (A T) * lossGrad
        float load = 0.0f;
        if (a.lossGrad != nullptr && total > 0) {
            load = a.lossGrad[0] * a.lossScale * float(E) / float(total) / float(a.counts[E]);
        }
        float sum = 0.0f, dot = 0.0f, g[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const int e = (i / 4 * kLanes + l) * 4 + i % 4;
            x[i] = expf(x[i] - top);
            sum += x[i];
            g[i] = a.lossGrad != nullptr && e < E ? load * float(a.counts[e]) : 0.0f;
        }
        // what the weights' gradients add: to g at the chosen, or with the quotient at the end
        float inside = 0.0f, mean = 0.0f;
        if (a.weightGrad != nullptr) {
            for (int j = 0; j < a.topK; j++) {
                const int c = chosen[j];
                if (c < 0) {
                    break;
                }
                const float dw = a.weightGrad[t * a.topK + j];
                if (a.renormalise) {
                    const float w = expf(float(in[c]) - top);
                    inside += w;
                    mean += w * dw;
                } else {
#pragma unroll
                    for (int i = 0; i < kEach; i++) {
                        g[i] += (i / 4 * kLanes + l) * 4 + i % 4 == c ? dw : 0.0f;
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            dot += x[i] * g[i];
        }
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) {
            sum += __shfl_xor(sum, d, 64);
            dot += __shfl_xor(dot, d, 64);
        }
        const float by = 1.0f / sum;
        dot *= by;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            x[i] = x[i] * by * (g[i] - dot);
        }
        if (a.weightGrad != nullptr && a.renormalise) {
            mean /= inside;
            for (int j = 0; j < a.topK; j++) {
                const int c = chosen[j];
                if (c < 0) {
                    break;
                }
                const float more = expf(float(in[c]) - top) / inside * (a.weightGrad[t * a.topK + j] - mean);
#pragma unroll
                for (int i = 0; i < kEach; i++) {
                    x[i] += (i / 4 * kLanes + l) * 4 + i % 4 == c ? more : 0.0f;
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kEach; i += 4) {
        const int e = (i / 4 * kLanes + l) * 4;
        const float v[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
        if (kWide) {
            if (e < E) {
                Store<true, 4>(out + e, v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (e + j < E) {
                    out[e + j] = T(v[j]);
                }
            }
        }
    }
}

// Tokens to a tile.  Up to 64 tokens one tile of 64 makes it a single launch; beyond, as many as leave a tile for each of the
// 256 compute units, and no more LDS than two workgroups can share.
int TileOf(uint64_t tokens, uint32_t experts)
{
    if (experts > 256) {
        return 16;
    }
    return tokens <= 64 || tokens >= 64 * 256 ? 64 : 16;
}

// LDS words from one token to the next: as many beyond a multiple of the 64 banks as lanes share a token, so that the
// lanes of a wave find their words in different banks.
int RowWords(uint32_t experts, int lanes) { return int((experts + 63 - uint32_t(lanes)) / 64 * 64) + lanes; }

template <typename T, int K, int kLanes>
void LaunchRoute(const RouteArgs &a, hipStream_t stream)
{
    constexpr int kTile = kThreads / kLanes;
    const size_t lds = 4 * (size_t(kTile) * a.rowWords + kTile + 4 * size_t(a.experts) + 2 * kThreads + 1);
    hipLaunchKernelGGL((RouteKernel<T, K, kLanes>), dim3(a.tiles), dim3(kThreads), lds, stream, a);
}

template <typename T, int K>
void LaunchRouteTile(const RouteArgs &a, int tile, hipStream_t stream)
{
    tile == 64 ? LaunchRoute<T, K, 4>(a, stream) : LaunchRoute<T, K, 16>(a, stream);
}

template <typename T>
void LaunchRouteType(const RouteArgs &a, int tile, hipStream_t stream)
{
    a.topK == 1   ? LaunchRouteTile<T, 1>(a, tile, stream)
    : a.topK == 2 ? LaunchRouteTile<T, 2>(a, tile, stream)
    : a.topK <= 4 ? LaunchRouteTile<T, 4>(a, tile, stream)
    : a.topK <= 8 ? LaunchRouteTile<T, 8>(a, tile, stream)
                  : LaunchRouteTile<T, 16>(a, tile, stream);
}

template <typename T, bool kWide>
void LaunchRouteGrad(const RouteGradArgs &a, hipStream_t stream)
{
    const auto go = [&](auto kernel, int lanes) {
        const int64_t blocks = (int64_t(a.tokens) * lanes + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(kernel, dim3(uint32_t(blocks)), dim3(kThreads), 0, stream, a);
    };
    if (a.experts <= 64) {
        go(RouteGradKernel<T, 16, 4, kWide>, 16);
    } else if (a.experts <= 128) {
        go(RouteGradKernel<T, 16, 8, kWide>, 16);
    } else if (a.experts <= 256) {
        go(RouteGradKernel<T, 16, 16, kWide>, 16);
    } else {
        go(RouteGradKernel<T, 64, 16, kWide>, 64);
    }
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
    const uint64_t tile = uint64_t(TileOf(tokens, experts)), tiles = (tokens + tile - 1) / tile;
    *bytes = tiles <= 1 ? 0 : 4 * (tiles * (2 * uint64_t(experts) + 1) + experts);
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
        EXPERTS_CHK(logitStride == 0 || logitStride >= experts);
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
    a.tiles = tokens == 0 ? 1 : int((tokens + uint64_t(tile) - 1) / uint64_t(tile));   // no token: the one tile writes the zeros
    a.tileCounts = static_cast<int32_t *>(workspace);
    a.tileSums = reinterpret_cast<float *>(a.tileCounts + int64_t(a.tiles) * (a.experts + 1));
    a.sums = a.tileSums + int64_t(a.tiles) * a.experts;
    a.rowWords = RowWords(experts, kThreads / tile);
    a.lossScale = lossScale;
    a.renormalise = renormalise != 0;
    const hipStream_t on = static_cast<hipStream_t>(stream);
    logitType == HCCL_DATA_TYPE_FP32   ? LaunchRouteType<float>(a, tile, on)
    : logitType == HCCL_DATA_TYPE_FP16 ? LaunchRouteType<_Float16>(a, tile, on)
                                       : LaunchRouteType<__bf16>(a, tile, on);
    HcclResult r = Launched("HcclAmdExpertRoute");
    if (r != HCCL_SUCCESS || a.tiles == 1) {
        return r;
    }
    hipLaunchKernelGGL(TileScanKernel, dim3(experts / 16 + 1), dim3(kThreads), 0, on, a);
    r = Launched("HcclAmdExpertRoute");
    if (r != HCCL_SUCCESS) {
        return r;
    }
    const uint64_t blocks = (tokens * topK + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(RowsKernel, dim3(uint32_t(blocks < 512 ? blocks : 512)), dim3(kThreads), 4 * (2 * size_t(experts) + 2 * kThreads), on, a, tile);
    return Launched("HcclAmdExpertRoute");
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
    EXPERTS_CHK(logitStride == 0 || logitStride >= experts);
    EXPERTS_CHK(logitGradStride == 0 || logitGradStride >= experts);
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
    switch (logitType) {
        case HCCL_DATA_TYPE_FP32:
            wide ? LaunchRouteGrad<float, true>(a, on) : LaunchRouteGrad<float, false>(a, on);
            break;
        case HCCL_DATA_TYPE_FP16:
            wide ? LaunchRouteGrad<_Float16, true>(a, on) : LaunchRouteGrad<_Float16, false>(a, on);
            break;
        default:
            wide ? LaunchRouteGrad<__bf16, true>(a, on) : LaunchRouteGrad<__bf16, false>(a, on);
    }
    return Launched("HcclAmdExpertRouteGrad");
}

}  // extern "C"
