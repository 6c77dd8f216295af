// Products of 8-bit operands with a scale for each block of 128: HcclAmdBlockMatmul and HcclAmdBlockMatmulGradWeight.
//
//   y[r][c] = sum over blocks b of ra[r][b] * ca[c][b] * sum over the 128 values of b of rows[r][.] * cols[c][.]
//
// rows: a group's rows, or the output gradient's columns; cols: an expert's weights, or the columns of the experts' inputs.  Both
// are widened to 16 bits on their way from LDS into the matrix instruction, 16 x 16 x 32, four of which take a block of 128.  Its first
// operand is `cols`, so that a lane holds four neighbouring values of one row of the result.  Scales that are powers of two go into the
// widened values; 32-bit ones multiply a block's sum, which is then added in 32 bits.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.h"

namespace hcclamd {
namespace experts {
namespace {

struct ProductArgs {
    const uint8_t *rows, *cols;
    const void *rowScales, *colScales;
    const int32_t *offsets;
    const int32_t *expertOfGroup;
    void *out;
    int64_t rowPitch, colPitch, outPitch;   // bytes, bytes, elements
    int64_t rowScalePitch;                  // matmul: scales from one row to the next
    int numRows;                            // matmul: rows of all groups; gradient: n
    int numCols;                            // matmul: n; gradient: k
    int blocks;                             // matmul: blocks of 128 along k
    int groups, experts;
    int groupedRows;                        // gradient: rows of all groups
    int colTiles;
    bool accumulate;
    bool wideOut;                           // results can be stored 16 bytes at once
};

// Why not the 8-bit matrix instructions, whose rate is twice as high (4.4 for 2.2 PFLOP/s): inside a block of 128 they drop what is small
// next to the block's largest product.  Measured, off by (2-norm): normally distributed values 1.5e-5; values of one sign over the type's
// whole range 7e-5, always downwards, and up to 2.2e-4 at one result; two large products that cancel, all other values around 2 instead
// of 448: 0.15.  A sum in 32 bits is 3.5e-5 off there and 1e-8 to 1e-7 elsewhere; so are those of the 16-bit instruction: 8-bit values fit
// 16-bit ones exactly, and so does their product with a power of two.  Widening costs an instruction per two values.
typedef __bf16 Half8 __attribute__((ext_vector_type(8)));

struct Wide32 {     // a lane's 32 values of a block
    Half8 v[4];
};

__device__ __forceinline__ Wide32 Widen(const Int8 &x, float scale)
{
    Wide32 w;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(x[i]), scale, false);
        const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(uint32_t(x[i]), scale, true);
        w.v[i / 2][i % 2 * 4 + 0] = lo[0];
        w.v[i / 2][i % 2 * 4 + 1] = lo[1];
        w.v[i / 2][i % 2 * 4 + 2] = hi[0];
        w.v[i / 2][i % 2 * 4 + 3] = hi[1];
    }
    return w;
}

__device__ __forceinline__ Float4 MfmaWide(const Wide32 &cols, const Wide32 &rows, Float4 sum)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cols.v[i], rows.v[i], sum, 0, 0, 0);
    }
    return sum;
}

__device__ __forceinline__ float PowerOf(uint8_t scale) { return __uint_as_float(scale == 0 ? 0x400000u : uint32_t(scale) << 23); }

// What values are multiplied by as they are widened, and what is left for their sum.
__device__ __forceinline__ float Inside(uint8_t scale) { return PowerOf(scale); }
__device__ __forceinline__ float Inside(float) { return 1.0f; }

// A lane's 32 of the 128 bytes of a block: those at 16 * (lane / 16) and 64 behind.  Which of a block's values meet in which
// lane does not matter, as long as both operands are cut alike.
__device__ __forceinline__ Int8 LoadLane(const uint8_t *p)
{
    const Int4 lo = *reinterpret_cast<const Int4 *>(p), hi = *reinterpret_cast<const Int4 *>(p + 64);
    return Int8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
}

__device__ __forceinline__ Float4 Zero4() { return Float4{0.0f, 0.0f, 0.0f, 0.0f}; }

template <typename T>
__device__ __forceinline__ void StoreFour(T *out, const float (&v)[4], int col, int numCols)
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (col + i < numCols) {
            out[col + i] = T(v[i]);
        }
    }
}

// 16 kRF rows by 16 kCF columns of the result to a workgroup, whose kWaves waves share the blocks out among them, kAhead at a time, and
// add up through LDS: for few rows, where the weights' bytes are what takes time and as many waves as possible should be reading
// them, all they need next at once.  8 rows at 8 of 64 experts by 4096 x 2048 (67 MB of weights): 13.3 us, 5.0 TB/s, what a copy
// reaches; one row by 4096 x 8192 (34 MB): 8 us.
template <typename T, HcclAmdScaleType kScale, int kRF, int kCF, int kWaves, int kAhead>
__global__ void __launch_bounds__(64 * kWaves) FewRowsKernel(ProductArgs a)
{
    constexpr bool kPowers = kScale == HCCL_AMD_SCALE_E8M0;
    typedef typename BlockScale<kScale>::Stored Stored;
    __shared__ Float4 part[kWaves][kRF * kCF][64];
    const int unit = int(blockIdx.x) / a.colTiles, col0 = int(blockIdx.x) % a.colTiles * 16 * kCF;
    const Unit u = FindUnit(a.offsets, a.groups, a.numRows, unit, 16 * kRF);
    if (u.group < 0) {
        return;
    }
    const int expert = a.expertOfGroup == nullptr ? u.group : a.expertOfGroup[u.group];
    if (expert < 0 || expert >= a.experts) {
        return;
    }
    const int lane = int(threadIdx.x) % 64, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64), l16 = lane % 16, piece = lane / 16 * 16;
    const uint8_t *rows[kRF], *cols[kCF];
    const Stored *rowScales[kRF];
    Float4 sum[kRF][kCF];
#pragma unroll
    for (int r = 0; r < kRF; r++) {
        const int64_t row = min(u.first + r * 16 + l16, u.last - 1);
        rows[r] = a.rows + row * a.rowPitch + piece;
        rowScales[r] = static_cast<const Stored *>(a.rowScales) + row * a.rowScalePitch;
    }
    // (a workgroup's columns lie within one block of 128 of the weights' scales)
    const Stored *colScales = static_cast<const Stored *>(a.colScales) + (int64_t(expert) * ((a.numCols + 127) / 128) + col0 / 128) * a.blocks;
#pragma unroll
    for (int f = 0; f < kCF; f++) {
        const int col = min(col0 + f * 16 + l16, a.numCols - 1);
        cols[f] = a.cols + (int64_t(expert) * a.numCols + col) * a.colPitch + piece;
#pragma unroll
        for (int r = 0; r < kRF; r++) {
            sum[r][f] = Zero4();
        }
    }
    for (int b0 = wave; b0 < a.blocks; b0 += kWaves * kAhead) {
        Int8 x[kAhead][kRF], w[kAhead][kCF];
        Stored rs[kAhead][kRF], cs[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int b = min(b0 + j * kWaves, a.blocks - 1);       // (past the end the last one again, not used)
#pragma unroll
            for (int f = 0; f < kCF; f++) {
                w[j][f] = LoadLane(cols[f] + int64_t(b) * 128);
            }
#pragma unroll
            for (int r = 0; r < kRF; r++) {
                x[j][r] = LoadLane(rows[r] + int64_t(b) * 128);
                rs[j][r] = rowScales[r][b];
            }
            cs[j] = colScales[b];
        }
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            if (b0 + j * kWaves < a.blocks) {
                Wide32 wide[kRF];
#pragma unroll
                for (int r = 0; r < kRF; r++) {
                    wide[r] = Widen(x[j][r], Inside(rs[j][r]));
                }
#pragma unroll
                for (int f = 0; f < kCF; f++) {
                    const Wide32 wideCol = Widen(w[j][f], Inside(cs[j]));
#pragma unroll
                    for (int r = 0; r < kRF; r++) {
                        if constexpr (kPowers) {
                            sum[r][f] = MfmaWide(wideCol, wide[r], sum[r][f]);
                        } else {
                            const Float4 p = MfmaWide(wideCol, wide[r], Zero4());
                            const float s = rs[j][r] * cs[j];
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                sum[r][f][i] = __builtin_fmaf(p[i], s, sum[r][f][i]);
                            }
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kRF; r++) {
#pragma unroll
        for (int f = 0; f < kCF; f++) {
            part[wave][r * kCF + f][lane] = sum[r][f];
        }
    }
    __syncthreads();
    // the waves take the 16 x 16 parts in turn
    for (int at = wave; at < kRF * kCF; at += kWaves) {
        Float4 total = part[0][at][lane];
#pragma unroll
        for (int w = 1; w < kWaves; w++) {
            const Float4 other = part[w][at][lane];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                total[i] += other[i];
            }
        }
        const int row = u.first + at / kCF * 16 + l16;
        if (row < u.last) {
            const float v[4] = {total[0], total[1], total[2], total[3]};
            StoreFour(static_cast<T *>(a.out) + int64_t(row) * a.outPitch, v, col0 + at % kCF * 16 + lane / 16 * 4, a.numCols);
        }
    }
}

// f(first block, number of blocks, one at least) for every group of the expert that has rows, ascending; blocks count over all
// groups.  Called by whole waves.
template <typename F>
__device__ __forceinline__ void ForGroupsOf(const ProductArgs &a, int expert, F f)
{
    if (a.offsets == nullptr) {
        if (a.groupedRows > 0 && (a.expertOfGroup == nullptr ? 0 : a.expertOfGroup[0]) == expert) {
            f(0, (a.groupedRows + 127) / 128);
        }
        return;
    }
    const int lane = int(__lane_id());
    const int64_t most = int64_t(a.groupedRows) / 128 + a.groups;   // blocks there can be: none beyond is looked at
    int64_t before = 0;
    for (int g0 = 0; g0 < a.groups && before < most; g0 += 64) {
        const int g = g0 + lane;
        int n = 0;
        bool is = false;
        if (g < a.groups) {
            const int lo = min(max(a.offsets[g], 0), a.groupedRows), hi = min(max(a.offsets[g + 1], lo), a.groupedRows);
            n = (hi - lo + 127) / 128;
            is = n > 0 && (a.expertOfGroup == nullptr ? g : a.expertOfGroup[g]) == expert;
        }
        int sum = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int other = __shfl_up(sum, d, 64);
            sum += lane >= d ? other : 0;
        }
        unsigned long long left = __ballot(is);
        while (left != 0) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll(left) - 1);
            left &= left - 1;
            const int64_t first = before + __builtin_amdgcn_readlane(sum - n, at);
            const int64_t last = first + __builtin_amdgcn_readlane(n, at);
            if (first < most) {
                f(int(first), int((last < most ? last : most) - first));
            }
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
}

// ---- many rows -------------------------------------------------------------------------------------------

[[maybe_unused]] constexpr int kBufferFlags = 0x00027000;    // a raw buffer of 32-bit words
typedef __attribute__((address_space(3))) void *LdsBytes;

// How many units of `per` rows all groups make, `most` at most.  Called by all 64 lanes of a wave.
__device__ __forceinline__ int CountUnits(const int32_t *__restrict__ offsets, int groups, int rows, int per, int most)
{
    if (offsets == nullptr) {
        return min((rows + per - 1) / per, most);
    }
    int64_t sum = 0;
    for (int g = int(__lane_id()); g < groups; g += 64) {
        const int lo = min(max(offsets[g], 0), rows), hi = min(max(offsets[g + 1], lo), rows);
        sum += (hi - lo + per - 1) / per;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        sum += __shfl_xor(sum, d, 64);
    }
    return __builtin_amdgcn_readfirstlane(int(sum < most ? sum : most));
}

// Workgroups go to the eight XCDs in turn, each of which has an L2 cache of its own: every XCD takes a run of neighbouring tiles.
__device__ __forceinline__ int TileOf(int block, int tiles)
{
    const int xcd = block % 8, more = tiles % 8;
    return xcd * (tiles / 8) + min(xcd, more) + block / 8;
}

struct Place {
    int unit, col;
};

// A tile's place among units x colTiles: bands of eight columns of tiles,
// unit by unit, so that the 32 tiles an XCD works on at a time share four units' rows and eight tiles' columns.
__device__ __forceinline__ Place PlaceOf(int tile, int units, int colTiles)
{
    const int band = tile / (units * 8), width = min(8, colTiles - band * 8);
    tile -= band * units * 8;
    return Place{tile / width, band * 8 + tile % width};
}

// 16 bytes to a lane, from base + own + shared into LDS in lane order; what lies at `bytes` and beyond reads as zeros.  (The host's
// pass over this file does not know buffers.)
__device__ __forceinline__ void LoadToLds(const uint8_t *base, uint32_t bytes, uint8_t *lds, int own, int shared)
{
#if defined(__HIP_DEVICE_COMPILE__)
    const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(base), 0, int(bytes), kBufferFlags);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (LdsBytes)lds, 16, own, shared, 0, 0);
#endif
}

// Loads that have been sent into LDS have arrived.
__device__ __forceinline__ void LoadsDone() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ uint32_t ScaleBits(float s) { return __float_as_uint(s); }
__device__ __forceinline__ uint32_t ScaleBits(uint8_t s) { return s; }

// kWR x kWC waves of 16 kRF rows by 16 kCF columns each.  A step is one block of 128 values: its bytes go from memory into one
// of two LDS buffers while the other one is multiplied, eight rows of 128 bytes to a wave's load, without passing through
// registers.  The 16-byte pieces of a row lie in LDS in an order that depends on the row (piece p of row r at p ^ (r / 2 % 8)), so that the
// 16 rows a lane group reads are in different banks; since such a load fills LDS in lane order, it is the lanes' addresses
// in memory that are swapped.  Scales pass through a register of one thread each.
// Bound by the matrix unit and the vector unit together: 128 x 128 to a workgroup of four waves takes 128 conversions and, with 32-bit
// scales, 80 multiplications and sums a wave and step, for 64 products.  256 x 256 to eight waves takes 192 for 128 and all there is of LDS and
// registers.  Measured: 8192 x 4096 x 8192, scales of powers of two, 256 x 256: 383 us (1.44 PFLOP/s, what a library's 16-bit product reaches;
// matrix unit busy 65 % of the time, vector unit 49 %), 128 x 128: 443; 32-bit scales 456 (1.2), where 256 x 256 takes 480.  32768 rows of 64 experts by
// 4096 x 2048, 32-bit scales: 563 us (0.98; 49 and 57 %), a ninth of it tiles that are not full.  The weights' gradient of 16 experts, 16411 rows,
// 2048 x 4096: 337 us (0.82; 37 and 55 %), of which its 0.5 GB of results take 100; added to what is there, 577.
// (Two waves to a SIMD are asked for: with the registers of one the compiler keeps products apart from what it computes with.)
// kGrad: the weights' gradient, scales by column too.
template <typename T, HcclAmdScaleType kScale, bool kGrad, int kRF, int kCF, int kWR, int kWC>
__global__ void __launch_bounds__(64 * kWR * kWC, 2) TileKernel(ProductArgs a)
{
    constexpr bool kPowers = kScale == HCCL_AMD_SCALE_E8M0;
    typedef typename BlockScale<kScale>::Stored Stored;
    constexpr int kTileRows = 16 * kRF * kWR, kTileCols = 16 * kCF * kWC, kTileWaves = kWR * kWC, kTileThreads = 64 * kTileWaves;
    constexpr int kLoads = (kTileRows + kTileCols) / 8 / kTileWaves, kRowLoads = kTileRows / 8 / kTileWaves;
    constexpr int kScales = (kTileRows + kTileCols + kTileThreads - 1) / kTileThreads;   // to a thread (past the last column's: that again)
    static_assert(kTileRows % (8 * kTileWaves) == 0 && kTileCols % (8 * kTileWaves) == 0, "whole loads");
    // (two variables, not halves of one: the compiler waits for all loads into LDS before it reads what they might write)
    __shared__ __align__(16) uint8_t tile0[(kTileRows + kTileCols) * 128];
    __shared__ __align__(16) uint8_t tile1[(kTileRows + kTileCols) * 128];
    __shared__ __align__(16) uint32_t scales0[kScales * kTileThreads];
    __shared__ __align__(16) uint32_t scales1[kScales * kTileThreads];

    const int lane = int(threadIdx.x) % 64, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / 64);
    const int l16 = lane % 16, quarter = lane / 16;
    int expert, row0, rowEnd, col0;
    if constexpr (kGrad) {
        const int rowTiles = (a.numRows + kTileRows - 1) / kTileRows;
        // (experts one after the other, each cut among the XCDs: their rows, and with them their tiles' costs, differ)
        const int each = rowTiles * a.colTiles, more = each % 8, block = int(blockIdx.x) % (8 * (each / 8 + (more != 0)));
        expert = int(blockIdx.x) / (8 * (each / 8 + (more != 0)));
        if (block / 8 >= each / 8 + (block % 8 < more)) {
            return;
        }
        const Place at = PlaceOf(TileOf(block, each), rowTiles, a.colTiles);
        row0 = at.unit * kTileRows;
        rowEnd = a.numRows;
        col0 = at.col * kTileCols;
    } else {
        const int units = CountUnits(a.offsets, a.groups, a.numRows, kTileRows, int(gridDim.x) / a.colTiles);
        if (int(blockIdx.x) >= units * a.colTiles) {
            return;
        }
        const Place at = PlaceOf(TileOf(int(blockIdx.x), units * a.colTiles), units, a.colTiles);
        const Unit u = FindUnit(a.offsets, a.groups, a.numRows, at.unit, kTileRows);
        if (u.group < 0) {
            return;
        }
        expert = a.expertOfGroup == nullptr ? u.group : a.expertOfGroup[u.group];
        if (expert < 0 || expert >= a.experts) {
            return;
        }
        row0 = u.first;
        rowEnd = u.last;
        col0 = at.col * kTileCols;
    }
    const int64_t colBase = kGrad ? 0 : int64_t(expert) * a.numCols;

    // what this lane loads: a 16-byte piece of a row, in every load (rows behind the last one are beyond the buffer and read as zeros)
    const uint8_t *rowsFrom = a.rows + int64_t(row0) * a.rowPitch, *colsFrom = a.cols + (colBase + col0) * a.colPitch;
    const uint32_t rowBytes = uint32_t(min(rowEnd - row0, kTileRows)) * uint32_t(a.rowPitch);
    const uint32_t colBytes = uint32_t(min(a.numCols - col0, kTileCols)) * uint32_t(a.colPitch);
    int from[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; j++) {
        const int oct = (j < kRowLoads ? j : j - kRowLoads) * kTileWaves + wave, piece = (lane % 8) ^ (lane / 16 + 4 * (oct % 2));
        from[j] = int(uint32_t(oct * 8 + lane / 8) * uint32_t(j < kRowLoads ? a.rowPitch : a.colPitch) + uint32_t(piece * 16));
    }
    // and its scales
    const Stored *scaleFrom[kScales];
    int64_t scaleStep[kScales];
#pragma unroll
    for (int j = 0; j < kScales; j++) {
        const int i = int(threadIdx.x) + j * kTileThreads;
        if (i < kTileRows) {
            const int64_t row = min(row0 + i, rowEnd - 1);
            scaleFrom[j] = static_cast<const Stored *>(a.rowScales) + (kGrad ? row : row * a.rowScalePitch);
            scaleStep[j] = kGrad ? a.numRows : 1;
        } else {
            const int64_t col = min(col0 + i - kTileRows, a.numCols - 1);
            scaleFrom[j] = static_cast<const Stored *>(a.colScales) + (kGrad ? col : (int64_t(expert) * ((a.numCols + 127) / 128) + col / 128) * a.blocks);
            scaleStep[j] = kGrad ? a.numCols : 1;
        }
    }
    uint32_t coming[kScales];
    // Sends for a block; with `any` false for none: everything lies beyond an empty buffer, which costs no traffic, and the code of
    // a step has no branch the scheduler could not look past.
    const auto fetch = [&](int block, bool any, uint8_t *tile) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kLoads; j++) {
            const int oct = (j < kRowLoads ? j : j - kRowLoads) * kTileWaves + wave;
            uint8_t *lds = tile + ((j < kRowLoads ? 0 : kTileRows) + oct * 8) * 128;
            LoadToLds(j < kRowLoads ? rowsFrom : colsFrom, !any ? 0 : j < kRowLoads ? rowBytes : colBytes, lds, from[j], block * 128);
        }
#pragma unroll
        for (int j = 0; j < kScales; j++) {
            coming[j] = ScaleBits(scaleFrom[j][block * scaleStep[j]]);
        }
    };

    const int rowAt = wave / kWC * 16 * kRF, colAt = wave % kWC * 16 * kCF;     // of this wave, in the tile
    const int laneAt = l16 * 128 + ((quarter ^ (l16 / 2)) * 16);
    const auto fragment = [&](const uint8_t *rows16) {
        const Int4 lo = *reinterpret_cast<const Int4 *>(rows16 + laneAt), hi = *reinterpret_cast<const Int4 *>(rows16 + (laneAt ^ 64));
        return Int8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    };
    Float4 sum[kRF][kCF];
#pragma unroll
    for (int r = 0; r < kRF; r++) {
#pragma unroll
        for (int c = 0; c < kCF; c++) {
            sum[r][c] = Zero4();
        }
    }
    const auto keepScales = [&](uint32_t *scale) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kScales; j++) {
            scale[int(threadIdx.x) + j * kTileThreads] = coming[j];
        }
    };
    // One step: the block after it is sent for first, then this one is read, widened and multiplied, in the order the compiler likes
    // (widening between the products).
    const auto step = [&](uint8_t *tile, uint32_t *scale, uint8_t *other, int next, int last) __attribute__((always_inline)) {
        keepScales(scale);
        LoadsDone();
        __syncthreads();     // this block is there, and nobody reads the other buffer any more
        fetch(min(next, last), next <= last, other);
        const uint8_t *rows = tile + rowAt * 128, *cols = tile + (kTileRows + colAt) * 128;
        const uint32_t *rowScale = scale + rowAt, *colScale = scale + kTileRows + colAt;
        Wide32 wide[kCF];
        float cs[kCF][4];
#pragma unroll
        for (int c = 0; c < kCF; c++) {
            wide[c] = Widen(fragment(cols + c * 16 * 128), kPowers ? PowerOf(uint8_t(colScale[c * 16 + l16])) : 1.0f);
            if constexpr (!kPowers) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    cs[c][i] = __uint_as_float(colScale[kGrad ? c * 16 + quarter * 4 + i : 0]);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < kRF; r++) {
            const uint32_t power = rowScale[r * 16 + l16];
            const Wide32 wideRow = Widen(fragment(rows + r * 16 * 128), kPowers ? PowerOf(uint8_t(power)) : 1.0f);
#pragma unroll
            for (int c = 0; c < kCF; c++) {
                if constexpr (kPowers) {
                    sum[r][c] = MfmaWide(wide[c], wideRow, sum[r][c]);
                } else {
                    const Float4 p = MfmaWide(wide[c], wideRow, Zero4());
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        sum[r][c][i] = __builtin_fmaf(p[i], __uint_as_float(power) * cs[c][i], sum[r][c][i]);
                    }
                }
            }
        }
    };
    // A wave all of whose rows lie behind the group's last one only loads.
    const bool idle = !kGrad && row0 + rowAt >= rowEnd;
    const auto idleStep = [&](uint8_t *to, uint32_t *scale, int next, int last) __attribute__((always_inline)) {
        keepScales(scale);
        LoadsDone();
        __syncthreads();
        fetch(min(next, last), next <= last, to);
    };
    const auto run = [&](int first, int count) __attribute__((always_inline)) {
        const int last = first + count - 1;
        LoadsDone();
        __syncthreads();     // (the buffers are free: the blocks of another group may have been in them)
        fetch(first, true, tile0);
        for (int i = 0; idle && i < count; i++) {
            idleStep(i % 2 == 0 ? tile1 : tile0, i % 2 == 0 ? scales0 : scales1, first + i + 1, last);
        }
        for (int i = 0; !idle && i < count; i += 2) {
            step(tile0, scales0, tile1, first + i + 1, last);
            if (i + 1 < count) {
                step(tile1, scales1, tile0, first + i + 2, last);
            }
        }
    };
    if constexpr (kGrad) {
        ForGroupsOf(a, expert, run);
    } else {
        if (a.blocks > 0) {
            run(0, a.blocks);
        }
    }

    // Out through LDS: a lane holds four neighbours of a row, the lanes of an instruction 16 rows; what leaves is whole rows of the
    // wave's part, 16 bytes to a lane.  Pieces of a row lie in an order that depends on the row here too.
    constexpr int kRowBytes = 16 * kCF * int(sizeof(T)), kPieces = kRowBytes / 16, kPer = 16 / int(sizeof(T));
    constexpr int kWaveBytes = 16 * kRF * kRowBytes, kHalf = kTileWaves / 2;
    static_assert(kWaveBytes * kHalf <= int(sizeof(tile0)), "the results fit the buffers");
    LoadsDone();
    __syncthreads();
    uint8_t *mine = wave < kHalf ? tile0 + wave * kWaveBytes : tile1 + (wave - kHalf) * kWaveBytes;
    const int64_t base = kGrad ? int64_t(expert) * a.numRows : 0;
    const auto key = [](int row) { return sizeof(T) == 4 ? row % kPieces : row / 2 % kPieces; };
#pragma unroll
    for (int r = 0; r < kRF; r++) {
#pragma unroll
        for (int c = 0; c < kCF; c++) {
            const int row = r * 16 + l16, byte = (c * 16 + quarter * 4) * int(sizeof(T));
            float v[4] = {sum[r][c][0], sum[r][c][1], sum[r][c][2], sum[r][c][3]};
            if (kGrad && a.accumulate) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int to = row0 + rowAt + row, col = col0 + colAt + c * 16 + quarter * 4 + i;
                    if (to < rowEnd && col < a.numCols) {
                        v[i] += float(static_cast<const T *>(a.out)[(base + to) * a.outPitch + col]);
                    }
                }
            }
            Store<true, 4>(reinterpret_cast<T *>(mine + row * kRowBytes + ((byte / 16 ^ key(row)) * 16 + byte % 16)), v);
        }
    }
#pragma unroll
    for (int i = 0; i < 16 * kRF * kPieces / 64; i++) {
        const int at = i * 64 + lane, rowHere = at / kPieces, row = row0 + rowAt + rowHere, col = col0 + colAt + at % kPieces * kPer;
        typedef T Vec __attribute__((ext_vector_type(kPer), aligned(16)));
        const Vec v = *reinterpret_cast<const Vec *>(mine + rowHere * kRowBytes + ((at % kPieces) ^ key(rowHere)) * 16);
        if (row >= rowEnd) {
            continue;
        }
        T *out = static_cast<T *>(a.out) + (base + row) * a.outPitch + col;
        if (a.wideOut && col < a.numCols) {
            __builtin_nontemporal_store(v, reinterpret_cast<Vec *>(out));
        } else if (!a.wideOut) {
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                if (col + j < a.numCols) {
                    out[j] = v[j];
                }
            }
        }
    }
}

// f(type, scale type) as constants
template <typename F>
HcclResult Choose(HcclDataType type, HcclAmdScaleType scaleType, F f)
{
    const auto byScale = [&](auto of) {
        return scaleType == HCCL_AMD_SCALE_FP32 ? f(of, std::integral_constant<HcclAmdScaleType, HCCL_AMD_SCALE_FP32>{})
                                                : f(of, std::integral_constant<HcclAmdScaleType, HCCL_AMD_SCALE_E8M0>{});
    };
    switch (type) {
        case HCCL_DATA_TYPE_FP32:
            return byScale(float{});
        case HCCL_DATA_TYPE_FP16:
            return byScale(_Float16{});
        default:
            return byScale(__bf16{});
    }
}

constexpr uint64_t kMostTiles = uint64_t(1) << 22;   // workgroups of up to 512 below 2^32 threads

// What a product takes in each form, in microseconds: `call`, and for every 256 workgroups, one to a compute unit, `round` and `block` times the
// blocks of 128 along its sums.  The form that should take least is taken.  The figures are least squares of the relative errors, rounded, over 876
// products: 1 to 128 groups, 1 to 12000 rows, 300 to 14336 columns, sums of 300 to 8192 values (256 x 256: over 28).  What is taken so is
// 1.4 % slower than the fastest of all on average, in 9 of the 876 by more than a quarter.  For instance, columns x sum, us in the order below:
//   one group     4096 x 8192:    1 row    8   20   22   58;   64 rows  38   24   31   60;   256 rows 142   81   54   68;   2048 rows  -   -   -  126
//                 1408 x 2048:    4 rows   6    7    7   17;   96 rows  16    9   10   19;   800 rows  82   30   24   20
//   64 groups     4096 x 2048:    8 rows  21   13   14   19;   60 groups, 1408 x 2048: 800 rows 105 42 37 41, 1500 rows 177 64 49 41
//   256 x 256 against 128 x 128, scales of powers of two, 4096 columns: 2048 rows x 8192 177 and 119, 4096 rows x 8192 190 and 228, 8192 rows x 1024 59
//                 and 63, x 512 36 and 35.  With 32-bit scales the larger is 2 % faster at best, mostly slower (8192 x 4096 x 8192: 480 and 444).
struct Form {
    uint32_t rows, cols;
    double call, round, block;
};
constexpr Form kNarrow = {16, 16, 2.4, 1.4, 0.1}, kFew = {16, 64, 3.0, 0.45, 0.3}, kTwice = {32, 64, 2.7, 0.75, 0.355};
constexpr Form kTile = {128, 128, 3.1, 1.0, 0.9}, kLargeTile = {256, 256, 3.0, 4.0, 2.85};

// How many groups have rows, and how many units their rows make, is known on the device only.  If rows fall to groups at random, `hit` of them have
// some; half of the last unit of each is counted, since the others' rows fill up one that is counted already.
double TimeOf(const Form &form, uint64_t rows, uint64_t groups, uint64_t n, uint64_t blocks)
{
    const uint64_t colTiles = (n + form.cols - 1) / form.cols;
    double units = double((rows + form.rows - 1) / form.rows);
    if (groups > 1) {
        const double hit = double(rows) * double(groups) / double(rows + groups);
        units = std::max(double(rows) / form.rows + hit / 2, hit);
    }
    return form.call + std::ceil(units * double(colTiles) / 256) * (form.round + form.block * double(blocks));
}

constexpr int64_t kMostPitch = int64_t(1) << 23;     // bytes of a row: those of a tile's 256 rows are within 2^31

bool WideOut(HcclDataType type, uint64_t width, const void *p, int64_t pitch)
{
    return width * SizeOf(type) % 16 == 0 && uint64_t(pitch) * SizeOf(type) % 16 == 0 && Aligned(p, 16);
}

}  // namespace
}  // namespace experts
}  // namespace hcclamd

using namespace hcclamd::experts;

extern "C" {

HcclResult HcclAmdBlockMatmul(const void *a, uint64_t aStride, const void *aScales, uint64_t aScaleStride, uint64_t rows,
    uint32_t groups, const int32_t *offsets, const int32_t *expertOfGroup, const void *w, const void *wScales, uint32_t experts,
    uint64_t n, uint64_t k, HcclAmdScaleType scaleType, void *y, HcclDataType yType, uint64_t yStride, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(yType));
    EXPERTS_CHK_TYPE(Scaled(scaleType));
    EXPERTS_CHK(rows <= kMaxGroupedRows && n <= kMaxSize - 256 && k <= kMaxSize - 256);
    EXPERTS_CHK(groups >= 1 && groups <= HCCL_AMD_MAX_GROUPS && experts >= 1 && experts <= HCCL_AMD_MAX_GROUPS);
    EXPERTS_CHK(offsets != nullptr || groups == 1);
    EXPERTS_CHK(expertOfGroup != nullptr || groups <= experts);
    if (rows == 0 || n == 0) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(y);
    if (k != 0) {
        EXPERTS_CHK_PTR(a);
        EXPERTS_CHK_PTR(aScales);
        EXPERTS_CHK_PTR(w);
        EXPERTS_CHK_PTR(wScales);
    }
    ProductArgs p{};
    p.rows = static_cast<const uint8_t *>(a);
    p.cols = static_cast<const uint8_t *>(w);
    p.rowScales = aScales;
    p.colScales = wScales;
    p.offsets = offsets;
    p.expertOfGroup = expertOfGroup;
    p.out = y;
    p.rowPitch = int64_t(aStride == 0 ? Up128(k) : aStride);
    p.colPitch = int64_t(Up128(k));
    p.outPitch = int64_t(yStride == 0 ? n : yStride);
    p.rowScalePitch = int64_t(aScaleStride == 0 ? Blocks(k) : aScaleStride);
    p.numRows = int(rows);
    p.numCols = int(n);
    p.blocks = int(Blocks(k));
    p.groups = int(groups);
    p.experts = int(experts);
    EXPERTS_CHK(Stride(aStride, Up128(k)) && aStride % 16 == 0 && Aligned(a, 16) && Aligned(w, 16));
    EXPERTS_CHK(Stride(aScaleStride, Blocks(k)) && ScaleAligned(scaleType, aScales) && ScaleAligned(scaleType, wScales));
    EXPERTS_CHK(Stride(yStride, n) && AlignedTo(yType, y));
    EXPERTS_CHK(Aligned(offsets, 4) && Aligned(expertOfGroup, 4));
    p.wideOut = WideOut(yType, n, y, p.outPitch);
    const auto columnsOf = [&](const Form &form) { return (n + form.cols - 1) / form.cols; };
    // units there can be: every group that has rows ends with a shorter one
    const auto unitsOf = [&](const Form &form) {
        return offsets == nullptr ? (rows + form.rows - 1) / form.rows : rows / form.rows + std::min<uint64_t>(rows, groups);
    };
    EXPERTS_CHK(unitsOf(kTile) * columnsOf(kTile) <= kMostTiles);
    const Form *form = &kTile;
    for (const Form *other : {&kNarrow, &kFew, &kTwice, &kLargeTile}) {
        const bool can = other != &kLargeTile || (scaleType == HCCL_AMD_SCALE_E8M0 && yType != HCCL_DATA_TYPE_FP32);
        if (can && unitsOf(*other) * columnsOf(*other) <= kMostTiles &&
            TimeOf(*other, rows, groups, n, Blocks(k)) < TimeOf(*form, rows, groups, n, Blocks(k))) {
            form = other;
        }
    }
    p.colTiles = int(columnsOf(*form));
    const uint64_t units = unitsOf(*form);
    EXPERTS_CHK(p.rowPitch < kMostPitch && p.colPitch < kMostPitch);
    return Choose(yType, scaleType, [&](auto of, auto scale) {
        typedef decltype(of) T;
        constexpr HcclAmdScaleType kScale = decltype(scale)::value;
        const auto go = [&](auto kernel, int threads) {
            return Launch("HcclAmdBlockMatmul", kernel, uint32_t(units * uint64_t(p.colTiles)), threads, 0, static_cast<hipStream_t>(stream), p);
        };
        if (form == &kNarrow) {
            return go(FewRowsKernel<T, kScale, 1, 1, 8, 4>, 512);
        }
        if (form == &kFew) {
            return go(FewRowsKernel<T, kScale, 1, 4, 4, 2>, 256);
        }
        if (form == &kTwice) {
            return go(FewRowsKernel<T, kScale, 2, 4, 4, 2>, 256);
        }
        if constexpr (sizeof(T) == 2 && kScale == HCCL_AMD_SCALE_E8M0) {
            if (form == &kLargeTile) {
                return go(TileKernel<T, kScale, false, 8, 4, 2, 4>, 512);
            }
        }
        return go(TileKernel<T, kScale, false, 4, 4, 2, 2>, 256);
    });
}

HcclResult HcclAmdBlockMatmulGradWeight(const void *yGradT, const void *yGradScales, const void *xT, const void *xScales,
    uint64_t columns, uint64_t rows, uint64_t n, uint64_t k, HcclAmdScaleType scaleType, uint32_t groups, const int32_t *offsets,
    const int32_t *expertOfGroup, uint32_t experts, void *wGrad, HcclDataType gradType, uint32_t accumulate, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_TYPE(Float(gradType));
    EXPERTS_CHK_TYPE(Scaled(scaleType));
    EXPERTS_CHK(rows <= kMaxGroupedRows && n <= kMaxSize - 256 && k <= kMaxSize - 256);
    EXPERTS_CHK(groups >= 1 && groups <= HCCL_AMD_MAX_GROUPS && experts >= 1 && experts <= HCCL_AMD_MAX_GROUPS);
    EXPERTS_CHK(offsets != nullptr || groups == 1);
    EXPERTS_CHK(expertOfGroup != nullptr || groups <= experts);
    EXPERTS_CHK(columns % 128 == 0 && columns >= (rows / 128 + groups) * 128 && columns <= kMaxSize);
    if (n == 0 || k == 0) {
        return HCCL_SUCCESS;
    }
    EXPERTS_CHK_PTR(wGrad);
    if (rows != 0) {
        EXPERTS_CHK_PTR(yGradT);
        EXPERTS_CHK_PTR(yGradScales);
        EXPERTS_CHK_PTR(xT);
        EXPERTS_CHK_PTR(xScales);
    }
    EXPERTS_CHK(Aligned(yGradT, 16) && Aligned(xT, 16) && ScaleAligned(scaleType, yGradScales) && ScaleAligned(scaleType, xScales));
    EXPERTS_CHK(AlignedTo(gradType, wGrad) && Aligned(offsets, 4) && Aligned(expertOfGroup, 4));
    ProductArgs p{};
    p.rows = static_cast<const uint8_t *>(yGradT);
    p.cols = static_cast<const uint8_t *>(xT);
    p.rowScales = yGradScales;
    p.colScales = xScales;
    p.offsets = offsets;
    p.expertOfGroup = expertOfGroup;
    p.out = wGrad;
    p.rowPitch = p.colPitch = int64_t(columns);
    p.outPitch = int64_t(k);
    p.numRows = int(n);
    p.numCols = int(k);
    p.groups = int(groups);
    p.experts = int(experts);
    p.groupedRows = int(rows);
    p.accumulate = accumulate != 0;
    EXPERTS_CHK(p.rowPitch < kMostPitch);
    p.wideOut = WideOut(gradType, k, wGrad, p.outPitch);
    p.colTiles = int((k + 127) / 128);
    const uint64_t tiles = ((n + 127) / 128 * uint64_t(p.colTiles) + 7) / 8 * 8 * experts;
    EXPERTS_CHK(tiles <= kMostTiles);
    return Choose(gradType, scaleType, [&](auto of, auto scale) {
        return Launch("HcclAmdBlockMatmulGradWeight", TileKernel<decltype(of), decltype(scale)::value, true, 4, 4, 2, 2>, uint32_t(tiles), 256, 0,
            static_cast<hipStream_t>(stream), p);
    });
}

}  // extern "C"
