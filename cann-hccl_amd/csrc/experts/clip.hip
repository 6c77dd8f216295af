// Gradients of many tensors held to a norm over all of them: HcclAmdGradSquares, HcclAmdGradClip.
//
// The tensors' table rides in the kernel arguments, up to 120 to a launch; tensors are cut into chunks, counted over the table, and a wave finds its
// chunk's tensor by looking at all of them at once.  Chunks start at 16-byte boundaries of the input, so that every load inside a tensor is aligned whatever its first
// element is.  Squares are added up in 64 bits: those of 32 bits are exact there, and neither 1e30 nor 1e-30 leaves the range.  A workgroup's sum has
// its own place in the workspace and a second launch adds the places up in their order: same inputs, same bits.
//
// Bytes moved bound both: 2^30 values in 16 bits (2.1 GB) are added up in 360 us, 6.0 TB/s, and scaled in 710 us, 6.0 TB/s, where a large copy reaches
// 5.15.  Four parts of 2048 elements to a chunk leave room for eight waves to a SIMD, so that all 2048 workgroups run at once; with eight parts
// seven do, and the last eighth waited (1190 us for both instead of 1096).  Twenty short tensors: 2.9 us, 1.6 and 3.4, a launch's own time each.
#include <type_traits>

#include "sums.h"

namespace hcclamd {
namespace experts {
namespace {

constexpr int kThreads = 256;
constexpr int kEach = 8;                           // neighbouring elements of a lane
constexpr int kPart = kThreads * kEach;            // elements that a workgroup takes at once
constexpr int kShort = 1, kLong = 4;               // such parts of a chunk
constexpr int kFew = 32, kMany = 120;              // tensors of a launch; 120 take 3840 of the 4096 bytes that arguments may
constexpr int kMostSlots = 2048;                   // workgroups of a launch that adds up: eight to a compute unit
constexpr uint32_t kMaxTensors = 1u << 24;         // of a list: its places are counted in 32 bits
constexpr uint64_t kMaxCount = uint64_t(1) << 36;  // elements of a tensor; the chunks of a launch are counted in 32 bits

struct Tensor {
    const void *in;       // moved down to a 16-byte boundary,
    void *out;            // and as many elements here
    int64_t last;         // elements from there to the tensor's end
    int32_t chunk;        // its first chunk's number
    int16_t type;
    int16_t lead;         // elements in front of the tensor's first
};
static_assert(sizeof(Tensor) == 32, "32 bytes a tensor");

template <int kTensors>
struct Table {
    Tensor tensor[kTensors];
    int32_t n, chunks;
};

// The tensor that `chunk` is of: as many as begin at or before it, less one.  Called by whole waves.
template <int kTensors>
__device__ __forceinline__ int Find(const Table<kTensors> &t, int chunk)
{
    int found = -1;
#pragma unroll
    for (int i = 0; i < kTensors; i += 64) {
        const int at = i + int(__lane_id());
        found += __popcll(__ballot(at < t.n && t.tensor[at < kTensors ? at : 0].chunk <= chunk));
    }
    return __builtin_amdgcn_readfirstlane(found);
}

// One of a lane's parts at the ends of a tensor, zeros outside.
template <typename T>
__device__ __forceinline__ void LoadEdge(const Tensor &t, int64_t at, float (&v)[kEach])
{
    const T *in = static_cast<const T *>(t.in);
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        v[i] = 0.0f;
    }
    if (at >= t.lead && at + kEach <= t.last) {
        Load<true, kEach>(in + at, v);
    } else if (at + kEach > t.lead && at < t.last) {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            v[i] = at + i >= t.lead && at + i < t.last ? float(in[at + i]) : 0.0f;
        }
    }
}

template <typename T, int kParts>
__device__ __forceinline__ double Squares(const Tensor &t, int chunk)
{
    const T *in = static_cast<const T *>(t.in);
    const int64_t from = int64_t(chunk - t.chunk) * (kParts * kPart) + int(threadIdx.x) * kEach;
    const int64_t whole = int64_t(chunk - t.chunk) * (kParts * kPart);
    double sum[2] = {0.0, 0.0};
    const auto add = [&](const float (&v)[kEach]) {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            sum[i % 2] = __builtin_fma(double(v[i]), double(v[i]), sum[i % 2]);
        }
    };
    if (whole >= t.lead && whole + kParts * kPart <= t.last) {
        float v[kParts][kEach];
#pragma unroll
        for (int p = 0; p < kParts; p++) {
            Load<true, kEach>(in + from + p * kPart, v[p]);
        }
#pragma unroll
        for (int p = 0; p < kParts; p++) {
            add(v[p]);
        }
    } else {
#pragma unroll 1
        for (int p = 0; p < kParts && whole + p * kPart < t.last; p++) {
            float v[kEach];
            LoadEdge<T>(t, from + p * kPart, v);
            add(v);
        }
    }
    return sum[0] + sum[1];
}

template <int kTensors, int kParts>
__global__ void __launch_bounds__(kThreads) SquaresKernel(Table<kTensors> t, double *slots)
{
    __shared__ double parts[kThreads / 64];
    double sum = 0.0;
    for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        const Tensor &of = t.tensor[Find(t, chunk)];
        switch (of.type) {
            case HCCL_DATA_TYPE_FP32:
                sum += Squares<float, kParts>(of, chunk);
                break;
            case HCCL_DATA_TYPE_FP16:
                sum += Squares<_Float16, kParts>(of, chunk);
                break;
            default:
                sum += Squares<__bf16, kParts>(of, chunk);
                break;
        }
    }
    sum = AddWave(sum);
    if (threadIdx.x % 64 == 0) {
        parts[threadIdx.x / 64] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        slots[blockIdx.x] = (parts[0] + parts[1]) + (parts[2] + parts[3]);
    }
}

__global__ void __launch_bounds__(1024) AddSlotsKernel(const double *slots, int n, double *squares, bool accumulate)
{
    __shared__ double parts[1024 / 64];
    double sum = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 1024) {
        sum += slots[i];
    }
    sum = AddWave(sum);
    if (threadIdx.x % 64 == 0) {
        parts[threadIdx.x / 64] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = accumulate ? squares[0] : 0.0;
#pragma unroll
        for (int i = 0; i < 1024 / 64; i++) {
            sum += parts[i];
        }
        squares[0] = sum;
    }
}

template <typename T, int kParts>
__device__ __forceinline__ void Scale(const Tensor &t, int chunk, float by)
{
    const T *in = static_cast<const T *>(t.in);
    T *out = static_cast<T *>(t.out);
    const int64_t whole = int64_t(chunk - t.chunk) * (kParts * kPart), from = whole + int(threadIdx.x) * kEach;
    const bool aligned = reinterpret_cast<uintptr_t>(out) % 16 == 0;
    const auto store = [&](int64_t at, float (&v)[kEach]) {
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            v[i] *= by;
        }
        if (aligned) {
            Store<true, kEach>(out + at, v);
        } else {
            Store<false, kEach>(out + at, v);
        }
    };
    if (whole >= t.lead && whole + kParts * kPart <= t.last) {
        float v[kParts][kEach];
#pragma unroll
        for (int p = 0; p < kParts; p++) {
            Load<true, kEach>(in + from + p * kPart, v[p]);
        }
#pragma unroll
        for (int p = 0; p < kParts; p++) {
            store(from + p * kPart, v[p]);
        }
        return;
    }
#pragma unroll 1
    for (int p = 0; p < kParts && whole + p * kPart < t.last; p++) {
        const int64_t at = from + p * kPart;
        float v[kEach];
        LoadEdge<T>(t, at, v);
        if (at >= t.lead && at + kEach <= t.last) {
            store(at, v);
        } else if (at + kEach > t.lead && at < t.last) {
#pragma unroll
            for (int i = 0; i < kEach; i++) {
                if (at + i >= t.lead && at + i < t.last) {
                    out[at + i] = T(v[i] * by);
                }
            }
        }
    }
}

// The first workgroup of the list's first launch (`norm` not null) leaves the norm.
template <int kTensors, int kParts>
__global__ void __launch_bounds__(kThreads) ClipKernel(Table<kTensors> t, const double *squares, float maxNorm, float *norm)
{
    const double length = __builtin_sqrt(squares[0]);
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
        norm[0] = float(length);
    }
    const bool within = length <= double(maxNorm);        // (not so where the norm is NaN)
    const float by = within ? 1.0f : float(double(maxNorm) / length);
    for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        const Tensor &of = t.tensor[Find(t, chunk)];
        if (within && of.out == of.in) {
            continue;
        }
        switch (of.type) {
            case HCCL_DATA_TYPE_FP32:
                Scale<float, kParts>(of, chunk, by);
                break;
            case HCCL_DATA_TYPE_FP16:
                Scale<_Float16, kParts>(of, chunk, by);
                break;
            default:
                Scale<__bf16, kParts>(of, chunk, by);
                break;
        }
    }
}

HcclResult Check(const char *fn, const HcclAmdGradTensor *tensors, uint32_t n, bool write)
{
    if (n > kMaxTensors) {
        HCCL_LOG_ERROR("%s: %u tensors", fn, n);
        return HCCL_E_PARA;
    }
    for (uint32_t i = 0; i < n; i++) {
        const HcclAmdGradTensor &t = tensors[i];
        if (!Float(t.type)) {
            HCCL_LOG_ERROR("%s: tensor %u: type not supported", fn, i);
            return HCCL_E_NOT_SUPPORT;
        }
        if (t.count > kMaxCount || t.reserved != 0 || !AlignedTo(t.type, t.in) || (write && !AlignedTo(t.type, t.out))) {
            HCCL_LOG_ERROR("%s: tensor %u: count or alignment", fn, i);
            return HCCL_E_PARA;
        }
        if (t.count != 0 && (t.in == nullptr || (write && t.out == nullptr))) {
            HCCL_LOG_ERROR("%s: tensor %u is null", fn, i);
            return HCCL_E_PTR;
        }
    }
    return HCCL_SUCCESS;
}

// The next launch's table, from tensor `at` on, which is moved behind it; false: there are no more elements.
template <int kTensors>
bool Next(const HcclAmdGradTensor *tensors, uint32_t n, int parts, uint32_t &at, Table<kTensors> &table)
{
    const uint64_t chunk = uint64_t(parts) * kPart;
    table.n = table.chunks = 0;
    for (; at < n && table.n < kTensors; at++) {
        const HcclAmdGradTensor &t = tensors[at];
        if (t.count == 0) {
            continue;
        }
        const uint64_t unit = SizeOf(t.type), lead = reinterpret_cast<uintptr_t>(t.in) % 16 / unit;
        Tensor &to = table.tensor[table.n++];
        to.in = reinterpret_cast<const void *>(reinterpret_cast<uintptr_t>(t.in) - lead * unit);
        to.out = reinterpret_cast<void *>(reinterpret_cast<uintptr_t>(t.out) - lead * unit);
        to.last = int64_t(t.count + lead);
        to.chunk = table.chunks;
        to.type = int16_t(t.type);
        to.lead = int16_t(lead);
        table.chunks += int32_t((t.count + lead + chunk - 1) / chunk);
    }
    return table.n != 0;
}

int Slots(int chunks) { return chunks < kMostSlots ? chunks : kMostSlots; }

// Parts of a chunk: as many as load well together, one where the chunks would not be enough for two workgroups to each compute unit.
int PartsOf(const HcclAmdGradTensor *tensors, uint32_t n)
{
    uint64_t parts = 0;
    for (uint32_t i = 0; i < n && parts < 512 * kLong; i++) {
        parts += (tensors[i].count + kPart - 1) / kPart;
    }
    return parts < 512 * kLong ? kShort : kLong;
}

template <int kTensors, int kParts>
HcclResult Squares(const HcclAmdGradTensor *tensors, uint32_t n, double *slots, int *used, hipStream_t on)
{
    Table<kTensors> table;
    for (uint32_t at = 0; Next(tensors, n, kParts, at, table);) {
        const int some = Slots(table.chunks);
        const HcclResult r = Launch("HcclAmdGradSquares", SquaresKernel<kTensors, kParts>, uint32_t(some), kThreads, 0, on, table, slots + *used);
        if (r != HCCL_SUCCESS) {
            return r;
        }
        *used += some;
    }
    return HCCL_SUCCESS;
}

template <int kTensors, int kParts>
HcclResult Clip(const HcclAmdGradTensor *tensors, uint32_t n, const double *squares, float maxNorm, float *norm, hipStream_t on)
{
    Table<kTensors> table;
    uint32_t at = 0;
    while (Next(tensors, n, kParts, at, table) || norm != nullptr) {
        // (no elements at all: the norm is left all the same)
        const int blocks = table.chunks < 1 ? 1 : table.chunks < (1 << 20) ? table.chunks : 1 << 20;
        const HcclResult r = Launch("HcclAmdGradClip", ClipKernel<kTensors, kParts>, uint32_t(blocks), kThreads, 0, on, table, squares, maxNorm, norm);
        if (r != HCCL_SUCCESS) {
            return r;
        }
        norm = nullptr;
    }
    return HCCL_SUCCESS;
}

// f(tensors of a launch, parts of a chunk), as constants.  A list of up to 32 tensors takes a launch with room for these alone: its arguments are a quarter
// as long.
template <typename F>
HcclResult ByList(const HcclAmdGradTensor *tensors, uint32_t n, F f)
{
    const auto byParts = [&](auto room) {
        return PartsOf(tensors, n) == kShort ? f(room, std::integral_constant<int, kShort>{}) : f(room, std::integral_constant<int, kLong>{});
    };
    return n <= kFew ? byParts(std::integral_constant<int, kFew>{}) : byParts(std::integral_constant<int, kMany>{});
}

}  // namespace
}  // namespace experts
}  // namespace hcclamd

using namespace hcclamd::experts;

extern "C" {

HcclResult HcclAmdGradSquaresWorkspace(const HcclAmdGradTensor *tensors, uint32_t n, uint64_t *bytes)
{
    EXPERTS_CHK_PTR(bytes);
    if (n != 0) {
        EXPERTS_CHK_PTR(tensors);
    }
    const HcclResult r = Check(__func__, tensors, n, false);
    if (r != HCCL_SUCCESS) {
        return r;
    }
    uint64_t slots = 0;
    const int parts = PartsOf(tensors, n);
    Table<kMany> table;
    for (uint32_t at = 0; Next(tensors, n, parts, at, table);) {
        slots += uint64_t(Slots(table.chunks));
    }
    *bytes = slots * sizeof(double);
    return HCCL_SUCCESS;
}

HcclResult HcclAmdGradSquares(const HcclAmdGradTensor *tensors, uint32_t n, uint32_t accumulate, double *squares, void *workspace,
    uint64_t workspaceBytes, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_PTR(squares);
    EXPERTS_CHK(Aligned(squares, 8));
    uint64_t needed = 0;
    const HcclResult checked = HcclAmdGradSquaresWorkspace(tensors, n, &needed);
    if (checked != HCCL_SUCCESS) {
        return checked;
    }
    if (needed != 0) {
        EXPERTS_CHK_PTR(workspace);
        EXPERTS_CHK(Aligned(workspace, 16));
        EXPERTS_CHK(workspaceBytes >= needed);
    }
    const hipStream_t on = static_cast<hipStream_t>(stream);
    double *slots = static_cast<double *>(workspace);
    int used = 0;
    const HcclResult r = ByList(tensors, n, [&](auto room, auto parts) {
        return Squares<decltype(room)::value, decltype(parts)::value>(tensors, n, slots, &used, on);
    });
    if (r != HCCL_SUCCESS) {
        return r;
    }
    return Launch("HcclAmdGradSquares", AddSlotsKernel, 1, 1024, 0, on, static_cast<const double *>(slots), used, squares, accumulate != 0);
}

HcclResult HcclAmdGradClip(const HcclAmdGradTensor *tensors, uint32_t n, const double *squares, float maxNorm, float *norm, void *stream)
{
    EXPERTS_CHK_PTR(stream);
    EXPERTS_CHK_PTR(squares);
    EXPERTS_CHK(Aligned(squares, 8) && Aligned(norm, 4));
    EXPERTS_CHK(maxNorm >= 0.0f);
    if (n != 0) {
        EXPERTS_CHK_PTR(tensors);
    }
    const HcclResult checked = Check(__func__, tensors, n, true);
    if (checked != HCCL_SUCCESS) {
        return checked;
    }
    const hipStream_t on = static_cast<hipStream_t>(stream);
    return ByList(tensors, n, [&](auto room, auto parts) {
        return Clip<decltype(room)::value, decltype(parts)::value>(tensors, n, squares, maxNorm, norm, on);
    });
}

}  // extern "C"
