// Operators on routed rows: slots sorted by expert, rows dispatched to their places and combined from them, gradients.
#include "operator_common.hip.h"

#include <algorithm>

namespace cbamd {
namespace op {

// ---------------------------------------------------------------- slots sorted by expert ----

constexpr int32_t kMaxExperts = 1024;
constexpr uint32_t kSortWaves = 4;
constexpr uint32_t kSortSteps = 16;                             // of 64 slots that a wave ranks
constexpr uint32_t kSortSlots = kSortWaves * kSortSteps * 64;   // of a workgroup

// counts[expert][block]: how many of the block's slots go to the expert
__global__ void __launch_bounds__(256) CountExpertsKernel(const int32_t* ids, uint32_t slots, uint32_t experts, uint32_t blocks, int32_t* counts) {
    __shared__ int32_t count[kMaxExperts];
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
        count[e] = 0;
    }
    __syncthreads();
    const uint32_t begin = blockIdx.x * kSortSlots;
    const uint32_t n = min(kSortSlots, slots - begin);
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint32_t e = static_cast<uint32_t>(ids[begin + i]);
        if (e < experts) {
            atomicAdd(&count[e], 1);
        }
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
        counts[size_t(e) * blocks + blockIdx.x] = count[e];
    }
}

// The sum of the workgroup's values before a thread's own (256 threads)
__device__ __forceinline__ int32_t SumBefore(int32_t x, int32_t* waveSums) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    int32_t sum = x;
    for (int step = 1; step < 64; step *= 2) {
        const int32_t other = __shfl_up(sum, step);
        sum += lane >= static_cast<uint32_t>(step) ? other : 0;
    }
    __syncthreads();
    if (lane == 63) {
        waveSums[wave] = sum;
    }
    __syncthreads();
    int32_t before = sum - x;
    for (uint32_t w = 0; w < wave; ++w) {
        before += waveSums[w];
    }
    return before;
}

// A workgroup for an expert: its counts become the sums of the blocks before each; totals[expert] their sum
__global__ void __launch_bounds__(256) ScanBlocksKernel(int32_t* counts, uint32_t blocks, int32_t* totals) {
    __shared__ int32_t waveSums[4];
    __shared__ int32_t carried;
    int32_t* mine = counts + size_t(blockIdx.x) * blocks;
    int32_t carry = 0;
    for (uint32_t begin = 0; begin < blocks; begin += 256) {
        const uint32_t b = begin + threadIdx.x;
        const int32_t x = b < blocks ? mine[b] : 0;
        const int32_t before = SumBefore(x, waveSums) + carry;
        if (b < blocks) {
            mine[b] = before;
        }
        if (threadIdx.x == 255) {
            carried = before + x;
        }
        __syncthreads();
        carry = carried;
    }
    if (threadIdx.x == 0) {
        totals[blockIdx.x] = carry;
    }
}

// Lanes of a wave whose value is the caller's own, out of values of `bits` bits; every lane takes part
__device__ __forceinline__ uint64_t LanesWithSame(uint32_t value, uint32_t bits) {
    uint64_t same = ~uint64_t(0);
    for (uint32_t b = 0; b < bits; ++b) {
        const bool set = value >> b & 1;
        const uint64_t with = __ballot(set);
        same &= set ? with : ~with;
    }
    return same;
}

// Places of a block's slots. A wave ranks its slots step by step: a slot's rank among the step's equal ids comes from
// ballots, what comes before the step from the wave's own counters, which begin with what comes before the wave
__global__ void __launch_bounds__(256) PlaceSlotsKernel(const int32_t* ids, uint32_t slots, uint32_t experts, uint32_t bits, uint32_t blocks,
                                                        const int32_t* counts, const int32_t* totals, int32_t* places, int32_t* offsets) {
    __shared__ int32_t next[kSortWaves][kMaxExperts];
    __shared__ int32_t waveSums[4];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    for (uint32_t e = threadIdx.x; e < experts; e += blockDim.x) {
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            next[w][e] = 0;
        }
    }
    __syncthreads();
    const uint32_t begin = blockIdx.x * kSortSlots + wave * kSortSteps * 64;
    for (uint32_t step = 0; step < kSortSteps; ++step) {
        const uint32_t slot = begin + step * 64 + lane;
        const uint32_t e = slot < slots ? static_cast<uint32_t>(ids[slot]) : ~0u;
        if (e < experts) {
            atomicAdd(&next[wave][e], 1);
        }
    }
    // four experts a thread: where each begins, what the blocks before this one and the waves before each have
    int32_t total[kMaxExperts / 256], sum = 0;
    for (uint32_t i = 0; i < kMaxExperts / 256; ++i) {
        const uint32_t e = threadIdx.x * (kMaxExperts / 256) + i;
        total[i] = e < experts ? totals[e] : 0;
        sum += total[i];
    }
    int32_t start = SumBefore(sum, waveSums);  // (its barriers stand behind the counting above)
    for (uint32_t i = 0; i < kMaxExperts / 256; ++i) {
        const uint32_t e = threadIdx.x * (kMaxExperts / 256) + i;
        if (e < experts) {
            int32_t at = start + counts[size_t(e) * blocks + blockIdx.x];
            for (uint32_t w = 0; w < kSortWaves; ++w) {
                const int32_t n = next[w][e];
                next[w][e] = at;
                at += n;
            }
            if (blockIdx.x == 0) {
                offsets[e] = start;
                if (e == experts - 1) {
                    offsets[experts] = start + total[i];
                }
            }
        }
        start += total[i];
    }
    __syncthreads();
    for (uint32_t step = 0; step < kSortSteps; ++step) {
        const uint32_t slot = begin + step * 64 + lane;
        const uint32_t e = slot < slots ? static_cast<uint32_t>(ids[slot]) : ~0u;
        const bool valid = e < experts;
        const uint64_t same = LanesWithSame(valid ? e : experts, bits);
        const uint32_t rank = __popcll(same & ((uint64_t(1) << lane) - 1));
        const int32_t at = valid ? next[wave][e] : 0;
        __builtin_amdgcn_wave_barrier();  // all lanes have read before the last one of each id writes
        if (valid && (same >> lane >> 1) == 0) {
            next[wave][e] = at + static_cast<int32_t>(rank) + 1;
        }
        __builtin_amdgcn_wave_barrier();
        if (slot < slots) {
            places[slot] = valid ? at + static_cast<int32_t>(rank) : -1;
        }
    }
}

// ---------------------------------------------------------------- rows to their places ----

// Where in a matrix of rows cut into `pieces` pieces each a thread's piece is: workgroups are 256 pieces long and may
// begin inside a row
struct TPiece {
    size_t Row;
    uint32_t Piece;
};

__device__ __forceinline__ TPiece PieceOf(size_t block, uint32_t pieces) {
    const size_t first = block * 256;
    const size_t row = first / pieces;
    const uint32_t at = static_cast<uint32_t>(first - row * pieces) + threadIdx.x;
    const uint32_t rows = at / pieces;
    return {row + rows, at - rows * pieces};
}

// A piece of a row of E is N values, the last one of a row may be shorter
template <typename T, int N>
__global__ void __launch_bounds__(256) DispatchRowsKernel(const T* source, size_t sourceStride, size_t rows, size_t width, uint32_t pieces,
                                                          uint32_t perRow, const int32_t* places, T* sorted, size_t sortedRows,
                                                          size_t sortedStride, size_t blocks) {
    for (size_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const TPiece p = PieceOf(block, pieces);
        if (p.Row >= rows) {
            return;
        }
        const size_t c = size_t(p.Piece) * N;
        const T* from = source + p.Row * sourceStride + c;
        const bool whole = c + N <= width;
        TValues<T, N> v{};
        if (whole) {
            v = TValues<T, N>::Load(from);
        } else {
            for (int i = 0; i < N; ++i) {
                if (c + i < width) {
                    v.V[i] = from[i];
                }
            }
        }
        for (uint32_t k = 0; k < perRow; ++k) {
            const int32_t place = places[p.Row * perRow + k];
            if (place < 0 || static_cast<size_t>(place) >= sortedRows) {
                continue;
            }
            T* to = sorted + static_cast<size_t>(place) * sortedStride + c;
            if (whole) {
                v.Store(to);
            } else {
                for (int i = 0; i < N; ++i) {
                    if (c + i < width) {
                        to[i] = v.V[i];
                    }
                }
            }
        }
    }
}

// ---------------------------------------------------------------- rows from their places ----

template <typename T, int N>
__global__ void __launch_bounds__(256) CombineRowsKernel(const T* sorted, size_t sortedRows, size_t sortedStride, size_t rows, size_t width,
                                                         uint32_t pieces, uint32_t perRow, const int32_t* places, const TAcc<T>* weights,
                                                         T* result, size_t resultStride, size_t blocks) {
    using A = TAcc<T>;
    for (size_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const TPiece p = PieceOf(block, pieces);
        if (p.Row >= rows) {
            return;
        }
        const size_t c = size_t(p.Piece) * N;
        const bool whole = c + N <= width;
        A sum[N] = {};
        for (uint32_t k = 0; k < perRow; ++k) {
            const int32_t place = places[p.Row * perRow + k];
            if (place < 0 || static_cast<size_t>(place) >= sortedRows) {
                continue;
            }
            const A w = weights != nullptr ? weights[p.Row * perRow + k] : A(1);
            const T* from = sorted + static_cast<size_t>(place) * sortedStride + c;
            if (whole) {
                const TValues<T, N> v = TValues<T, N>::Load(from);
                for (int i = 0; i < N; ++i) {
                    sum[i] += w * static_cast<A>(v.V[i]);
                }
            } else {
                for (int i = 0; i < N; ++i) {
                    if (c + i < width) {
                        sum[i] += w * static_cast<A>(from[i]);
                    }
                }
            }
        }
        T* to = result + p.Row * resultStride + c;
        TValues<T, N> v;
        for (int i = 0; i < N; ++i) {
            v.V[i] = static_cast<T>(sum[i]);
        }
        if (whole) {
            v.Store(to);
        } else {
            for (int i = 0; i < N; ++i) {
                if (c + i < width) {
                    to[i] = v.V[i];
                }
            }
        }
    }
}

// A wave for a row. Each lane adds the products of its own columns in their order, the lanes' sums are added by a
// butterfly: the same order for every call
template <typename T, int N>
__global__ void __launch_bounds__(256) CombineRowsBackwardKernel(const T* gradients, size_t gradientStride, const T* sorted, size_t sortedRows,
                                                                 size_t sortedStride, size_t rows, size_t width, uint32_t perRow,
                                                                 const int32_t* places, const TAcc<T>* weights, T* sortedGradients,
                                                                 size_t sortedGradientStride, TAcc<T>* weightGradients) {
    using A = TAcc<T>;
    const uint32_t lane = threadIdx.x & 63;
    for (size_t row = size_t(blockIdx.x) * 4 + threadIdx.x / 64; row < rows; row += size_t(gridDim.x) * 4) {
        const T* from = gradients + row * gradientStride;
        for (uint32_t k = 0; k < perRow; ++k) {
            const size_t slot = row * perRow + k;
            const int32_t place = places[slot];
            const bool there = place >= 0 && static_cast<size_t>(place) < sortedRows;
            A product = 0;
            if (there) {
                const A w = weights != nullptr ? weights[slot] : A(1);
                const T* y = sorted + static_cast<size_t>(place) * sortedStride;
                T* to = sortedGradients + static_cast<size_t>(place) * sortedGradientStride;
                for (size_t c = size_t(lane) * N; c < width; c += 64 * N) {
                    if (c + N <= width) {
                        const TValues<T, N> g = TValues<T, N>::Load(from + c);
                        if (weightGradients != nullptr) {
                            const TValues<T, N> v = TValues<T, N>::Load(y + c);
                            for (int i = 0; i < N; ++i) {
                                product += static_cast<A>(g.V[i]) * static_cast<A>(v.V[i]);
                            }
                        }
                        if (sortedGradients != nullptr) {
                            TValues<T, N> v;
                            for (int i = 0; i < N; ++i) {
                                v.V[i] = static_cast<T>(w * static_cast<A>(g.V[i]));
                            }
                            v.Store(to + c);
                        }
                    } else {
                        for (size_t i = c; i < width; ++i) {
                            if (weightGradients != nullptr) {
                                product += static_cast<A>(from[i]) * static_cast<A>(y[i]);
                            }
                            if (sortedGradients != nullptr) {
                                to[i] = static_cast<T>(w * static_cast<A>(from[i]));
                            }
                        }
                    }
                }
            }
            if (weightGradients != nullptr) {
                for (int step = 32; step > 0; step /= 2) {
                    product += __shfl_xor(product, step);
                }
                if (lane == 0) {
                    weightGradients[slot] = product;
                }
            }
        }
    }
}

}  // namespace op

using namespace op;

namespace {

uint32_t SortBlocks(size_t slots) {
    return static_cast<uint32_t>((slots + kSortSlots - 1) / kSortSlots);
}

}  // namespace

size_t SortByExpertBytes(size_t slots, int32_t experts) {
    if (experts <= 0 || experts > kMaxExperts || slots > 0x7fffffffu) {
        return 0;
    }
    return (size_t(std::max<uint32_t>(1, SortBlocks(slots))) + 1) * static_cast<size_t>(experts) * 4;
}

void SortByExpert(size_t slots, int32_t experts, const int32_t* ids, int32_t* places, int32_t* offsets, void* workspace,
                  size_t workspaceBytes, void* stream) {
    CBAMD_ENSURE(experts >= 1 && experts <= kMaxExperts, "experts: " + std::to_string(experts) + ", 1 to " + std::to_string(kMaxExperts) + " are supported");
    CBAMD_ENSURE(slots <= 0x7fffffffu, "too many slots to sort: " + std::to_string(slots));
    CBAMD_ENSURE((ids != nullptr && places != nullptr) || slots == 0, "ids or places pointer is null");
    CBAMD_ENSURE(offsets != nullptr, "offsets pointer is null");
    const size_t needed = SortByExpertBytes(slots, experts);
    CBAMD_ENSURE(workspace != nullptr && workspaceBytes >= needed, "workspace of " + std::to_string(workspaceBytes) + " bytes, " + std::to_string(needed) + " are needed");
    CBAMD_ENSURE(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "workspace pointer is not a multiple of 4");
    const TCallDevice call(offsets, stream);
    const uint32_t blocks = std::max<uint32_t>(1, SortBlocks(slots));
    int32_t* totals = static_cast<int32_t*>(workspace);
    int32_t* counts = totals + experts;
    const uint32_t e = static_cast<uint32_t>(experts), n = static_cast<uint32_t>(slots);
    uint32_t bits = 1;
    while (e >> bits != 0) {
        ++bits;
    }
    call.Launch(CountExpertsKernel, blocks, 256, 0, ids, n, e, blocks, counts);
    call.Launch(ScanBlocksKernel, e, 256, 0, counts, blocks, totals);
    call.Launch(PlaceSlotsKernel, blocks, 256, 0, ids, n, e, bits, blocks, counts, totals, places, offsets);
}

namespace {

constexpr int32_t kMaxPerRow = 64;
constexpr size_t kMaxGroups = size_t(1) << 20;

void CheckRoutes(size_t rows, size_t width, int32_t perRow, const int32_t* places, size_t sortedRows) {
    CBAMD_ENSURE(perRow >= 1 && perRow <= kMaxPerRow, "slots per row: " + std::to_string(perRow) + ", 1 to " + std::to_string(kMaxPerRow) + " are supported");
    CBAMD_ENSURE(places != nullptr, "places pointer is null");
    CBAMD_ENSURE(width < size_t(1) << 31, "rows are too wide: " + std::to_string(width));
    CBAMD_ENSURE(rows <= size_t(1) << 40, "too many rows");
    CBAMD_ENSURE(sortedRows <= 0x7fffffffu, "too many sorted rows: " + std::to_string(sortedRows));
}

}  // namespace

void DispatchRows(int valueType, size_t rows, size_t width, int32_t perRow, const void* source, size_t sourceStride,
                  const int32_t* places, void* sorted, size_t sortedRows, size_t sortedStride, void* stream) {
    const size_t size = ValueSize(valueType);
    if (rows == 0 || width == 0 || sortedRows == 0) {
        return;
    }
    CheckRoutes(rows, width, perRow, places, sortedRows);
    CheckMatrix("source", source, rows, width, sourceStride, size);
    CheckMatrix("sorted rows", sorted, sortedRows, width, sortedStride, size);
    const TCallDevice call(sorted, stream);
    const auto launch = [&](auto value) {
        using T = decltype(value);
        constexpr int N = 16 / sizeof(T);
        const uint32_t pieces = static_cast<uint32_t>((width + N - 1) / N);
        const size_t blocks = (rows * pieces + 255) / 256;
        call.Launch(DispatchRowsKernel<T, N>, std::min(blocks, kMaxGroups), 256, 0, static_cast<const T*>(source), sourceStride, rows, width,
                    pieces, static_cast<uint32_t>(perRow), places, static_cast<T*>(sorted), sortedRows, sortedStride, blocks);
    };
    // the values' bits are moved as they are
    switch (size) {
        case 8: return launch(uint64_t());
        case 4: return launch(uint32_t());
        default: return launch(uint16_t());
    }
}

void CombineRows(int valueType, size_t rows, size_t width, int32_t perRow, const void* sorted, size_t sortedRows,
                 size_t sortedStride, const int32_t* places, const void* weights, void* result, size_t resultStride,
                 void* stream) {
    const size_t size = ValueSize(valueType);
    if (rows == 0 || width == 0) {
        return;
    }
    CheckRoutes(rows, width, perRow, places, sortedRows);
    if (sortedRows > 0) {
        CheckMatrix("sorted rows", sorted, sortedRows, width, sortedStride, size);
    }
    CheckMatrix("result", result, rows, width, resultStride, size);
    const TCallDevice call(result, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        constexpr int N = 16 / sizeof(T);
        const uint32_t pieces = static_cast<uint32_t>((width + N - 1) / N);
        const size_t blocks = (rows * pieces + 255) / 256;
        call.Launch(CombineRowsKernel<T, N>, std::min(blocks, kMaxGroups), 256, 0, static_cast<const T*>(sorted), sortedRows, sortedStride, rows,
                    width, pieces, static_cast<uint32_t>(perRow), places, static_cast<const TAcc<T>*>(weights), static_cast<T*>(result),
                    resultStride, blocks);
    });
}

void CombineRowsBackward(int valueType, size_t rows, size_t width, int32_t perRow, const void* resultGradients,
                         size_t gradientStride, const void* sorted, size_t sortedRows, size_t sortedStride,
                         const int32_t* places, const void* weights, void* sortedGradients,
                         size_t sortedGradientStride, void* weightGradients, void* stream) {
    const size_t size = ValueSize(valueType);
    if (rows == 0 || (sortedGradients == nullptr && weightGradients == nullptr)) {
        return;
    }
    CheckRoutes(rows, width, perRow, places, sortedRows);
    if (width > 0) {
        CheckMatrix("result gradients", resultGradients, rows, width, gradientStride, size);
    }
    if (weightGradients != nullptr && sortedRows > 0 && width > 0) {
        CheckMatrix("sorted rows", sorted, sortedRows, width, sortedStride, size);
    }
    if (sortedGradients != nullptr && sortedRows > 0 && width > 0) {
        CheckMatrix("sorted gradients", sortedGradients, sortedRows, width, sortedGradientStride, size);
    }
    const TCallDevice call(weightGradients != nullptr ? weightGradients : sortedGradients, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        constexpr int N = 16 / sizeof(T);
        call.Launch(CombineRowsBackwardKernel<T, N>, std::min((rows + 3) / 4, kMaxGroups), 256, 0, static_cast<const T*>(resultGradients),
                    gradientStride, static_cast<const T*>(sorted), sortedRows, sortedStride, rows, width, static_cast<uint32_t>(perRow), places,
                    static_cast<const TAcc<T>*>(weights), static_cast<T*>(sortedGradients), sortedGradientStride,
                    static_cast<TAcc<T>*>(weightGradients));
    });
}

}  // namespace cbamd
