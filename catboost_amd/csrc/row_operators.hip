// Operators on routed rows: slots sorted by expert, rows dispatched to their places and combined from them, gradients.
#include "operator_common.hip.h"

#include <algorithm>
#include <type_traits>

namespace cbamd {
namespace op {

// ---------------------------------------------------------------- slots sorted by expert ----

constexpr int32_t kMaxExperts = 1024;
constexpr uint32_t kSortWaves = 16;
constexpr uint32_t kSortThreads = kSortWaves * 64;

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

// A wave's slots, STEPS times 64 in a row, ranked: how many slots of the same step and expert come before each, and whether
// it is the last one of them. `own` counts the wave's slots of each expert; one lane adds for all that are alike, which needs
// no atomics (those of many lanes on few addresses take turns).
template <int STEPS>
struct TRankedSlots {
    uint32_t Expert[STEPS];
    uint32_t Rank[STEPS];  // bit 31: the last one

    __device__ __forceinline__ TRankedSlots(const int32_t* ids, uint32_t begin, uint32_t slots, uint32_t experts, uint32_t bits, int32_t* own) {
        const uint32_t lane = threadIdx.x & 63;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint32_t slot = begin + s * 64 + lane;
            const uint32_t e = slot < slots ? static_cast<uint32_t>(ids[slot]) : ~0u;
            Expert[s] = e < experts ? e : experts;
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint64_t same = LanesWithSame(Expert[s], bits);
            const bool last = (same >> lane >> 1) == 0;
            Rank[s] = static_cast<uint32_t>(__popcll(same & ((uint64_t(1) << lane) - 1))) | (last ? 0x80000000u : 0u);
            if (last && Expert[s] < experts) {
                own[Expert[s]] += static_cast<int32_t>(Rank[s] & 0x7fffffffu) + 1;
            }
            WaveHandover();  // the steps' additions stay in order
        }
    }
};

// counts[b * experts + e] (or [e * blocks + b] for the scan): how many slots of workgroup b go to expert e
template <int STEPS>
__global__ void __launch_bounds__(kSortThreads) CountExpertsKernel(const int32_t* ids, uint32_t slots, uint32_t experts, uint32_t bits, bool forScan,
                                                                   int32_t* counts) {
    extern __shared__ int32_t own[];  // [wave][expert]
    for (uint32_t i = threadIdx.x; i < kSortWaves * experts; i += kSortThreads) {
        own[i] = 0;
    }
    __syncthreads();
    const uint32_t wave = threadIdx.x / 64;
    const TRankedSlots<STEPS> ranked(ids, (blockIdx.x * kSortWaves + wave) * STEPS * 64, slots, experts, bits, own + wave * experts);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads) {
        int32_t sum = 0;
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            sum += own[w * experts + e];
        }
        counts[forScan ? size_t(e) * gridDim.x + blockIdx.x : size_t(blockIdx.x) * experts + e] = sum;
    }
}

// The sum of the workgroup's values before a thread's own
template <uint32_t WAVES>
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
    for (uint32_t w = 0; w < WAVES; ++w) {
        before += w < wave ? waveSums[w] : 0;
    }
    return before;
}

// A workgroup for an expert: its counts become the sums of the workgroups before each; totals[expert] their sum
__global__ void __launch_bounds__(256) ScanBlocksKernel(int32_t* counts, uint32_t blocks, int32_t* totals) {
    __shared__ int32_t waveSums[4];
    __shared__ int32_t carried;
    int32_t* mine = counts + size_t(blockIdx.x) * blocks;
    int32_t carry = 0;
    for (uint32_t begin = 0; begin < blocks; begin += 256) {
        const uint32_t b = begin + threadIdx.x;
        const int32_t x = b < blocks ? mine[b] : 0;
        const int32_t before = SumBefore<4>(x, waveSums) + carry;
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

// Places of a workgroup's slots: where the expert begins, what the workgroups before this one and the waves before the
// slot's have, what the wave's steps before it have, its rank. A single workgroup counts for itself. Of few workgroups each
// adds up all their counts (`totals` null), which takes less than a launch that does so; of many they come scanned. Launches and
// the steps' order bound the sort, not its bytes: 65536 slots of 64 experts take 10 us in two launches, a million 14 in three.
template <int STEPS>
__global__ void __launch_bounds__(kSortThreads) PlaceSlotsKernel(const int32_t* ids, uint32_t slots, uint32_t experts, uint32_t bits,
                                                                 const int32_t* counts, const int32_t* totals, int32_t* places, int32_t* offsets) {
    extern __shared__ int32_t lds[];
    __shared__ int32_t waveSums[kSortWaves];
    int32_t* next = lds;                              // [wave][expert]
    int32_t* sums = lds + kSortWaves * experts;       // the counts of all workgroups
    int32_t* sumsBefore = sums + experts;             // and of those before this one
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    for (uint32_t i = threadIdx.x; i < (kSortWaves + 2) * experts; i += kSortThreads) {
        lds[i] = 0;
    }
    __syncthreads();
    int32_t* own = next + wave * experts;
    const uint32_t begin = (blockIdx.x * kSortWaves + wave) * STEPS * 64;
    const TRankedSlots<STEPS> ranked(ids, begin, slots, experts, bits, own);
    if (gridDim.x > 1 && totals == nullptr) {
        for (uint32_t i = threadIdx.x; i < gridDim.x * experts; i += kSortThreads) {
            const uint32_t b = i / experts;
            const int32_t n = counts[i];
            atomicAdd(&sums[i - b * experts], n);
            if (b < blockIdx.x) {
                atomicAdd(&sumsBefore[i - b * experts], n);
            }
        }
    }
    __syncthreads();
    const uint32_t e = threadIdx.x;  // at most as many experts as threads
    int32_t total = 0, before = 0;
    if (e < experts) {
        if (gridDim.x == 1) {
            for (uint32_t w = 0; w < kSortWaves; ++w) {
                total += next[w * experts + e];
            }
        } else {
            total = totals != nullptr ? totals[e] : sums[e];
            before = totals != nullptr ? counts[size_t(e) * gridDim.x + blockIdx.x] : sumsBefore[e];
        }
    }
    const int32_t start = SumBefore<kSortWaves>(total, waveSums);
    if (e < experts) {
        int32_t at = start + before;
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            const int32_t n = next[w * experts + e];
            next[w * experts + e] = at;
            at += n;
        }
        if (blockIdx.x == 0) {
            offsets[e] = start;
            if (e == experts - 1) {
                offsets[experts] = start + total;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const bool valid = ranked.Expert[s] < experts;
        const int32_t place = valid ? own[ranked.Expert[s]] + static_cast<int32_t>(ranked.Rank[s] & 0x7fffffffu) : -1;
        WaveHandover();  // all lanes have read before the last one of each expert writes
        if (valid && (ranked.Rank[s] & 0x80000000u) != 0) {
            own[ranked.Expert[s]] = place + 1;
        }
        WaveHandover();
        const uint32_t slot = begin + s * 64 + lane;
        if (slot < slots) {
            places[slot] = place;
        }
    }
}

// ---------------------------------------------------------------- rows to their places and back ----

// Rows are cut into pieces of 16 bytes, one for a thread, in the order in which they are in memory. The last piece of a row
// ends with the row: it holds some values of the piece before it again, which then come from two threads, alike. (Loads and
// stores of what is left of a row instead took branches that every load waited in: 164 us for 16384 rows of 8 KB to four
// places each where whole pieces take 130.) Rows of less than 16 bytes have pieces of one value.
struct TPieces {
    size_t Rows, Width;   // values
    uint32_t PerRow;      // slots
    uint32_t Pieces;      // of a row
    uint64_t Inverse;     // floor(i / Pieces) = floor(i Inverse / 2^64) as long as i Pieces < 2^64, which memory sees to

    // of N values each
    template <int N>
    __device__ __forceinline__ bool Of(size_t* row, size_t* column) const {
        const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
        *row = Inverse != 0 ? __umul64hi(i, Inverse) : i;
        const size_t c = (i - *row * Pieces) * N;
        *column = N == 1 || c + N <= Width ? c : Width - N;
        return *row < Rows;
    }
};

// The next K places of a row from slot k on, -1 for those that are left out
template <int K>
struct TPlaces {
    int32_t At[K];
    __device__ __forceinline__ TPlaces(const int32_t* places, uint32_t k, uint32_t perRow, size_t sortedRows) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            At[j] = k + j < perRow ? places[k + j] : -1;
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
            At[j] = static_cast<size_t>(At[j]) < sortedRows ? At[j] : -1;  // (negative ones are large)
        }
    }
};

// A row's places are requested K at a time, so that the stores do not wait for one after the other. Memory bounds it: 16384 rows
// of 8 KB to four places each take 118 us (5.7 TB/s).
template <typename T, int N, int K>
__global__ void __launch_bounds__(256) DispatchRowsKernel(const T* source, size_t sourceStride, TPieces p, const int32_t* places, T* sorted,
                                                          size_t sortedRows, size_t sortedStride) {
    using TPiece = std::conditional_t<N == 1, TValues<T, 1>, TValues<uint32_t, 4>>;
    size_t row, c;
    if (!p.Of<N>(&row, &c)) {
        return;
    }
    const TPiece v = TPiece::Load(source + row * sourceStride + c);
    for (uint32_t k = 0; k < p.PerRow; k += K) {
        const TPlaces<K> to(places + row * p.PerRow, k, p.PerRow, sortedRows);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (to.At[j] >= 0) {
                v.Store(sorted + static_cast<size_t>(to.At[j]) * sortedStride + c);
            }
        }
    }
}

// Slots that are left out are read at the row's first place that is not, and add nothing: no load waits in a branch. Memory bounds
// it: 16384 rows of 8 KB from four places each take 134 us (5 TB/s).
template <typename T, int N, int K>
__global__ void __launch_bounds__(256) CombineRowsKernel(const T* sorted, size_t sortedRows, size_t sortedStride, TPieces p, const int32_t* places,
                                                         const TAcc<T>* weights, T* result, size_t resultStride) {
    using A = TAcc<T>;
    size_t row, c;
    if (!p.Of<N>(&row, &c)) {
        return;
    }
    A sum[N] = {};
    for (uint32_t k = 0; k < p.PerRow; k += K) {
        const TPlaces<K> from(places + row * p.PerRow, k, p.PerRow, sortedRows);
        int32_t any = -1;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            any = any >= 0 ? any : from.At[j];
        }
        if (any < 0) {
            continue;
        }
        A w[K];
        TValues<T, N> v[K];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            w[j] = weights != nullptr && from.At[j] >= 0 ? weights[row * p.PerRow + k + j] : A(1);
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
            v[j] = TValues<T, N>::Load(sorted + static_cast<size_t>(from.At[j] >= 0 ? from.At[j] : any) * sortedStride + c);
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const A term = w[j] * static_cast<A>(v[j].V[i]);
                sum[i] += from.At[j] >= 0 ? term : A(0);
            }
        }
    }
    TValues<T, N> out;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        out.V[i] = static_cast<T>(sum[i]);
    }
    out.Store(result + row * resultStride + c);
}

// L threads for a row. A thread takes every L-th piece of the row's gradient and, for K slots at a time, what is at their
// places; its products are added in that order, then the threads' sums by a butterfly: the same order for every call. Both gradients
// come from one reading of the row's. Memory bounds it: both of 16384 rows of 8 KB with four places each take 222 us (5.4 TB/s).
template <typename T, int N, int L, int K>
__global__ void __launch_bounds__(256) CombineRowsBackwardKernel(const T* gradients, size_t gradientStride, const T* sorted, size_t sortedRows,
                                                                 size_t sortedStride, size_t rows, size_t width, uint32_t perRow,
                                                                 const int32_t* places, const TAcc<T>* weights, T* sortedGradients,
                                                                 size_t sortedGradientStride, TAcc<T>* weightGradients) {
    using A = TAcc<T>;
    __shared__ A waveSums[4][K];
    const uint32_t lane = threadIdx.x % L;
    const size_t row = size_t(blockIdx.x) * (256 / L) + threadIdx.x / L;
    const bool there = row < rows;  // (false for whole groups of L threads)
    for (uint32_t k = 0; k < perRow; k += K) {
        A product[K] = {};
        if (there) {
            const TPlaces<K> at(places + row * perRow, k, perRow, sortedRows);
            int32_t any = -1;
            A w[K];
#pragma unroll
            for (int j = 0; j < K; ++j) {
                any = any >= 0 ? any : at.At[j];
                w[j] = weights != nullptr && at.At[j] >= 0 ? weights[row * perRow + k + j] : A(1);
            }
            for (size_t begin = size_t(lane) * N; any >= 0 && begin < width; begin += L * N) {
                const size_t c = N == 1 || begin + N <= width ? begin : width - N;
                TValues<T, N> g = TValues<T, N>::Load(gradients + row * gradientStride + c);
                TValues<T, N> v[K];
                if (weightGradients != nullptr) {
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        v[j] = TValues<T, N>::Load(sorted + static_cast<size_t>(at.At[j] >= 0 ? at.At[j] : any) * sortedStride + c);
                    }
                }
                if (sortedGradients != nullptr) {
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        if (at.At[j] >= 0) {
                            TValues<T, N> out;
#pragma unroll
                            for (int i = 0; i < N; ++i) {
                                out.V[i] = static_cast<T>(w[j] * static_cast<A>(g.V[i]));
                            }
                            out.Store(sortedGradients + static_cast<size_t>(at.At[j]) * sortedGradientStride + c);
                        }
                    }
                }
                if (weightGradients != nullptr) {
                    // (of a row's last piece, only what the piece before it does not have)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const A gi = c + i >= begin ? static_cast<A>(g.V[i]) : A(0);
#pragma unroll
                        for (int j = 0; j < K; ++j) {
                            const A term = gi * static_cast<A>(v[j].V[i]);
                            product[j] += c + i >= begin && at.At[j] >= 0 ? term : A(0);
                        }
                    }
                }
            }
        }
        if (weightGradients == nullptr) {
            continue;
        }
#pragma unroll
        for (int j = 0; j < K; ++j) {
            for (int step = (L < 64 ? L : 64) / 2; step > 0; step /= 2) {
                product[j] += __shfl_xor(product[j], step);
            }
        }
        if constexpr (L > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    waveSums[threadIdx.x / 64][j] = product[j];
                }
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < K; ++j) {
                product[j] = (waveSums[0][j] + waveSums[1][j]) + (waveSums[2][j] + waveSums[3][j]);
            }
        }
        if (there && lane == 0) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                if (k + j < perRow) {
                    weightGradients[row * perRow + k + j] = product[j];
                }
            }
        }
    }
}

}  // namespace op

using namespace op;

namespace {

constexpr uint32_t kStepsOfMany = 4;  // when there are several workgroups
// that one workgroup sorts (8192 of 64 experts: 8.4 us, 9.7 in two launches of several workgroups, which also cost the host one more)
constexpr size_t kSlotsOfOne = 8 * kSortThreads;
constexpr size_t kSlotsOfBlock = size_t(kStepsOfMany) * kSortThreads;
// by each workgroup, eight for a thread (131072 slots of 256 experts, as many counts: 13.6 us, 14.1 with a launch that scans them; 65536 of
// 1024, twice as many: 18.5 and 17.1)
constexpr size_t kCountsToAdd = 8192;

size_t SortBlocks(size_t slots) {
    return slots <= kSlotsOfOne ? 1 : (slots + kSlotsOfBlock - 1) / kSlotsOfBlock;
}

}  // namespace

size_t SortByExpertBytes(size_t slots, int32_t experts) {
    if (experts <= 0 || experts > kMaxExperts || slots > 0x7fffffffu) {
        return 0;
    }
    return (SortBlocks(slots) + 1) * static_cast<size_t>(experts) * 4;
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
    const size_t blocks = SortBlocks(slots);
    int32_t* totals = static_cast<int32_t*>(workspace);
    int32_t* counts = totals + experts;
    const uint32_t e = static_cast<uint32_t>(experts), n = static_cast<uint32_t>(slots);
    uint32_t bits = 1;
    while (e >> bits != 0) {
        ++bits;
    }
    const auto place = [&](auto kernel, const int32_t* scannedTotals) {
        const size_t lds = (kSortWaves + 2) * static_cast<size_t>(e) * 4;
        call.AllowLds(reinterpret_cast<const void*>(kernel), lds);
        call.Launch(kernel, blocks, kSortThreads, lds, ids, n, e, bits, static_cast<const int32_t*>(counts), scannedTotals, places, offsets);
    };
    if (blocks == 1) {
        return slots <= kSortThreads ? place(PlaceSlotsKernel<1>, nullptr) : slots <= 4 * kSortThreads ? place(PlaceSlotsKernel<4>, nullptr)
            : place(PlaceSlotsKernel<8>, nullptr);
    }
    const bool scan = blocks * e > kCountsToAdd;
    call.Launch(CountExpertsKernel<kStepsOfMany>, blocks, kSortThreads, kSortWaves * static_cast<size_t>(e) * 4, ids, n, e, bits, scan, counts);
    if (scan) {
        call.Launch(ScanBlocksKernel, e, 256, 0, counts, static_cast<uint32_t>(blocks), totals);
    }
    place(PlaceSlotsKernel<kStepsOfMany>, scan ? totals : nullptr);
}

namespace {

constexpr int32_t kMaxPerRow = 64;
constexpr size_t kRowsOfWaves = 4096, kRowsOfLanes = 16384;
constexpr size_t kMaxGroups = size_t(1) << 23;  // of 256 threads in a launch

void CheckRoutes(size_t rows, size_t width, int32_t perRow, const int32_t* places, size_t sortedRows) {
    CBAMD_ENSURE(perRow >= 1 && perRow <= kMaxPerRow, "slots per row: " + std::to_string(perRow) + ", 1 to " + std::to_string(kMaxPerRow) + " are supported");
    CBAMD_ENSURE(places != nullptr, "places pointer is null");
    CBAMD_ENSURE(width < size_t(1) << 31, "rows are too wide: " + std::to_string(width));
    CBAMD_ENSURE(rows <= size_t(1) << 40, "too many rows");
    CBAMD_ENSURE(sortedRows <= 0x7fffffffu, "too many sorted rows: " + std::to_string(sortedRows));
}

TPieces PiecesOf(size_t rows, size_t width, int32_t perRow, size_t valueSize) {
    TPieces p{};
    p.Rows = rows;
    p.Width = width;
    p.PerRow = static_cast<uint32_t>(perRow);
    p.Pieces = static_cast<uint32_t>(width * valueSize < 16 ? width : (width * valueSize + 15) / 16);
    p.Inverse = p.Pieces > 1 ? ~uint64_t(0) / p.Pieces + 1 : 0;
    return p;
}

// f(first row, rows, workgroups) for rows that one launch takes (a workgroup has one part of them: a loop would keep the
// arguments in registers all along)
template <typename F>
void ForLaunches(size_t rows, size_t threadsPerRow, F&& f) {
    const size_t most = std::max<size_t>(1, kMaxGroups * 256 / threadsPerRow);
    for (size_t first = 0; first < rows; first += most) {
        const size_t n = std::min(rows - first, most);
        f(first, n, (n * threadsPerRow + 255) / 256);
    }
}

// f(values of a piece, slots that are taken at a time)
template <typename T, typename F>
void WithShape(size_t width, int32_t perRow, F&& f) {
    using std::integral_constant;
    constexpr int N = 16 / sizeof(T);
    const auto slots = [&](auto values) {
        return perRow == 1 ? f(values, integral_constant<int, 1>()) : perRow == 2 ? f(values, integral_constant<int, 2>())
            : perRow <= 4 ? f(values, integral_constant<int, 4>()) : f(values, integral_constant<int, 8>());
    };
    return width >= N ? slots(integral_constant<int, N>()) : slots(integral_constant<int, 1>());
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
    // LDS that no one uses keeps a compute unit to four workgroups, six where a row is stored to one or two places: fewer
    // stores on their way at a time are faster once they go to memory (16384 rows of 8 KB to four places 114 us, 117 with six and 139
    // with the eight that there is room for; 300000 rows of 800 bytes to one 93.3, 94.0 with four, 94.5 with eight), and make little
    // difference where the caches hold them (4096 rows of 8 KB to four places 32.6 and 33.9 with eight, 1024 rows 8.0 and 7.7; 65536
    // rows of 512 bytes to one 11.8, 12.8 with four, 11.6 with eight)
    const size_t unusedLds = (160 * 1024) / (perRow <= 2 ? 6 : 4) / 1024 * 1024;
    const auto launch = [&](auto value) {
        using T = decltype(value);
        WithShape<T>(width, perRow, [&](auto values, auto slots) {
            ForLaunches(rows, PiecesOf(rows, width, perRow, size).Pieces, [&](size_t first, size_t n, size_t groups) {
                call.Launch(DispatchRowsKernel<T, decltype(values)::value, decltype(slots)::value>, groups, 256, unusedLds,
                            static_cast<const T*>(source) + first * sourceStride, sourceStride, PiecesOf(n, width, perRow, size),
                            places + first * perRow, static_cast<T*>(sorted), sortedRows, sortedStride);
            });
        });
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
        WithShape<T>(width, perRow, [&](auto values, auto slots) {
            ForLaunches(rows, PiecesOf(rows, width, perRow, size).Pieces, [&](size_t first, size_t n, size_t groups) {
                call.Launch(CombineRowsKernel<T, decltype(values)::value, decltype(slots)::value>, groups, 256, 0, static_cast<const T*>(sorted),
                            sortedRows, sortedStride, PiecesOf(n, width, perRow, size), places + first * perRow,
                            weights != nullptr ? static_cast<const TAcc<T>*>(weights) + first * perRow : nullptr,
                            static_cast<T*>(result) + first * resultStride, resultStride);
            });
        });
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
        const size_t pieces = (width * size + 15) / 16;
        WithShape<T>(width, perRow, [&](auto values, auto slots) {
            constexpr int N = decltype(values)::value, K = decltype(slots)::value;
            const auto launch = [&](auto kernel, size_t threadsPerRow) {
                ForLaunches(rows, threadsPerRow, [&](size_t first, size_t n, size_t groups) {
                    call.Launch(kernel, groups, 256, 0, static_cast<const T*>(resultGradients) + first * gradientStride, gradientStride,
                                static_cast<const T*>(sorted), sortedRows, sortedStride, n, width, static_cast<uint32_t>(perRow),
                                places + first * perRow, weights != nullptr ? static_cast<const TAcc<T>*>(weights) + first * perRow : nullptr,
                                static_cast<T*>(sortedGradients), sortedGradientStride,
                                weightGradients != nullptr ? static_cast<TAcc<T>*>(weightGradients) + first * perRow : nullptr);
                });
            };
            // eight threads for a row with two pieces each at most or, where the rows alone fill the chip, four (two slots of 32-bit values: 65536
            // rows of 512 bytes 29 us, 32 with a wave for each; 4096 rows 5.8 and 5.1); a wave up to one piece for a thread or, of more rows,
            // under four (4096 rows of 2 KB 8.8 us, 10.6 with four waves for each; 512 rows 5.0 and 4.7; 65536 rows of 4 KB 276 and 267)
            if (pieces <= 16 || (pieces <= 32 && rows >= kRowsOfLanes)) {
                launch(CombineRowsBackwardKernel<T, N, 8, K>, 8);
            } else if (pieces <= 64 || (pieces < 256 && rows >= kRowsOfWaves)) {
                launch(CombineRowsBackwardKernel<T, N, 64, K>, 64);
            } else {
                launch(CombineRowsBackwardKernel<T, N, 256, K>, 256);
            }
        });
    });
}

}  // namespace cbamd
