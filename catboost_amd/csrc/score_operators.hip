// Operators on scores: penalties, biases and masks; the best classes of a row and their weights.
#include "operator_common.hip.h"

#include <algorithm>
#include <limits>
#include <type_traits>

namespace cbamd {
namespace op {

// ---------------------------------------------------------------- penalties, biases, masks ----

struct TAdjustArgs {
    const void* Scores;
    void* Result;
    size_t ScoreStride, ResultStride;
    size_t Rows, Tiles;
    uint32_t Classes, Slices;
    uint32_t RowsPerTile, LanesPerRow, Pitch;  // of AdjustRowsKernel
    CbHipScoreAdjustment A;
};

__device__ __forceinline__ int64_t Clamped(int64_t at, size_t count) {
    return at < 0 ? 0 : at > static_cast<int64_t>(count) ? static_cast<int64_t>(count) : at;
}

// What a row's scores have in common
template <typename A>
struct TRowAdjustment {
    A Repetition, Frequency, Presence;
    const float* ClassBias;
    const uint32_t* Allowed;  // null: no mask

    __device__ __forceinline__ TRowAdjustment(const CbHipScoreAdjustment& p, size_t row) {
        Repetition = p.HistoryOffsets != nullptr && p.Repetition != nullptr ? p.Repetition[row] : 1.f;
        Frequency = p.HistoryOffsets != nullptr && p.Frequency != nullptr ? p.Frequency[row] : 0.f;
        Presence = p.HistoryOffsets != nullptr && p.Presence != nullptr ? p.Presence[row] : 0.f;
        ClassBias = p.ClassBias != nullptr ? p.ClassBias + row * p.ClassBiasStride : nullptr;
        Allowed = nullptr;
        if (p.Allowed != nullptr) {
            const int64_t mask = p.AllowedRows != nullptr ? static_cast<int64_t>(p.AllowedRows[row]) : static_cast<int64_t>(row);
            if (mask >= 0 && static_cast<size_t>(mask) < p.AllowedCount) {
                Allowed = p.Allowed + static_cast<size_t>(mask) * p.AllowedStride;
            }
        }
    }
};

// A tile's table in LDS has a word for each of its scores that counts the row's history: 1 for a class that was given, 2
// for each time that it was generated, so that a word is 0 exactly for the classes outside the history. A second table
// holds the last bias entry of each class, counted from 1. Both are made by integer atomics, whose order does not show.
__device__ __forceinline__ void CountEntry(uint32_t* word, bool given) {
    if (given) {
        atomicOr(word, 1u);
    } else {
        atomicAdd(word, 2u);
    }
}

// N scores from class c on: `words` and `last` their places in the two tables, or null. (A part that a call leaves out has
// the value that changes nothing: a repetition penalty of 1, a frequency and a presence penalty of 0.)
template <typename T, int N>
__device__ __forceinline__ void AdjustValues(TValues<T, N>& v, const TRowAdjustment<TAcc<T>>& row, const CbHipScoreAdjustment& p, uint32_t c, uint32_t classes,
                                             const uint32_t* words, const uint32_t* last, int64_t firstBias) {
    using A = TAcc<T>;
    A x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[i] = static_cast<A>(v.V[i]);
    }
    if (words != nullptr) {
        uint32_t w[N], any = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i] = words[i];
            any |= w[i];
        }
        if (any != 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (w[i] != 0) {
                    x[i] = x[i] > 0 ? x[i] / row.Repetition : x[i] * row.Repetition;
                }
                if (w[i] > 1) {
                    x[i] -= row.Frequency * static_cast<A>(w[i] >> 1);
                    x[i] -= row.Presence;
                }
            }
        }
    }
    if (row.ClassBias != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (c + i < classes) {
                x[i] += row.ClassBias[c + i];
            }
        }
    }
    if (last != nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (last[i] != 0) {
                x[i] += p.BiasValues[firstBias + last[i] - 1];
            }
        }
    }
    if (row.Allowed != nullptr) {
        // (N classes from a multiple of N on are in one word)
        const uint32_t bits = row.Allowed[c >> 5] >> (c & 31);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] = (bits >> i & 1) != 0 ? x[i] : -std::numeric_limits<A>::infinity();
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v.V[i] = static_cast<T>(x[i]);
    }
}

// What a load of N values at a row's end leaves out
template <typename T, int N>
__device__ __forceinline__ TValues<T, N> LoadUpTo(const T* at, uint32_t n) {
    if (n >= N) {
        return TValues<T, N>::Load(at);
    }
    TValues<T, N> v{};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (static_cast<uint32_t>(i) < n) {
            v.V[i] = at[i];
        }
    }
    return v;
}
template <typename T, int N>
__device__ __forceinline__ void StoreUpTo(const TValues<T, N>& v, T* at, uint32_t n) {
    if (n >= N) {
        v.Store(at);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (static_cast<uint32_t>(i) < n) {
            at[i] = v.V[i];
        }
    }
}

// A workgroup for THREADS * P pieces of 16 bytes of one row. The scores are requested before the tables are made, so that
// they arrive meanwhile; every slice of a row looks through the row's whole history.
template <typename T, int THREADS, int P>
__global__ void __launch_bounds__(THREADS) AdjustSliceKernel(TAdjustArgs a) {
    using A = TAcc<T>;
    constexpr int N = 16 / sizeof(T);
    constexpr uint32_t S = THREADS * P * N;
    extern __shared__ uint4 tables[];
    const CbHipScoreAdjustment& p = a.A;
    const bool history = p.HistoryOffsets != nullptr, biases = p.BiasOffsets != nullptr;
    uint32_t* words = reinterpret_cast<uint32_t*>(tables);
    uint32_t* last = history ? words + S : words;
    for (size_t tile = blockIdx.x; tile < a.Tiles; tile += gridDim.x) {
        const size_t row = tile / a.Slices;
        const uint32_t c0 = static_cast<uint32_t>(tile - row * a.Slices) * S;
        const uint32_t width = min(S, a.Classes - c0);
        const T* from = static_cast<const T*>(a.Scores) + row * a.ScoreStride + c0;
        TValues<T, N> v[P];
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint32_t c = (j * THREADS + threadIdx.x) * N;
            if (c < width) {
                v[j] = LoadUpTo<T, N>(from + c, width - c);
            }
        }
        int64_t firstBias = 0;
        if (history || biases) {
            __syncthreads();  // the tile before this one is done with the tables
            for (uint32_t i = threadIdx.x; i < S / 4 * (history + biases); i += THREADS) {
                tables[i] = uint4{0, 0, 0, 0};
            }
            __syncthreads();
            if (history) {
                const int64_t start = p.HistoryOffsets[row];
                const int64_t begin = Clamped(start, p.HistoryCount);
                const int64_t end = Clamped(p.HistoryOffsets[row + 1], p.HistoryCount);
                const int64_t given = start + (p.PromptLengths != nullptr ? p.PromptLengths[row] : 0);
                for (int64_t e = begin + threadIdx.x * 4; e < end; e += THREADS * 4) {
                    const uint32_t n = end - e < 4 ? static_cast<uint32_t>(end - e) : 4;
                    const TValues<int32_t, 4> entries = LoadUpTo<int32_t, 4>(p.History + e, n);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t c = static_cast<uint32_t>(entries.V[i]) - c0;  // outside of the slice: large
                        if (c < width && static_cast<uint32_t>(i) < n) {
                            CountEntry(&words[c], e + i < given);
                        }
                    }
                }
            }
            if (biases) {
                firstBias = Clamped(p.BiasOffsets[row], p.BiasCount);
                const int64_t end = Clamped(p.BiasOffsets[row + 1], p.BiasCount);
                for (int64_t e = firstBias + threadIdx.x; e < end; e += THREADS) {
                    const uint32_t c = static_cast<uint32_t>(p.BiasClasses[e]) - c0;
                    if (c < width) {
                        atomicMax(&last[c], static_cast<uint32_t>(e - firstBias) + 1);
                    }
                }
            }
            __syncthreads();
        }
        const TRowAdjustment<A> common(p, row);
        T* to = static_cast<T*>(a.Result) + row * a.ResultStride + c0;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint32_t c = (j * THREADS + threadIdx.x) * N;
            if (c < width) {
                AdjustValues<T, N>(v[j], common, p, c0 + c, a.Classes, history ? words + c : nullptr, biases ? last + c : nullptr, firstBias);
                StoreUpTo<T, N>(v[j], to + c, width - c);
            }
        }
    }
}

// Rows that are shorter than a slice: a workgroup for RowsPerTile of them, LanesPerRow threads for a row's pieces
constexpr uint32_t kMaxRowsPerTile = 256;

// The row that entry `e` of a list with these offsets belongs to: the last one that begins at or before it
__device__ __forceinline__ uint32_t RowOfEntry(const int64_t* offsets, uint32_t rows, int64_t e) {
    uint32_t low = 0, high = rows;
    while (high - low > 1) {
        const uint32_t middle = (low + high) / 2;
        if (offsets[middle] <= e) {
            low = middle;
        } else {
            high = middle;
        }
    }
    return low;
}

template <typename T>
__global__ void __launch_bounds__(256) AdjustRowsKernel(TAdjustArgs a) {
    using A = TAcc<T>;
    constexpr int N = 16 / sizeof(T);
    extern __shared__ uint4 tables[];
    __shared__ int64_t offsets[kMaxRowsPerTile];
    const CbHipScoreAdjustment& p = a.A;
    const bool history = p.HistoryOffsets != nullptr, biases = p.BiasOffsets != nullptr;
    const uint32_t tableWords = a.RowsPerTile * a.Pitch;
    uint32_t* words = reinterpret_cast<uint32_t*>(tables);
    uint32_t* last = history ? words + tableWords : words;
    const uint32_t lane = threadIdx.x & (a.LanesPerRow - 1), first = threadIdx.x / a.LanesPerRow;
    for (size_t tile = blockIdx.x; tile < a.Tiles; tile += gridDim.x) {
        const size_t r0 = tile * a.RowsPerTile;
        const uint32_t rows = static_cast<uint32_t>(a.Rows - r0 < a.RowsPerTile ? a.Rows - r0 : a.RowsPerTile);
        int64_t firstBias = 0;
        if (history || biases) {
            __syncthreads();  // the tile before this one is done with the tables
            for (uint32_t i = threadIdx.x; i < tableWords * (history + biases); i += 256) {
                words[i] = 0;
            }
        }
        if (history) {
            if (threadIdx.x < rows) {
                offsets[threadIdx.x] = p.HistoryOffsets[r0 + threadIdx.x];
            }
            __syncthreads();
            const int64_t begin = Clamped(offsets[0], p.HistoryCount);
            const int64_t end = Clamped(p.HistoryOffsets[r0 + rows], p.HistoryCount);
            for (int64_t e = begin + threadIdx.x; e < end; e += 256) {
                const uint32_t c = static_cast<uint32_t>(p.History[e]);
                if (c < a.Classes) {
                    const uint32_t r = RowOfEntry(offsets, rows, e);
                    CountEntry(&words[r * a.Pitch + c], p.PromptLengths != nullptr && e - offsets[r] < p.PromptLengths[r0 + r]);
                }
            }
        }
        if (biases) {
            __syncthreads();
            if (threadIdx.x < rows) {
                offsets[threadIdx.x] = p.BiasOffsets[r0 + threadIdx.x];
            }
            __syncthreads();
            firstBias = Clamped(offsets[0], p.BiasCount);
            const int64_t end = Clamped(p.BiasOffsets[r0 + rows], p.BiasCount);
            for (int64_t e = firstBias + threadIdx.x; e < end; e += 256) {
                const uint32_t c = static_cast<uint32_t>(p.BiasClasses[e]);
                if (c < a.Classes) {
                    atomicMax(&last[RowOfEntry(offsets, rows, e) * a.Pitch + c], static_cast<uint32_t>(e - firstBias) + 1);
                }
            }
        }
        if (history || biases) {
            __syncthreads();
        }
        for (uint32_t r = first; r < rows; r += 256 / a.LanesPerRow) {
            const size_t row = r0 + r;
            const TRowAdjustment<A> common(p, row);
            const T* from = static_cast<const T*>(a.Scores) + row * a.ScoreStride;
            T* to = static_cast<T*>(a.Result) + row * a.ResultStride;
            for (uint32_t c = lane * N; c < a.Classes; c += a.LanesPerRow * N) {
                TValues<T, N> v = LoadUpTo<T, N>(from + c, a.Classes - c);
                AdjustValues<T, N>(v, common, p, c, a.Classes, history ? words + r * a.Pitch + c : nullptr, biases ? last + r * a.Pitch + c : nullptr,
                                   firstBias);
                StoreUpTo<T, N>(v, to + c, a.Classes - c);
            }
        }
    }
}

// ---------------------------------------------------------------- the best classes ----

// A score with its class as one value that orders them: larger scores first, of equal ones the lower class first. What is
// never selected (minus infinity, NaN) comes behind all others. 16-bit scores and their class fit 32 bits, 32-bit ones 64.
template <typename T>
struct TRanked {
    using Bits = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
    using Key = std::conditional_t<sizeof(T) == 2, uint32_t, uint64_t>;
    static constexpr int kBits = 8 * sizeof(T);
    Key K;

    __device__ __forceinline__ static TRanked None() { return {0}; }
    __device__ __forceinline__ static TRanked Of(T score, uint32_t c) {
        const float x = static_cast<float>(score);
        if (!(x > -std::numeric_limits<float>::infinity())) {
            return None();
        }
        Bits bits = __builtin_bit_cast(Bits, score);
        bits = x == 0 ? Bits(0) : bits;  // zeros of both signs are equal
        const Bits sign = Bits(1) << (kBits - 1);
        bits = (bits & sign) != 0 ? static_cast<Bits>(~bits) : static_cast<Bits>(bits | sign);
        return {static_cast<Key>(bits) << kBits | static_cast<Bits>(~c)};
    }
    __device__ __forceinline__ bool IsNone() const { return K == 0; }
    __device__ __forceinline__ uint32_t Class() const { return static_cast<Bits>(~static_cast<Bits>(K)); }
    __device__ __forceinline__ float Score() const {
        Bits bits = static_cast<Bits>(K >> kBits);
        const Bits sign = Bits(1) << (kBits - 1);
        bits = (bits & sign) != 0 ? static_cast<Bits>(bits & ~sign) : static_cast<Bits>(~bits);
        return IsNone() ? -std::numeric_limits<float>::infinity() : static_cast<float>(__builtin_bit_cast(T, bits));
    }
    __device__ __forceinline__ TRanked Better(const TRanked& other) const { return other.K > K ? other : *this; }
    __device__ __forceinline__ bool Same(const TRanked& other) const { return K == other.K; }
};
template <>
struct TRanked<double> {
    double Value;
    uint32_t C, Unused;

    __device__ __forceinline__ static TRanked None() { return {-std::numeric_limits<double>::infinity(), ~0u, 0}; }
    __device__ __forceinline__ static TRanked Of(double x, uint32_t c) {
        return x > -std::numeric_limits<double>::infinity() ? TRanked{x, c, 0} : None();
    }
    __device__ __forceinline__ bool IsNone() const { return C == ~0u; }
    __device__ __forceinline__ uint32_t Class() const { return C; }
    __device__ __forceinline__ double Score() const { return Value; }
    __device__ __forceinline__ TRanked Better(const TRanked& other) const {
        return other.Value > Value || (other.Value == Value && other.C < C) ? other : *this;
    }
    __device__ __forceinline__ bool Same(const TRanked& other) const { return C == other.C; }
};

// What a lane gets from another one: STEP lanes on, around in its row of 16 (a modifier of the instruction that uses it, and
// no trip through LDS), or the lane whose number differs in the bit STEP
template <int STEP, typename V>
__device__ __forceinline__ V FromLane(const V& x) {
    V r;
    constexpr int words = sizeof(V) / 4;
    int from[words], to[words];
    __builtin_memcpy(from, &x, sizeof(V));
#pragma unroll
    for (int i = 0; i < words; ++i) {
        if constexpr (STEP < 16) {
            to[i] = __builtin_amdgcn_update_dpp(0, from[i], 0x120 + STEP, 0xf, 0xf, false);
        } else {
            to[i] = __shfl_xor(from[i], STEP);
        }
    }
    __builtin_memcpy(&r, to, sizeof(V));
    return r;
}

// f over the values of a group of 16 or 64 lanes, in the same order in each of them
template <int G, typename V, typename F>
__device__ __forceinline__ V OverGroup(V x, F&& f) {
    static_assert(G == 16 || G == 64);
    x = f(x, FromLane<8>(x));
    x = f(x, FromLane<4>(x));
    x = f(x, FromLane<2>(x));
    x = f(x, FromLane<1>(x));
    if constexpr (G == 64) {
        x = f(x, FromLane<16>(x));
        x = f(x, FromLane<32>(x));
    }
    return x;
}

template <int G, typename A>
__device__ __forceinline__ A GroupSum(A x) {
    return OverGroup<G>(x, [](A a, A b) { return a + b; });
}

// exp(x - most), 1 for the largest also where it is infinite; 0 for minus infinity
__device__ __forceinline__ float WeightOf(float x, float most) {
    return x == most ? 1.f : expf(x - most);
}
__device__ __forceinline__ double WeightOf(double x, double most) {
    return x == most ? 1. : exp(x - most);
}

template <typename T>
struct TTopArgs {
    const T* Scores;
    size_t Stride, Rows;
    uint32_t Classes, Count;
    bool Among;
};

// G lanes for a row, V classes next to each other for each of them. A round finds the best class that is left: in the
// lane's own, then over the group; whoever has it takes it out. Lane k % G keeps what round k finds.
template <typename T, int G, int V>
__global__ void __launch_bounds__(256) SelectTopKernel(TTopArgs<T> a, int32_t* indexes, TAcc<T>* weights) {
    using A = TAcc<T>;
    using R = TRanked<T>;
    constexpr int kept = 32 / G > 0 ? 32 / G : 1;
    const uint32_t lane = threadIdx.x & (G - 1);
    for (size_t row = size_t(blockIdx.x) * (256 / G) + threadIdx.x / G; row < a.Rows; row += size_t(gridDim.x) * (256 / G)) {
        const uint32_t c = lane * V;
        TValues<T, V> v{};
        if (c < a.Classes) {
            v = LoadUpTo<T, V>(a.Scores + row * a.Stride + c, a.Classes - c);
        }
        R left[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            left[j] = c + j < a.Classes ? R::Of(v.V[j], c + j) : R::None();
        }
        R mine[kept];
#pragma unroll
        for (int i = 0; i < kept; ++i) {
            mine[i] = R::None();
        }
        A most = 0, total = 0;
        for (uint32_t k = 0; k < a.Count; ++k) {
            R best = left[0];
#pragma unroll
            for (int j = 1; j < V; ++j) {
                best = best.Better(left[j]);
            }
            best = OverGroup<G>(best, [](const R& x, const R& y) { return x.Better(y); });
            if (k == 0) {
                most = best.Score();
                if (!a.Among) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        total += left[j].IsNone() ? A(0) : WeightOf(left[j].Score(), most);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                left[j] = left[j].Same(best) ? R::None() : left[j];
            }
#pragma unroll
            for (int i = 0; i < kept; ++i) {
                mine[i] = k == lane + i * G ? best : mine[i];
            }
        }
        A e[kept];
#pragma unroll
        for (int i = 0; i < kept; ++i) {
            e[i] = mine[i].IsNone() ? A(0) : WeightOf(mine[i].Score(), most);
            total += a.Among ? e[i] : A(0);
        }
        total = GroupSum<G>(total);
#pragma unroll
        for (int i = 0; i < kept; ++i) {
            const uint32_t k = lane + i * G;
            if (k < a.Count) {
                indexes[row * a.Count + k] = mine[i].IsNone() ? -1 : static_cast<int32_t>(mine[i].Class());
                weights[row * a.Count + k] = mine[i].IsNone() ? A(0) : e[i] / total;
            }
        }
    }
}

// The row of C classes at most that a thread has to itself
template <typename T, int C>
__device__ __forceinline__ TValues<T, C> LoadRow(const T* from, uint32_t classes) {
    constexpr int N = C < 16 / static_cast<int>(sizeof(T)) ? C : 16 / sizeof(T);
    TValues<T, C> v{};
#pragma unroll
    for (int j = 0; j < C; j += N) {
        if (static_cast<uint32_t>(j) < classes) {
            const TValues<T, N> part = LoadUpTo<T, N>(from + j, classes - j);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v.V[j + i] = part.V[i];
            }
        }
    }
    return v;
}

// Rows of few classes: a thread for a row of at most C
template <typename T, int C>
__global__ void __launch_bounds__(256) SelectTopOfFewKernel(TTopArgs<T> a, int32_t* indexes, TAcc<T>* weights) {
    using A = TAcc<T>;
    using R = TRanked<T>;
    for (size_t row = size_t(blockIdx.x) * 256 + threadIdx.x; row < a.Rows; row += size_t(gridDim.x) * 256) {
        const TValues<T, C> v = LoadRow<T, C>(a.Scores + row * a.Stride, a.Classes);
        R left[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            left[j] = static_cast<uint32_t>(j) < a.Classes ? R::Of(v.V[j], j) : R::None();
        }
        A most = 0, total = 0;
        for (uint32_t k = 0; k < a.Count; ++k) {
            R best = left[0];
#pragma unroll
            for (int j = 1; j < C; ++j) {
                best = best.Better(left[j]);
            }
            if (k == 0) {
                most = best.Score();
                if (!a.Among) {
#pragma unroll
                    for (int j = 0; j < C; ++j) {
                        total += left[j].IsNone() ? A(0) : WeightOf(left[j].Score(), most);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < C; ++j) {
                left[j] = left[j].Same(best) ? R::None() : left[j];
            }
            const A e = best.IsNone() ? A(0) : WeightOf(best.Score(), most);
            indexes[row * a.Count + k] = best.IsNone() ? -1 : static_cast<int32_t>(best.Class());
            weights[row * a.Count + k] = a.Among || best.IsNone() ? e : e / total;
            total += a.Among ? e : A(0);
        }
        if (a.Among && total > 0) {
            for (uint32_t k = 0; k < a.Count; ++k) {
                weights[row * a.Count + k] /= total;
            }
        }
    }
}

template <typename T>
struct TTopGradientArgs {
    const int32_t* Indexes;
    const TAcc<T>* Weights;
    const TAcc<T>* WeightGradients;
    T* Gradients;
    size_t GradientStride;
};

// With w the weights, p the softmax over all classes and g the weights' gradients, m = sum of g w over the selected:
// among the selected only w_k (g_k - m) and 0 elsewhere, else w_k g_k - p m with the first part 0 elsewhere.
// A row's gradients are put together in LDS, where the selected classes' lanes add their parts.
template <typename T, int G, int V>
__global__ void __launch_bounds__(256) SelectTopBackwardKernel(TTopArgs<T> a, TTopGradientArgs<T> b) {
    using A = TAcc<T>;
    constexpr int kept = 32 / G > 0 ? 32 / G : 1;
    __shared__ __align__(16) A sums[256 * V];
    const uint32_t lane = threadIdx.x & (G - 1);
    A* mySums = sums + threadIdx.x / G * (G * V);
    for (size_t row = size_t(blockIdx.x) * (256 / G) + threadIdx.x / G; row < a.Rows; row += size_t(gridDim.x) * (256 / G)) {
        const uint32_t c = lane * V;
        int32_t index[kept];
        A part[kept], mean = 0;
#pragma unroll
        for (int i = 0; i < kept; ++i) {
            const uint32_t k = lane + i * G;
            index[i] = k < a.Count ? b.Indexes[row * a.Count + k] : -1;
            const A w = index[i] >= 0 ? b.Weights[row * a.Count + k] : A(0);
            const A g = index[i] >= 0 ? b.WeightGradients[row * a.Count + k] : A(0);
            part[i] = a.Among ? g : w * g;
            mean += w * g;
        }
        mean = GroupSum<G>(mean);
        if (a.Among) {
#pragma unroll
            for (int i = 0; i < kept; ++i) {
                part[i] = index[i] >= 0 ? b.Weights[row * a.Count + lane + i * G] * (part[i] - mean) : A(0);
            }
        }
        TValues<A, V> x{};
        if (!a.Among) {
            TValues<T, V> v{};
            if (c < a.Classes) {
                v = LoadUpTo<T, V>(a.Scores + row * a.Stride + c, a.Classes - c);
            }
            A most = -std::numeric_limits<A>::infinity();
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const A s = static_cast<A>(v.V[j]);
                x.V[j] = c + j < a.Classes && s == s ? s : -std::numeric_limits<A>::infinity();
                most = x.V[j] > most ? x.V[j] : most;
            }
            most = OverGroup<G>(most, [](A y, A z) { return z > y ? z : y; });
            A total = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x.V[j] = x.V[j] > -std::numeric_limits<A>::infinity() ? WeightOf(x.V[j], most) : A(0);
                total += x.V[j];
            }
            total = GroupSum<G>(total);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x.V[j] = total > 0 ? -(x.V[j] / total) * mean : A(0);
            }
        }
        x.Store(mySums + c);
        __builtin_amdgcn_wave_barrier();  // a row's lanes are of one wave, whose LDS operations are done in order
#pragma unroll
        for (int i = 0; i < kept; ++i) {
            if (static_cast<uint32_t>(index[i]) < a.Classes) {
                mySums[index[i]] += part[i];
            }
        }
        __builtin_amdgcn_wave_barrier();
        x = TValues<A, V>::Load(mySums + c);
        __builtin_amdgcn_wave_barrier();
        if (c < a.Classes) {
            TValues<T, V> v;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v.V[j] = static_cast<T>(x.V[j]);
            }
            StoreUpTo<T, V>(v, b.Gradients + row * b.GradientStride + c, a.Classes - c);
        }
    }
}

template <typename T, int C>
__global__ void __launch_bounds__(256) SelectTopOfFewBackwardKernel(TTopArgs<T> a, TTopGradientArgs<T> b) {
    using A = TAcc<T>;
    for (size_t row = size_t(blockIdx.x) * 256 + threadIdx.x; row < a.Rows; row += size_t(gridDim.x) * 256) {
        const int32_t* indexes = b.Indexes + row * a.Count;
        const A* weights = b.Weights + row * a.Count;
        const A* gradients = b.WeightGradients + row * a.Count;
        A mean = 0;
        for (uint32_t k = 0; k < a.Count; ++k) {
            mean += indexes[k] >= 0 ? weights[k] * gradients[k] : A(0);
        }
        A x[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            x[j] = 0;
        }
        if (!a.Among) {
            const TValues<T, C> v = LoadRow<T, C>(a.Scores + row * a.Stride, a.Classes);
            A most = -std::numeric_limits<A>::infinity(), total = 0;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const A s = static_cast<A>(v.V[j]);
                x[j] = static_cast<uint32_t>(j) < a.Classes && s == s ? s : -std::numeric_limits<A>::infinity();
                most = x[j] > most ? x[j] : most;
            }
#pragma unroll
            for (int j = 0; j < C; ++j) {
                x[j] = x[j] > -std::numeric_limits<A>::infinity() ? WeightOf(x[j], most) : A(0);
                total += x[j];
            }
#pragma unroll
            for (int j = 0; j < C; ++j) {
                x[j] = total > 0 ? -(x[j] / total) * mean : A(0);
            }
        }
        for (uint32_t k = 0; k < a.Count; ++k) {
            const int32_t index = indexes[k];
            if (index >= 0) {
                const A part = a.Among ? weights[k] * (gradients[k] - mean) : weights[k] * gradients[k];
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    x[j] += index == j ? part : A(0);
                }
            }
        }
        constexpr int N = C < 16 / static_cast<int>(sizeof(T)) ? C : 16 / sizeof(T);
#pragma unroll
        for (int j = 0; j < C; j += N) {
            if (static_cast<uint32_t>(j) < a.Classes) {
                TValues<T, N> v;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    v.V[i] = static_cast<T>(x[j + i]);
                }
                StoreUpTo<T, N>(v, b.Gradients + row * b.GradientStride + j, a.Classes - j);
            }
        }
    }
}

}  // namespace op

using namespace op;

namespace {

constexpr uint32_t kRowTileWords = 4096;      // of a table of AdjustRowsKernel
constexpr size_t kWorkgroupsWanted = 512;     // two for each compute unit

}  // namespace

void AdjustScores(int valueType, size_t rows, size_t classes, const void* scores, size_t scoreStride,
                  const CbHipScoreAdjustment& p, void* result, size_t resultStride, void* stream) {
    const size_t size = ValueSize(valueType);
    CBAMD_ENSURE(classes <= 0x7fffffffu, "too many classes: " + std::to_string(classes));
    if (rows == 0 || classes == 0) {
        return;
    }
    CheckMatrix("scores", scores, rows, classes, scoreStride, size);
    CheckMatrix("result", result, rows, classes, resultStride, size);
    CBAMD_ENSURE(scores != result || rows == 1 || scoreStride == resultStride, "scores adjusted in place need the same stride");
    const bool history = p.HistoryOffsets != nullptr;
    CBAMD_ENSURE(!history || p.History != nullptr || p.HistoryCount == 0, "history pointer is null");
    CBAMD_ENSURE(p.History == nullptr || history, "history offsets pointer is null");
    const bool biases = p.BiasOffsets != nullptr;
    CBAMD_ENSURE(!biases || (p.BiasClasses != nullptr && p.BiasValues != nullptr) || p.BiasCount == 0, "bias classes or values pointer is null");
    CBAMD_ENSURE((p.BiasClasses == nullptr && p.BiasValues == nullptr) || biases, "bias offsets pointer is null");
    CBAMD_ENSURE(p.BiasCount <= 0x7fffffffu, "too many biases: " + std::to_string(p.BiasCount));
    CBAMD_ENSURE(p.ClassBias == nullptr || p.ClassBiasStride == 0 || p.ClassBiasStride >= classes, "class bias stride is shorter than a row");
    if (p.Allowed != nullptr) {
        CBAMD_ENSURE(p.AllowedStride >= (classes + 31) / 32 || p.AllowedCount <= 1, "mask stride is shorter than a mask");
        CBAMD_ENSURE(p.AllowedRows != nullptr || p.AllowedCount >= rows, "fewer masks than rows");
    }
    CBAMD_ENSURE(p.AllowedRows == nullptr || p.Allowed != nullptr, "mask pointer is null");
    TAdjustArgs a{};
    a.Scores = scores;
    a.Result = result;
    a.ScoreStride = scoreStride;
    a.ResultStride = resultStride;
    a.Rows = rows;
    a.Classes = static_cast<uint32_t>(classes);
    a.A = p;
    const TCallDevice call(result, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        constexpr uint32_t N = 16 / sizeof(T);
        const size_t tables = size_t(history) + size_t(biases);
        if (a.Classes <= kRowTileWords / 2) {
            const uint32_t pieces = (a.Classes + N - 1) / N;
            a.Pitch = (pieces | 1) * N;  // an odd number of pieces: rows begin in different LDS banks
            a.RowsPerTile = std::min<uint32_t>(kMaxRowsPerTile, std::max<uint32_t>(1, kRowTileWords / a.Pitch));
            a.LanesPerRow = 1;
            while (a.LanesPerRow < 256 && a.LanesPerRow * 8 < pieces) {
                a.LanesPerRow *= 2;
            }
            a.Tiles = (rows + a.RowsPerTile - 1) / a.RowsPerTile;
            call.Launch(AdjustRowsKernel<T>, std::min<size_t>(a.Tiles, 1u << 20), 256, size_t(a.RowsPerTile) * a.Pitch * 4 * tables, a);
            return;
        }
        const auto slices = [&](uint32_t size) { return (a.Classes + size - 1) / size; };
        const auto launch = [&](auto threads, auto perThread) {
            constexpr int THREADS = decltype(threads)::value, P = decltype(perThread)::value;
            a.Slices = slices(THREADS * P * N);
            a.Tiles = rows * a.Slices;
            const auto kernel = AdjustSliceKernel<T, THREADS, P>;
            const size_t lds = size_t(THREADS) * P * N * 4 * tables;
            call.AllowLds(reinterpret_cast<const void*>(kernel), lds);
            call.Launch(kernel, std::min<size_t>(a.Tiles, 1u << 20), THREADS, lds, a);
        };
        const auto atLeast = [&](uint32_t size) { return rows >= (kWorkgroupsWanted + slices(size) - 1) / slices(size); };
        using std::integral_constant;
        if (atLeast(16384)) {
            launch(integral_constant<int, 1024>(), integral_constant<int, 16 / N>());
        } else if (atLeast(8192)) {
            launch(integral_constant<int, 1024>(), integral_constant<int, 8 / N>());
        } else if (atLeast(4096)) {
            launch(integral_constant<int, (4096 / N < 1024 ? 4096 / N : 1024)>(), integral_constant<int, (4096 / N < 1024 ? 1 : 4096 / N / 1024)>());
        } else {
            launch(integral_constant<int, (2048 / N < 1024 ? 2048 / N : 1024)>(), integral_constant<int, (2048 / N < 1024 ? 1 : 2048 / N / 1024)>());
        }
    });
}

namespace {

constexpr size_t kMaxTopClasses = 1024;
constexpr int32_t kMaxTopCount = 32;
constexpr size_t kRowsForThreads = 16384;  // a wave for each compute unit

void CheckTop(size_t rows, size_t classes, int32_t count) {
    CBAMD_ENSURE(classes <= kMaxTopClasses, "too many classes to select from: " + std::to_string(classes) + ", at most " + std::to_string(kMaxTopClasses));
    CBAMD_ENSURE(count >= 1 && count <= kMaxTopCount, "selected classes per row: " + std::to_string(count) + ", 1 to " + std::to_string(kMaxTopCount) + " are supported");
    CBAMD_ENSURE(classes > 0 || rows == 0, "no classes to select from");
    CBAMD_ENSURE(rows <= size_t(1) << 48, "too many rows");
}

// f(lanes of a row, classes of a lane), 1 lane: a thread has the row to itself. That reads each line of memory once as long
// as a row is short, and needs rows enough to fill the chip with threads.
template <typename F>
void WithShape(size_t classes, size_t rows, F&& f) {
    using std::integral_constant;
    const auto shape = [&](auto lanes, auto perLane) { f(lanes, perLane); };
    if (rows >= kRowsForThreads && classes <= 32) {
        const integral_constant<int, 1> alone;
        return classes <= 4 ? shape(alone, integral_constant<int, 4>()) : classes <= 8 ? shape(alone, integral_constant<int, 8>())
            : classes <= 16 ? shape(alone, integral_constant<int, 16>()) : shape(alone, integral_constant<int, 32>());
    }
    const integral_constant<int, 16> sixteen;
    const integral_constant<int, 64> wave;
    return classes <= 16 ? shape(sixteen, integral_constant<int, 1>()) : classes <= 32 ? shape(sixteen, integral_constant<int, 2>())
        : classes <= 64 ? shape(sixteen, integral_constant<int, 4>()) : classes <= 128 ? shape(sixteen, integral_constant<int, 8>())
        : classes <= 256 ? shape(sixteen, integral_constant<int, 16>()) : classes <= 512 ? shape(wave, integral_constant<int, 8>())
        : shape(wave, integral_constant<int, 16>());
}

size_t GroupsOf(size_t rows, int lanes) {
    const size_t rowsPerGroup = 256 / lanes;
    return std::min<size_t>((rows + rowsPerGroup - 1) / rowsPerGroup, 1u << 20);
}

}  // namespace

void SelectTop(int valueType, size_t rows, size_t classes, const void* scores, size_t scoreStride, int32_t count,
               bool amongSelected, int32_t* indexes, void* weights, void* stream) {
    const size_t size = ValueSize(valueType);
    CheckTop(rows, classes, count);
    if (rows == 0) {
        return;
    }
    CheckMatrix("scores", scores, rows, classes, scoreStride, size);
    CBAMD_ENSURE(indexes != nullptr && weights != nullptr, "indexes or weights pointer is null");
    const TCallDevice call(indexes, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        const TTopArgs<T> a{static_cast<const T*>(scores), scoreStride, rows, static_cast<uint32_t>(classes), static_cast<uint32_t>(count), amongSelected};
        WithShape(classes, rows, [&](auto lanes, auto perLane) {
            constexpr int G = decltype(lanes)::value, V = decltype(perLane)::value;
            if constexpr (G == 1) {
                call.Launch(SelectTopOfFewKernel<T, V>, GroupsOf(rows, G), 256, 0, a, indexes, static_cast<TAcc<T>*>(weights));
            } else {
                call.Launch(SelectTopKernel<T, G, V>, GroupsOf(rows, G), 256, 0, a, indexes, static_cast<TAcc<T>*>(weights));
            }
        });
    });
}

void SelectTopBackward(int valueType, size_t rows, size_t classes, const void* scores, size_t scoreStride, int32_t count,
                       bool amongSelected, const int32_t* indexes, const void* weights, const void* weightGradients,
                       void* scoreGradients, size_t gradientStride, void* stream) {
    const size_t size = ValueSize(valueType);
    CheckTop(rows, classes, count);
    if (rows == 0) {
        return;
    }
    if (!amongSelected) {
        CheckMatrix("scores", scores, rows, classes, scoreStride, size);
    }
    CheckMatrix("score gradients", scoreGradients, rows, classes, gradientStride, size);
    CBAMD_ENSURE(indexes != nullptr && weights != nullptr && weightGradients != nullptr, "indexes, weights or weight gradients pointer is null");
    const TCallDevice call(scoreGradients, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        const TTopArgs<T> a{static_cast<const T*>(scores), scoreStride, rows, static_cast<uint32_t>(classes), static_cast<uint32_t>(count), amongSelected};
        const TTopGradientArgs<T> b{indexes, static_cast<const TAcc<T>*>(weights), static_cast<const TAcc<T>*>(weightGradients),
                                    static_cast<T*>(scoreGradients), gradientStride};
        WithShape(classes, rows, [&](auto lanes, auto perLane) {
            constexpr int G = decltype(lanes)::value, V = decltype(perLane)::value;
            if constexpr (G == 1) {
                call.Launch(SelectTopOfFewBackwardKernel<T, V>, GroupsOf(rows, G), 256, 0, a, b);
            } else {
                call.Launch(SelectTopBackwardKernel<T, G, V>, GroupsOf(rows, G), 256, 0, a, b);
            }
        });
    });
}

}  // namespace cbamd
