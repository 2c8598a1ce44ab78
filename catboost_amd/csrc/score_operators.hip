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
    uint32_t Classes, Slices;       // a tile: RowsPerTile rows, or one slice of SliceClasses classes of one row
    uint32_t RowsPerTile, SliceClasses;
    CbHipScoreAdjustment A;
};

__device__ __forceinline__ int64_t Clamped(int64_t at, size_t count) {
    return at < 0 ? 0 : at > static_cast<int64_t>(count) ? static_cast<int64_t>(count) : at;
}

// The row of [first, first + rows) that entry `e` of a list with these offsets belongs to: the last one that begins at or before it
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

// A tile's table in LDS has a word for each of its scores that counts the row's history: 1 for a class that was given, 2
// for each time that it was generated, so that a word is 0 exactly for the classes outside the history. A second table
// holds the last bias entry of each class. Both are made by integer atomics, whose order does not show in the result.
template <typename T, bool HISTORY, bool BIASES>
__global__ void __launch_bounds__(256) AdjustKernel(TAdjustArgs a) {
    using A = TAcc<T>;
    extern __shared__ uint32_t table[];
    const CbHipScoreAdjustment& p = a.A;
    for (size_t tile = blockIdx.x; tile < a.Tiles; tile += gridDim.x) {
        const size_t r0 = tile / a.Slices * a.RowsPerTile;
        const uint32_t rows = static_cast<uint32_t>(a.Rows - r0 < a.RowsPerTile ? a.Rows - r0 : a.RowsPerTile);
        const uint32_t c0 = static_cast<uint32_t>(tile % a.Slices) * a.SliceClasses;
        const uint32_t width = min(a.SliceClasses, a.Classes - c0);
        const uint32_t n = rows * width;
        uint32_t* last = HISTORY ? table + n : table;
        int64_t firstBias = 0;
        if (HISTORY || BIASES) {
            __syncthreads();  // the tile before this one is done with the tables
            for (uint32_t i = threadIdx.x; i < n * (HISTORY + BIASES); i += blockDim.x) {
                table[i] = 0;
            }
            __syncthreads();
        }
        if (HISTORY) {
            const int64_t begin = Clamped(p.HistoryOffsets[r0], p.HistoryCount);
            const int64_t end = Clamped(p.HistoryOffsets[r0 + rows], p.HistoryCount);
            for (int64_t e = begin + threadIdx.x; e < end; e += blockDim.x) {
                const uint32_t c = static_cast<uint32_t>(p.History[e]) - c0;  // outside of the slice: large
                if (c < width) {
                    const uint32_t r = RowOfEntry(p.HistoryOffsets + r0, rows, e);
                    const int64_t within = e - p.HistoryOffsets[r0 + r];
                    if (p.PromptLengths != nullptr && within < p.PromptLengths[r0 + r]) {
                        atomicOr(&table[r * width + c], 1u);
                    } else {
                        atomicAdd(&table[r * width + c], 2u);
                    }
                }
            }
        }
        if (BIASES) {
            firstBias = Clamped(p.BiasOffsets[r0], p.BiasCount);
            const int64_t end = Clamped(p.BiasOffsets[r0 + rows], p.BiasCount);
            for (int64_t e = firstBias + threadIdx.x; e < end; e += blockDim.x) {
                const uint32_t c = static_cast<uint32_t>(p.BiasClasses[e]) - c0;
                if (c < width) {
                    atomicMax(&last[RowOfEntry(p.BiasOffsets + r0, rows, e) * width + c], static_cast<uint32_t>(e - firstBias) + 1);
                }
            }
        }
        if (HISTORY || BIASES) {
            __syncthreads();
        }
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
            const uint32_t r = i / width;
            const uint32_t c = c0 + (i - r * width);
            const size_t row = r0 + r;
            A x = static_cast<A>(static_cast<const T*>(a.Scores)[row * a.ScoreStride + c]);
            if (HISTORY) {
                const uint32_t word = table[i];
                if (word != 0) {
                    if (p.Repetition != nullptr) {
                        const A repetition = p.Repetition[row];
                        x = x > 0 ? x / repetition : x * repetition;
                    }
                    const uint32_t generated = word >> 1;
                    if (generated != 0) {
                        if (p.Frequency != nullptr) {
                            x -= static_cast<A>(p.Frequency[row]) * static_cast<A>(generated);
                        }
                        if (p.Presence != nullptr) {
                            x -= p.Presence[row];
                        }
                    }
                }
            }
            if (p.ClassBias != nullptr) {
                x += p.ClassBias[row * p.ClassBiasStride + c];
            }
            if (BIASES) {
                const uint32_t entry = last[i];
                if (entry != 0) {
                    x += p.BiasValues[firstBias + entry - 1];
                }
            }
            if (p.Allowed != nullptr) {
                const int64_t mask = p.AllowedRows != nullptr ? static_cast<int64_t>(p.AllowedRows[row]) : static_cast<int64_t>(row);
                if (mask >= 0 && static_cast<size_t>(mask) < p.AllowedCount &&
                    (p.Allowed[mask * p.AllowedStride + (c >> 5)] >> (c & 31) & 1) == 0) {
                    x = -std::numeric_limits<A>::infinity();
                }
            }
            static_cast<T*>(a.Result)[row * a.ResultStride + c] = static_cast<T>(x);
        }
    }
}

// ---------------------------------------------------------------- the best classes ----

template <typename A>
struct TCandidate {
    A Value;
    uint32_t Class;
    // larger first, of equal ones the lower class first
    __device__ __forceinline__ bool Before(const TCandidate& other) const {
        return Value > other.Value || (Value == other.Value && Class < other.Class);
    }
};

template <typename A>
__device__ __forceinline__ A WaveSum(A x) {
    for (int step = 32; step > 0; step /= 2) {
        x += __shfl_xor(x, step);
    }
    return x;
}

// A row's scores as they take part: minus infinity for what is never selected
template <typename A>
__device__ __forceinline__ A Selectable(A x) {
    return x == x ? x : -std::numeric_limits<A>::infinity();
}

// exp(x - most), 1 for the largest also where it is infinite
template <typename A>
__device__ __forceinline__ A WeightOf(A x, A most) {
    return x == most ? A(1) : sizeof(A) == 8 ? static_cast<A>(exp(static_cast<double>(x - most))) : static_cast<A>(expf(static_cast<float>(x - most)));
}

// A wave for a row, V classes a lane
template <typename T, int V>
__global__ void __launch_bounds__(256) SelectTopKernel(const T* scores, size_t stride, size_t rows, uint32_t classes, uint32_t count,
                                                       bool among, int32_t* indexes, TAcc<T>* weights) {
    using A = TAcc<T>;
    const A none = -std::numeric_limits<A>::infinity();
    const uint32_t lane = threadIdx.x & 63;
    for (size_t row = size_t(blockIdx.x) * 4 + threadIdx.x / 64; row < rows; row += size_t(gridDim.x) * 4) {
        A v[V];
        A most = none;
        for (int j = 0; j < V; ++j) {
            const uint32_t c = lane + 64 * j;
            v[j] = c < classes ? Selectable(static_cast<A>(scores[row * stride + c])) : none;
            most = v[j] > most ? v[j] : most;
        }
        for (int step = 32; step > 0; step /= 2) {
            const A other = __shfl_xor(most, step);
            most = other > most ? other : most;
        }
        A total = 0;
        if (!among && most > none) {
            for (int j = 0; j < V; ++j) {
                total += v[j] > none ? WeightOf(v[j], most) : A(0);
            }
            total = WaveSum(total);
        }
        A mine = none;  // lane k: the k-th selected score and its class
        int32_t mineClass = -1;
        for (uint32_t k = 0; k < count; ++k) {
            TCandidate<A> best{none, ~0u};
            for (int j = 0; j < V; ++j) {
                const TCandidate<A> x{v[j], lane + 64 * j};
                best = x.Before(best) ? x : best;
            }
            for (int step = 32; step > 0; step /= 2) {
                const TCandidate<A> other{__shfl_xor(best.Value, step), static_cast<uint32_t>(__shfl_xor(static_cast<int>(best.Class), step))};
                best = other.Before(best) ? other : best;
            }
            if (!(best.Value > none)) {
                break;
            }
            for (int j = 0; j < V; ++j) {
                if (best.Class == lane + 64 * j) {
                    v[j] = none;
                }
            }
            if (lane == k) {
                mine = best.Value;
                mineClass = static_cast<int32_t>(best.Class);
            }
        }
        const A e = mineClass >= 0 ? WeightOf(mine, most) : A(0);
        if (among) {
            total = WaveSum(e);
        }
        if (lane < count) {
            indexes[row * count + lane] = mineClass;
            weights[row * count + lane] = mineClass >= 0 ? e / total : A(0);
        }
    }
}

// With w the weights, p the softmax over all classes and g the weights' gradients, m = sum of g w over the selected:
// among the selected only w_k (g_k - m) and 0 elsewhere, else w_k g_k - p m with the first part 0 elsewhere
template <typename T, int V>
__global__ void __launch_bounds__(256) SelectTopBackwardKernel(const T* scores, size_t stride, size_t rows, uint32_t classes, uint32_t count,
                                                               bool among, const int32_t* indexes, const TAcc<T>* weights,
                                                               const TAcc<T>* weightGradients, T* gradients, size_t gradientStride) {
    using A = TAcc<T>;
    const A none = -std::numeric_limits<A>::infinity();
    const uint32_t lane = threadIdx.x & 63;
    for (size_t row = size_t(blockIdx.x) * 4 + threadIdx.x / 64; row < rows; row += size_t(gridDim.x) * 4) {
        const int32_t index = lane < count ? indexes[row * count + lane] : -1;
        const A w = index >= 0 ? weights[row * count + lane] : A(0);
        const A g = index >= 0 ? weightGradients[row * count + lane] : A(0);
        const A mean = WaveSum(w * g);
        const A part = among ? w * (g - mean) : w * g;
        A v[V];
        for (int j = 0; j < V; ++j) {
            v[j] = 0;
        }
        if (!among) {
            A most = none;
            for (int j = 0; j < V; ++j) {
                const uint32_t c = lane + 64 * j;
                v[j] = c < classes ? Selectable(static_cast<A>(scores[row * stride + c])) : none;
                most = v[j] > most ? v[j] : most;
            }
            for (int step = 32; step > 0; step /= 2) {
                const A other = __shfl_xor(most, step);
                most = other > most ? other : most;
            }
            A total = 0;
            for (int j = 0; j < V; ++j) {
                v[j] = v[j] > none ? WeightOf(v[j], most) : A(0);
                total += v[j];
            }
            total = WaveSum(total);
            for (int j = 0; j < V; ++j) {
                v[j] = total > 0 ? -(v[j] / total) * mean : A(0);
            }
        }
        for (uint32_t k = 0; k < count; ++k) {
            const int32_t c = __shfl(index, k);
            const A add = __shfl(part, k);
            for (int j = 0; j < V; ++j) {
                v[j] += c == static_cast<int32_t>(lane + 64 * j) ? add : A(0);
            }
        }
        for (int j = 0; j < V; ++j) {
            const uint32_t c = lane + 64 * j;
            if (c < classes) {
                gradients[row * gradientStride + c] = static_cast<T>(v[j]);
            }
        }
    }
}

}  // namespace op

using namespace op;

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
    constexpr uint32_t tileScores = 4096;
    a.SliceClasses = std::min<uint32_t>(a.Classes, tileScores);
    a.Slices = (a.Classes + a.SliceClasses - 1) / a.SliceClasses;
    a.RowsPerTile = a.Slices > 1 ? 1 : static_cast<uint32_t>(std::min<size_t>(rows, std::max<uint32_t>(1, tileScores / a.Classes)));
    a.Tiles = (rows + a.RowsPerTile - 1) / a.RowsPerTile * a.Slices;
    const TCallDevice call(result, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        const auto launch = [&](auto kernel) {
            call.Launch(kernel, std::min<size_t>(a.Tiles, 1u << 20), 256, tileScores * 4 * (size_t(history) + size_t(biases)), a);
        };
        if (history && biases) {
            launch(AdjustKernel<T, true, true>);
        } else if (history) {
            launch(AdjustKernel<T, true, false>);
        } else if (biases) {
            launch(AdjustKernel<T, false, true>);
        } else {
            launch(AdjustKernel<T, false, false>);
        }
    });
}

namespace {

constexpr size_t kMaxTopClasses = 1024;
constexpr int32_t kMaxTopCount = 32;

void CheckTop(size_t rows, size_t classes, int32_t count) {
    CBAMD_ENSURE(classes <= kMaxTopClasses, "too many classes to select from: " + std::to_string(classes) + ", at most " + std::to_string(kMaxTopClasses));
    CBAMD_ENSURE(count >= 1 && count <= kMaxTopCount, "selected classes per row: " + std::to_string(count) + ", 1 to " + std::to_string(kMaxTopCount) + " are supported");
    CBAMD_ENSURE(classes > 0 || rows == 0, "no classes to select from");
    CBAMD_ENSURE(rows <= size_t(1) << 48, "too many rows");
}

template <typename F>
void WithClasses(size_t classes, F&& f) {
    if (classes <= 64) {
        f(std::integral_constant<int, 1>());
    } else if (classes <= 128) {
        f(std::integral_constant<int, 2>());
    } else if (classes <= 256) {
        f(std::integral_constant<int, 4>());
    } else if (classes <= 512) {
        f(std::integral_constant<int, 8>());
    } else {
        f(std::integral_constant<int, 16>());
    }
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
        WithClasses(classes, [&](auto v) {
            call.Launch(SelectTopKernel<T, decltype(v)::value>, std::min<size_t>((rows + 3) / 4, 1u << 20), 256, 0, static_cast<const T*>(scores),
                        scoreStride, rows, static_cast<uint32_t>(classes), static_cast<uint32_t>(count), amongSelected, indexes,
                        static_cast<TAcc<T>*>(weights));
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
        WithClasses(classes, [&](auto v) {
            call.Launch(SelectTopBackwardKernel<T, decltype(v)::value>, std::min<size_t>((rows + 3) / 4, 1u << 20), 256, 0,
                        static_cast<const T*>(scores), scoreStride, rows, static_cast<uint32_t>(classes), static_cast<uint32_t>(count),
                        amongSelected, indexes, static_cast<const TAcc<T>*>(weights), static_cast<const TAcc<T>*>(weightGradients),
                        static_cast<T*>(scoreGradients), gradientStride);
        });
    });
}

}  // namespace cbamd
