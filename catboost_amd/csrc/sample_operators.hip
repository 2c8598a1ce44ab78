// A class of every row drawn by the softmax of its scores, of the classes that temperature, rank, share and least weight leave.
//
// All limits and the draw itself are positions in one order: best score first, of equal ones the lowest class first. A limit is a sum of
// weights from the front of that order, the draw is the first class whose sum passes uniform * the smallest of those sums. So no
// row is sorted: a position is found digit by digit, from sums of weights by the leading bits of the scores' keys. Weights are
// exp((x - best) / temperature) in 64 bits, added as whole numbers: sums do not depend on their order.
#include "operator_common.hip.h"

#include <algorithm>
#include <type_traits>

namespace cbamd {
namespace op {

// ---------------------------------------------------------------- keys and weights ----

// Keys grow with the scores; 0: minus infinity and NaN, which never take part. Both zeros have the same key.
template <typename T>
struct TKeys {
    using TBits = std::conditional_t<sizeof(T) == 8, uint64_t, std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>>;
    using TKey = std::conditional_t<sizeof(T) == 8, uint64_t, uint32_t>;
    static constexpr int kBits = sizeof(T) * 8;
    static constexpr TKey kSign = TKey(1) << (kBits - 1);

    __device__ __forceinline__ static TKey Of(T x) {
        const TKey b = __builtin_bit_cast(TBits, x);
        const TKey key = b == kSign ? kSign : b & kSign ? kSign - (b & (kSign - 1)) : b | kSign;
        const TKey lowest = kSign - Infinity();  // of minus infinity; NaN are under it, or over plus infinity
        return key > lowest && key <= (kSign | Infinity()) ? key - lowest : 0;
    }
    __device__ __forceinline__ static double Value(TKey key) {
        const TKey full = key + (kSign - Infinity());
        const TKey b = full & kSign ? full & (kSign - 1) : kSign | (kSign - full);
        return static_cast<double>(__builtin_bit_cast(T, static_cast<TBits>(b)));
    }

private:
    __device__ __forceinline__ static constexpr TKey Infinity() {
        return sizeof(T) == 8 ? TKey(0x7ff0000000000000ull) : sizeof(T) == 4 ? TKey(0x7f800000u) : std::is_same_v<T, _Float16> ? TKey(0x7c00u) : TKey(0x7f80u);
    }
};

// The weight of a score beside the row's best one
struct TWeigh {
    double Best, Rate;  // 1 / temperature
    double Unit;        // 2^shift: how many whole numbers a weight of 1 is

    __device__ __forceinline__ double Weight(double x) const {
        if (Best == __builtin_inf()) {
            return x == Best ? 1.0 : 0.0;
        }
        // (a difference of the largest scores may pass the largest number, which no temperature is to turn into NaN)
        return exp(fmax(x - Best, -1.7976931348623157e308) * Rate);
    }
    __device__ __forceinline__ uint64_t Whole(double weight) const {
        return static_cast<uint64_t>(weight * Unit + 0.5);
    }
};

// ---------------------------------------------------------------- one workgroup for a row ----

constexpr uint32_t kDigitBits = 11, kDigits = 1u << kDigitBits;

struct TDigitSums {
    uint64_t Weights[kDigits];
    uint32_t Counts[kDigits];
};

// Sums over a workgroup of WAVES waves; every lane gets them
template <int WAVES>
__device__ __forceinline__ uint64_t SumOf(uint64_t v, uint64_t* shared) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
        v += __shfl_xor(v, d);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        shared[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        v += shared[w];
    }
    return v;
}
template <int WAVES, typename TKey>
__device__ __forceinline__ TKey MostOf(TKey v, uint64_t* shared) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
        const TKey other = __shfl_xor(v, d);
        v = other > v ? other : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        shared[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const TKey other = static_cast<TKey>(shared[w]);
        v = other > v ? other : v;
    }
    return v;
}

// f(score, class) for this thread's scores of a row, 16 bytes at a time
template <typename T, int THREADS, typename F>
__device__ __forceinline__ void ForRow(const T* row, uint32_t classes, F&& f) {
    constexpr uint32_t N = 16 / sizeof(T);
    const uint32_t whole = classes / N;
    for (uint32_t c = threadIdx.x; c < whole; c += THREADS) {
        const auto v = TValues<T, N>::Load(row + c * N);
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
            f(v.V[i], c * N + i);
        }
    }
    for (uint32_t c = whole * N + threadIdx.x; c < classes; c += THREADS) {
        f(row[c], c);
    }
}

// A position in a row's order: the key there, how many classes and which weights are before those of that key
template <typename TKey>
struct TPosition {
    TKey Key;
    uint32_t Before, Alike;
    uint64_t WeightBefore;
};

struct TSampleArguments {
    size_t First;  // row of the launch
    uint32_t Classes;
    uint32_t Shift;  // whole numbers of a weight of 1: 2^Shift
    size_t Stride;
    CbHipSampling Sampling;
    const float* Uniform;
    int32_t* Indexes;
    void* Weights;
};

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) SampleRowKernel(const T* scores, TSampleArguments p) {
    using TK = TKeys<T>;
    using TKey = typename TK::TKey;
    constexpr int kWaves = THREADS / 64;
    constexpr uint32_t kMine = kDigits / THREADS;
    __shared__ TDigitSums first, later;
    __shared__ uint64_t shared[kWaves];
    __shared__ uint64_t found[4];
    __shared__ uint32_t counted[kWaves];

    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t r = p.First + blockIdx.x;
    const T* row = scores + r * p.Stride;
    const uint32_t classes = p.Classes;

    TKey most = 0;
    ForRow<T, THREADS>(row, classes, [&](T x, uint32_t) {
        const TKey key = TK::Of(x);
        most = key > most ? key : most;
    });
    most = MostOf<kWaves>(most, shared);
    const auto answer = [&](int32_t index, double weight) {
        if (threadIdx.x == 0) {
            p.Indexes[r] = index;
            if (p.Weights != nullptr) {
                static_cast<TAcc<T>*>(p.Weights)[r] = static_cast<TAcc<T>>(weight);
            }
        }
    };
    if (most == 0) {
        answer(-1, 0);
        return;
    }

    // the lowest class of the (nth + 1)-th of those with this key
    const auto classOf = [&](TKey key, uint32_t nth) {
        // which wave's part of the row has it, then which of the part's 64 * pieces classes
        const uint32_t part = (classes + kWaves - 1) / kWaves;
        uint32_t begin = wave * part, end = begin + part < classes ? begin + part : classes, n = 0;
        for (uint32_t c = begin + lane; c < end; c += 64) {
            n += TK::Of(row[c]) == key;
        }
#pragma unroll
        for (int d = 32; d > 0; d /= 2) {
            n += __shfl_xor(n, d);
        }
        __syncthreads();
        if (lane == 0) {
            counted[wave] = n;
        }
        __syncthreads();
        uint32_t w = 0;
        while (w + 1 < kWaves && nth >= counted[w]) {
            nth -= counted[w++];
        }
        begin = w * part;
        end = begin + part < classes ? begin + part : classes;
        // every thread of the workgroup has some classes in a row of that part
        const uint32_t each = (part + THREADS - 1) / THREADS;
        const uint32_t mine = begin + threadIdx.x * each, last = mine + each < end ? mine + each : end;
        n = 0;
        for (uint32_t c = mine; c < last; ++c) {
            n += TK::Of(row[c]) == key;
        }
        uint32_t sum = n;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t other = __shfl_up(sum, d);
            sum += lane >= static_cast<uint32_t>(d) ? other : 0;
        }
        __syncthreads();
        if (lane == 63) {
            counted[wave] = sum;
        }
        __syncthreads();
        uint32_t before = sum - n;
        for (uint32_t v = 0; v < wave; ++v) {
            before += counted[v];
        }
        if (nth >= before && nth < before + n) {
            for (uint32_t c = mine; c < last; ++c) {
                if (TK::Of(row[c]) == key && before++ == nth) {
                    found[0] = c;
                }
            }
        }
        __syncthreads();
        return static_cast<int32_t>(found[0]);
    };

    const float temperature = p.Sampling.Temperature != nullptr ? p.Sampling.Temperature[r] : 1.0f;
    if (!(temperature > 0)) {
        const int32_t index = classOf(most, 0);
        answer(index, 1);
        return;
    }
    const TWeigh weigh{TK::Value(most), 1.0 / static_cast<double>(temperature), static_cast<double>(uint64_t(1) << p.Shift)};
    const float least = p.Sampling.MinP != nullptr ? p.Sampling.MinP[r] : 0.0f;
    const double minP = least > 0 ? (least < 1 ? least : 1.0) : 0.0;

    // sums by the first digit of how far a key is under the best one, and the limits that need nothing else
    constexpr int kLevels = (TK::kBits + kDigitBits - 1) / kDigitBits;
    constexpr uint32_t kTop = (kLevels - 1) * kDigitBits;
    for (uint32_t d = threadIdx.x; d < kDigits; d += THREADS) {
        first.Weights[d] = 0;
        first.Counts[d] = 0;
    }
    __syncthreads();
    uint64_t all = 0, likely = 0, there = 0;
    ForRow<T, THREADS>(row, classes, [&](T x, uint32_t) {
        const TKey key = TK::Of(x);
        if (key != 0) {
            const double weight = weigh.Weight(static_cast<double>(x));
            const uint64_t whole = weigh.Whole(weight);
            ++there;
            all += whole;
            likely += weight >= minP ? whole : 0;
            const uint32_t digit = static_cast<uint32_t>((most - key) >> kTop);
            atomicAdd(reinterpret_cast<unsigned long long*>(&first.Weights[digit]), static_cast<unsigned long long>(whole));
            atomicAdd(&first.Counts[digit], 1u);
        }
    });
    all = SumOf<kWaves>(all, shared);
    likely = SumOf<kWaves>(likely, shared);
    there = SumOf<kWaves>(there, shared);

    // The position where the count (byCount) or the weights from the front of the order, its own among them, reach `target`, which
    // they do somewhere
    const auto reach = [&](bool byCount, uint64_t target) {
        TPosition<TKey> at{0, 0, 0, 0};
        TKey prefix = 0;  // the digits so far
        for (int level = kLevels - 1; level >= 0; --level) {
            const uint32_t shift = level * kDigitBits;
            TDigitSums& sums = level == kLevels - 1 ? first : later;
            if (level < kLevels - 1) {
                __syncthreads();
                for (uint32_t d = threadIdx.x; d < kDigits; d += THREADS) {
                    later.Weights[d] = 0;
                    later.Counts[d] = 0;
                }
                __syncthreads();
                ForRow<T, THREADS>(row, classes, [&](T x, uint32_t) {
                    const TKey key = TK::Of(x), under = most - key;
                    if (key != 0 && under >> (shift + kDigitBits) == prefix) {
                        const uint32_t digit = static_cast<uint32_t>(under >> shift) & (kDigits - 1);
                        atomicAdd(reinterpret_cast<unsigned long long*>(&later.Weights[digit]),
                                  static_cast<unsigned long long>(weigh.Whole(weigh.Weight(static_cast<double>(x)))));
                        atomicAdd(&later.Counts[digit], 1u);
                    }
                });
            }
            __syncthreads();
            // every thread has kMine digits in a row
            uint64_t mine = 0;
            const uint32_t begin = threadIdx.x * kMine;
            for (uint32_t d = begin; d < begin + kMine; ++d) {
                mine += byCount ? sums.Counts[d] : sums.Weights[d];
            }
            uint64_t sum = mine;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const uint64_t other = __shfl_up(sum, d);
                sum += lane >= static_cast<uint32_t>(d) ? other : 0;
            }
            if (lane == 63) {
                shared[wave] = sum;
            }
            __syncthreads();
            uint64_t before = (byCount ? at.Before : at.WeightBefore) + sum - mine;
            for (uint32_t w = 0; w < wave; ++w) {
                before += shared[w];
            }
            if (before < target && before + mine >= target) {
                uint32_t d = begin;
                for (; d + 1 < begin + kMine; ++d) {
                    const uint64_t more = byCount ? sums.Counts[d] : sums.Weights[d];
                    if (before + more >= target) {
                        break;
                    }
                    before += more;
                }
                found[0] = d;
                found[1] = before;
            }
            __syncthreads();
            const uint32_t digit = static_cast<uint32_t>(found[0]);
            // the other sum before that digit
            uint64_t rest = 0;
            for (uint32_t d = threadIdx.x; d < digit; d += THREADS) {
                rest += byCount ? sums.Weights[d] : sums.Counts[d];
            }
            const uint64_t reached = found[1];
            rest = SumOf<kWaves>(rest, shared);
            if (byCount) {
                at.Before = static_cast<uint32_t>(reached);
                at.WeightBefore += rest;
            } else {
                at.Before += static_cast<uint32_t>(rest);
                at.WeightBefore = reached;
            }
            at.Alike = sums.Counts[digit];
            prefix = prefix << kDigitBits | digit;
        }
        at.Key = most - prefix;
        return at;
    };
    const auto wholeOf = [&](TKey key) { return weigh.Whole(weigh.Weight(TK::Value(key))); };

    // what the limits leave, as sums from the front of the order: the smallest holds
    const int32_t topK = p.Sampling.TopK != nullptr ? p.Sampling.TopK[r] : 0;
    if (topK > 0 && static_cast<uint64_t>(topK) < there) {
        const auto at = reach(true, static_cast<uint64_t>(topK));
        all = at.WeightBefore + (static_cast<uint32_t>(topK) - at.Before) * wholeOf(at.Key);
    }
    uint64_t kept = all < likely ? all : likely;
    const float topP = p.Sampling.TopP != nullptr ? p.Sampling.TopP[r] : 1.0f;
    if (topP < 1) {
        const double share = ceil((topP > 0 ? static_cast<double>(topP) : 0.0) * static_cast<double>(all));
        const uint64_t target = share < 1 ? 1 : share < static_cast<double>(all) ? static_cast<uint64_t>(share) : all;
        const auto at = reach(false, target);
        const uint64_t whole = wholeOf(at.Key);
        const uint64_t sum = at.WeightBefore + ((target - at.WeightBefore + whole - 1) / whole) * whole;
        kept = sum < kept ? sum : kept;
    }
    const float uniform = p.Uniform[r];
    const double passed = (uniform > 0 ? static_cast<double>(uniform) : 0.0) * static_cast<double>(kept);
    const uint64_t draw = passed < static_cast<double>(kept) && static_cast<uint64_t>(passed) < kept ? static_cast<uint64_t>(passed) : kept - 1;
    const auto at = reach(false, draw + 1);
    const double weight = weigh.Weight(TK::Value(at.Key));
    const int32_t index = classOf(at.Key, static_cast<uint32_t>((draw - at.WeightBefore) / weigh.Whole(weight)));
    answer(index, weight * weigh.Unit / static_cast<double>(kept));
}

}  // namespace op

using namespace op;

namespace {

constexpr size_t kMostClassesToSample = size_t(1) << 24;
constexpr size_t kMostRowsOfLaunch = size_t(1) << 21;

}  // namespace

size_t SampleClassesBytes(int, size_t, size_t) {
    return 0;
}

void SampleClasses(int valueType, size_t rows, size_t classes, const void* scores, size_t scoreStride, const CbHipSampling& sampling,
                   const float* uniform, int32_t* indexes, void* weights, void* workspace, size_t workspaceBytes, void* stream) {
    const size_t size = ValueSize(valueType);
    if (rows == 0) {
        return;
    }
    CBAMD_ENSURE(classes > 0, "no classes to draw from");
    CBAMD_ENSURE(classes <= kMostClassesToSample, "too many classes: " + std::to_string(classes) + ", at most " + std::to_string(kMostClassesToSample) + " are supported");
    CBAMD_ENSURE(rows <= size_t(1) << 40, "too many rows");
    CheckMatrix("scores", scores, rows, classes, scoreStride, size);
    CBAMD_ENSURE(uniform != nullptr, "uniform pointer is null");
    CBAMD_ENSURE(indexes != nullptr, "indexes pointer is null");
    const TCallDevice call(indexes, stream);
    TSampleArguments p{};
    p.Classes = static_cast<uint32_t>(classes);
    // a row of the best score alone adds up to under 2^63
    p.Shift = 62;
    while (p.Shift > 0 && (size_t(1) << (63 - p.Shift)) <= classes) {
        --p.Shift;
    }
    p.Stride = scoreStride;
    p.Sampling = sampling;
    p.Uniform = uniform;
    p.Indexes = indexes;
    p.Weights = weights;
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        for (p.First = 0; p.First < rows; p.First += kMostRowsOfLaunch) {
            const size_t n = std::min(rows - p.First, kMostRowsOfLaunch);
            if (classes <= 4096) {
                call.Launch(SampleRowKernel<T, 256>, n, 256, 0, static_cast<const T*>(scores), p);
            } else {
                call.Launch(SampleRowKernel<T, 1024>, n, 1024, 0, static_cast<const T*>(scores), p);
            }
        }
    });
}

}  // namespace cbamd
