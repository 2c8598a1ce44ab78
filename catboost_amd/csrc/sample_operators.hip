// A class of every row drawn by the softmax of its scores, of the classes that temperature, rank, share and least weight leave.
//
// All limits and the draw itself are positions in one order: best score first, of equal ones the lowest class first. A limit is a sum of
// weights from the front of that order, the draw is the first class whose sum passes uniform * the smallest of those sums. Weights are
// 2^-t, t = (best - x) / temperature * log2(e), in 64 bits, added as whole numbers: sums do not depend on their order, so a class is the
// same whichever way it is found. Short rows are sorted, in a thread's registers or a wave's; of long ones only the sums of weights
// around the positions are needed: by how often each key comes (16 bits), or by t and then by the keys of the part where a
// position is.
#include "operator_common.hip.h"

#include <algorithm>
#include <limits>
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

constexpr uint32_t kPowers = 64;  // (shifts by 6 below)

// 2^(-i / 64), which a workgroup computes for its weights
__device__ __forceinline__ void FillPowers(double* powers) {
    if (threadIdx.x < kPowers) {
        powers[threadIdx.x] = exp2(static_cast<double>(threadIdx.x) * -0.015625);
    }
}

// The weights of a row's scores
template <bool TABLE>
struct TWeigh {
    double Best;           // the best score
    double Rate;           // log2(e) / temperature
    double Unit;           // 2^shift: how many whole numbers a weight of 1 is, at most 2^51 (what Whole takes)
    const double* Powers;  // in LDS, of TABLE

    // How far under the best one, in powers of two; never less for a smaller score. All of plus infinity are alike, and the others
    // too far under it (a difference that is no number counts as 4096).
    template <typename T>
    __device__ __forceinline__ double Under(T x) const {
        double under = Best - static_cast<double>(x);
        if constexpr (std::is_same_v<T, double>) {
            // (may pass the largest number, which no temperature is to turn into NaN)
            under = Best < __builtin_inf() ? fmin(under, 1.7976931348623157e308) : under;
        }
        under = fmin(under * Rate, 4096.0);
        return static_cast<double>(x) == Best ? 0.0 : under;
    }
    // 2^-under. With the table the rest beside the nearest 64th is under 1/128 and the series of exp ends with its fifth power (the
    // sixth is under 2^-54): a third of the steps of exp, which is most of what a row of 100000 classes costs. Where a workgroup has
    // few weights to compute the rest beside the nearest whole number is up to 1/2, and the series has 13.
    __device__ __forceinline__ double Weight(double under) const {
        if constexpr (TABLE) {
            const double steps = rint(under * kPowers);
            const double y = fma(steps, 1.0 / kPowers, -under) * 0.69314718055994530942;
            const int n = static_cast<int>(steps);
            double e = fma(y, 1.0 / 120, 1.0 / 24);
            e = fma(e, y, 1.0 / 6);
            e = fma(e, y, 0.5);
            e = fma(e, y, 1.0);
            e = fma(e, y, 1.0);
            return ldexp(e * Powers[n & (kPowers - 1)], -(n >> 6));
        } else {
            const double steps = rint(under);
            const double y = (steps - under) * 0.69314718055994530942;
            double e = 1.0 / 6227020800.0;
            constexpr double kTerms[] = {1.0 / 479001600, 1.0 / 39916800, 1.0 / 3628800, 1.0 / 362880, 1.0 / 40320, 1.0 / 5040, 1.0 / 720, 1.0 / 120, 1.0 / 24, 1.0 / 6, 0.5, 1.0, 1.0};
#pragma unroll
            for (const double term : kTerms) {
                e = fma(e, y, term);
            }
            return ldexp(e, -static_cast<int>(steps));
        }
    }
    // (what adding 2^52 leaves in the last bits is the nearest whole number)
    __device__ __forceinline__ uint64_t Whole(double weight) const {
        return __builtin_bit_cast(uint64_t, fma(weight, Unit, 4503599627370496.0)) & 0xfffffffffffffull;
    }
    template <typename T>
    __device__ __forceinline__ uint64_t WholeOf(T x) const {
        return Whole(Weight(Under(x)));
    }
};

constexpr uint32_t kMostBits = 51;  // of a weight (see Whole)

// Arguments of a launch, and what they say of a row
struct TSampleArguments {
    size_t First, Rows;  // of the launch
    uint32_t Classes;
    uint32_t Shift;

    // Whole numbers of 2^-Shift leave room for a row of nothing but best scores. What they round away, half of one for each class at most, is
    // under 2^-28 of the sum up to 2^18 classes and in any flat row. Of other rows the weights are added a second time (1M f32 classes
    // 678 us for eight rows, 429 without), in as many more bits as the sum leaves: with the roundings of both it stays under 2^63. Before,
    // draws of 4M classes passed over 2^-20 of a row.
    __device__ __forceinline__ uint32_t MoreBits(uint64_t all) const {
        const uint32_t room = all >> 27 >= Classes ? 0 : __clzll(static_cast<long long>(all + Classes));
        return room < 2 ? 0 : room - 2 < kMostBits - Shift ? room - 2 : kMostBits - Shift;
    }
    size_t Stride;
    CbHipSampling Sampling;
    const float* Uniform;
    int32_t* Indexes;
    void* Weights;
};

struct TLimits {
    float Temperature, TopP, Uniform;
    int32_t TopK;
    double MinP;

    __device__ __forceinline__ TLimits(const TSampleArguments& p, size_t r)
        : Temperature(p.Sampling.Temperature != nullptr ? p.Sampling.Temperature[r] : 1.0f)
        , TopP(p.Sampling.TopP != nullptr ? p.Sampling.TopP[r] : 1.0f)
        , Uniform(p.Uniform[r])
        , TopK(p.Sampling.TopK != nullptr ? p.Sampling.TopK[r] : 0)
    {
        const float least = p.Sampling.MinP != nullptr ? p.Sampling.MinP[r] : 0.0f;
        MinP = least > 0 ? (least < 1 ? static_cast<double>(least) : 1.0) : 0.0;
    }
    __device__ __forceinline__ bool Greedy() const {
        return !(Temperature > 0);
    }
    template <bool TABLE>
    __device__ __forceinline__ TWeigh<TABLE> Weigh(double best, uint32_t shift, const double* powers) const {
        return {best, 1.44269504088896340736 / static_cast<double>(Temperature), static_cast<double>(uint64_t(1) << shift), powers};
    }
    // The sum that the classes of the share reach first, of `all`
    __device__ __forceinline__ uint64_t ShareOf(uint64_t all) const {
        const double share = ceil((TopP > 0 ? static_cast<double>(TopP) : 0.0) * static_cast<double>(all));
        return share < 1 ? 1 : share < static_cast<double>(all) ? static_cast<uint64_t>(share) : all;
    }
    // The sum that the drawn class is the first to reach, of those kept
    __device__ __forceinline__ uint64_t DrawOf(uint64_t kept) const {
        const double passed = (Uniform > 0 ? static_cast<double>(Uniform) : 0.0) * static_cast<double>(kept);
        return (passed < static_cast<double>(kept) && static_cast<uint64_t>(passed) < kept ? static_cast<uint64_t>(passed) : kept - 1) + 1;
    }
};

template <typename T>
__device__ __forceinline__ void Answer(const TSampleArguments& p, size_t r, int32_t index, double weight) {
    p.Indexes[r] = index;
    if (p.Weights != nullptr) {
        static_cast<TAcc<T>*>(p.Weights)[r] = static_cast<TAcc<T>>(weight);
    }
}

// ---------------------------------------------------------------- a thread for a row ----

// Rows of exactly C classes, sorted in registers by neighbours that trade places, which keeps equal ones in order
template <typename T, int C>
__global__ void __launch_bounds__(256) SampleOfFewKernel(const T* scores, TSampleArguments p) {
    using A = TAcc<T>;
    __shared__ double powers[kPowers];
    FillPowers(powers);
    __syncthreads();
    const size_t n = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    if (n >= p.Rows) {
        return;
    }
    const size_t r = p.First + n;
    const T* row = scores + r * p.Stride;
    constexpr A kNone = -std::numeric_limits<A>::infinity();
    A x[C];
    int32_t index[C];
    constexpr int N = std::min<int>(C, 16 / sizeof(T));
#pragma unroll
    for (int c = 0; c < C; c += N) {
        // (a last piece that overlaps the one before it)
        const int from = c + N <= C ? c : C - N;
        const auto v = TValues<T, N>::Load(row + from);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const A value = static_cast<A>(v.V[i]);
            x[from + i] = value == value ? value + A(0) : kNone;  // (one zero of both)
        }
    }
    const TLimits limits(p, r);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        index[c] = c;
    }
#pragma unroll
    for (int round = 0; round < C; ++round) {
#pragma unroll
        for (int c = 0; c + 1 < C; ++c) {
            if ((c & 1) != (round & 1)) {
                continue;
            }
            // (values of their own: a choice between elements would be one between addresses, and the rows would leave their registers)
            const A a = x[c], b = x[c + 1];
            const int32_t i = index[c], j = index[c + 1];
            const bool trade = b > a;
            x[c] = trade ? b : a;
            x[c + 1] = trade ? a : b;
            index[c] = trade ? j : i;
            index[c + 1] = trade ? i : j;
        }
    }
    if (x[0] == kNone) {
        return Answer<T>(p, r, -1, 0);
    }
    if (limits.Greedy()) {
        return Answer<T>(p, r, index[0], 1);
    }
    const auto weigh = limits.Weigh<true>(static_cast<double>(x[0]), p.Shift, powers);
    double weight[C];
    uint64_t sum[C], all = 0, likely = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const double w = weigh.Weight(weigh.Under(x[c]));
        weight[c] = x[c] > kNone ? w : 0.0;
        const uint64_t whole = weigh.Whole(weight[c]);
        all += limits.TopK <= 0 || c < limits.TopK ? whole : 0;
        likely += weight[c] >= limits.MinP ? whole : 0;
        sum[c] = (c > 0 ? sum[c > 0 ? c - 1 : 0] : 0) + whole;
    }
    uint64_t kept = all < likely ? all : likely;
    if (p.Sampling.TopP != nullptr) {
        const uint64_t target = limits.ShareOf(all);
        uint64_t reached = all;
#pragma unroll
        for (int c = C - 1; c >= 0; --c) {
            const uint64_t here = sum[c];
            reached = here >= target ? here : reached;
        }
        kept = limits.TopP < 1 && reached < kept ? reached : kept;
    }
    const uint64_t target = limits.DrawOf(kept);
    int32_t found = index[C - 1];
    double foundWeight = weight[C - 1];
#pragma unroll
    for (int c = C - 2; c >= 0; --c) {
        const int32_t here = index[c];
        const double hereWeight = weight[c];
        const bool there = sum[c] >= target;
        found = there ? here : found;
        foundWeight = there ? hereWeight : foundWeight;
    }
    Answer<T>(p, r, found, foundWeight * weigh.Unit / static_cast<double>(kept));
}

// ---------------------------------------------------------------- lanes for a row ----

// The sum over the lanes up to this one. Steps are moves within the vector unit (rows of 16 lanes, then from the last lane of a row to the
// next rows), a tenth of the time of trips through LDS.
template <int CONTROL, int ROWS, typename V>
__device__ __forceinline__ V MovedOver(V v) {
    if constexpr (sizeof(V) == 8) {
        const uint32_t low = __builtin_amdgcn_update_dpp(0u, static_cast<uint32_t>(v), CONTROL, ROWS, 0xf, false);
        const uint32_t high = __builtin_amdgcn_update_dpp(0u, static_cast<uint32_t>(v >> 32), CONTROL, ROWS, 0xf, false);
        return static_cast<V>(high) << 32 | low;
    } else {
        return __builtin_amdgcn_update_dpp(0u, v, CONTROL, ROWS, 0xf, false);
    }
}
template <typename V>
__device__ __forceinline__ V SumUpTo(V v) {
    v += MovedOver<0x111, 0xf>(v);  // 1, 2, 4, 8 lanes on in a row
    v += MovedOver<0x112, 0xf>(v);
    v += MovedOver<0x114, 0xf>(v);
    v += MovedOver<0x118, 0xf>(v);
    v += MovedOver<0x142, 0xa>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
    v += MovedOver<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
    return v;
}
template <typename V>
__device__ __forceinline__ V OfLane(V v, int lane) {
    if constexpr (sizeof(V) == 8) {
        const uint32_t low = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane), high = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane);
        return static_cast<V>(high) << 32 | low;
    } else {
        return __builtin_amdgcn_readlane(v, lane);
    }
}
// The largest of the wave's
template <typename V>
__device__ __forceinline__ V MostOfWave(V v) {
    const auto larger = [&](V other) { v = other > v ? other : v; };
    larger(MovedOver<0x111, 0xf>(v));
    larger(MovedOver<0x112, 0xf>(v));
    larger(MovedOver<0x114, 0xf>(v));
    larger(MovedOver<0x118, 0xf>(v));
    larger(MovedOver<0x142, 0xa>(v));
    larger(MovedOver<0x143, 0xc>(v));
    return OfLane(v, 63);
}

// The value of the lane that differs in this bit: moves within the vector unit where rows of 16 lanes have both (trips through LDS take
// half as long again for a whole sort: 250000 x 64 f64 310 us, 202)
template <int LANES, typename V>
__device__ __forceinline__ V AcrossLanes(V v) {
    if constexpr (sizeof(V) == 8) {
        return static_cast<V>(AcrossLanes<LANES>(static_cast<uint32_t>(v >> 32))) << 32 | AcrossLanes<LANES>(static_cast<uint32_t>(v));
    } else if constexpr (LANES == 1) {
        return __builtin_amdgcn_update_dpp(0u, v, 0xb1, 0xf, 0xf, true);
    } else if constexpr (LANES == 2) {
        return __builtin_amdgcn_update_dpp(0u, v, 0x4e, 0xf, 0xf, true);
    } else if constexpr (LANES == 4) {
        // (eight lanes the other way round, then each four of them)
        return __builtin_amdgcn_update_dpp(0u, __builtin_amdgcn_update_dpp(0u, v, 0x141, 0xf, 0xf, true), 0x1b, 0xf, 0xf, true);
    } else if constexpr (LANES == 8) {
        return __builtin_amdgcn_update_dpp(0u, v, 0x128, 0xf, 0xf, true);
    } else {
        return __shfl_xor(v, LANES);
    }
}

// A key and its class as one value that orders them, the lowest class first: 32 bits for 16-bit scores, 64 for 32-bit ones
template <typename T>
struct TOrdered {
    using TKey = typename TKeys<T>::TKey;
    using TWord = std::conditional_t<sizeof(T) == 2, uint32_t, uint64_t>;
    TWord Word;

    __device__ __forceinline__ static TOrdered Of(TKey key, uint32_t index) {
        constexpr int kShift = sizeof(T) == 2 ? 16 : 32;
        return {static_cast<TWord>(key) << kShift | (~index & static_cast<uint32_t>((TWord(1) << kShift) - 1))};
    }
    __device__ __forceinline__ TKey Key() const {
        return static_cast<TKey>(Word >> (sizeof(T) == 2 ? 16 : 32));
    }
    __device__ __forceinline__ uint32_t Index() const {
        return ~static_cast<uint32_t>(Word) & (sizeof(T) == 2 ? 0xffffu : ~0u);
    }
    __device__ __forceinline__ bool Before(const TOrdered& other) const {
        return Word > other.Word;
    }
    __device__ __forceinline__ static TOrdered Choose(bool first, const TOrdered& a, const TOrdered& b) {
        return {first ? a.Word : b.Word};
    }
    template <int LANES>
    __device__ __forceinline__ TOrdered Across() const {
        return {AcrossLanes<LANES>(Word)};
    }
};
template <>
struct TOrdered<double> {
    uint64_t Word;
    uint32_t Class;

    __device__ __forceinline__ static TOrdered Of(uint64_t key, uint32_t index) {
        return {key, index};
    }
    __device__ __forceinline__ uint64_t Key() const {
        return Word;
    }
    __device__ __forceinline__ uint32_t Index() const {
        return Class;
    }
    __device__ __forceinline__ bool Before(const TOrdered& other) const {
        return (Word > other.Word) | ((Word == other.Word) & (Class < other.Class));
    }
    // (member by member: a choice between structs went by way of memory, ten times as slow)
    __device__ __forceinline__ static TOrdered Choose(bool first, const TOrdered& a, const TOrdered& b) {
        return {first ? a.Word : b.Word, first ? a.Class : b.Class};
    }
    template <int LANES>
    __device__ __forceinline__ TOrdered Across() const {
        return {AcrossLanes<LANES>(Word), AcrossLanes<LANES>(Class)};
    }
};

// Places lane * P + i in order: runs of SIZE places, each the other way round than the next, are merged to ones of twice that, by
// trades between places STEP apart
template <int LANES, int P, int SIZE, int STEP, typename TItem>
__device__ __forceinline__ void Merge(TItem (&item)[P], uint32_t lane) {
    if constexpr (STEP >= P) {
        const bool low = (lane & (STEP / P)) == 0, down = (lane * P & SIZE) == 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const TItem other = item[i].template Across<STEP / P>();
            item[i] = TItem::Choose(item[i].Before(other) == (low == down), item[i], other);
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if ((i & STEP) == 0) {
                const bool down = ((lane * P + i) & SIZE) == 0;
                const TItem a = item[i], b = item[i + STEP];
                const bool trade = a.Before(b) != down;
                item[i] = TItem::Choose(trade, b, a);
                item[i + STEP] = TItem::Choose(trade, a, b);
            }
        }
    }
    if constexpr (STEP > 1) {
        Merge<LANES, P, SIZE, STEP / 2>(item, lane);
    } else if constexpr (SIZE < LANES * P) {
        Merge<LANES, P, SIZE * 2, SIZE>(item, lane);
    }
}

// Rows of at most LANES * P classes: place i of the order ends up as value i % P of lane i / P
template <typename T, int LANES, int P>
__global__ void __launch_bounds__(256) SampleByLanesKernel(const T* scores, TSampleArguments p) {
    using TK = TKeys<T>;
    using TItem = TOrdered<T>;
    const uint32_t lane = threadIdx.x % LANES;
    const size_t n = static_cast<size_t>(blockIdx.x) * (256 / LANES) + threadIdx.x / LANES;
    // (rows behind the last one do as it does, so that every lane is there to be read, and store nothing)
    const size_t r = p.First + (n < p.Rows ? n : p.Rows - 1);
    const T* row = scores + r * p.Stride;
    const TLimits limits(p, r);
    TItem item[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const uint32_t c = lane + i * LANES;
        item[i] = TItem::Of(c < p.Classes ? TK::Of(row[c]) : 0, c);
    }
    Merge<LANES, P, 2, 1>(item, lane);
    const bool mine = n < p.Rows && lane == 0;
    const uint32_t base = threadIdx.x & 63 & ~(LANES - 1);  // the row's first lane in its wave
    const TItem best{item[0]};
    const auto bestKey = __shfl(best.Key(), base);
    const uint32_t bestClass = __shfl(best.Index(), base);
    if (bestKey == 0 || limits.Greedy()) {
        if (mine) {
            Answer<T>(p, r, bestKey == 0 ? -1 : static_cast<int32_t>(bestClass), bestKey == 0 ? 0 : 1);
        }
    }
    // (every lane goes on: rows of a wave differ; the values of such a row are not used)
    auto weigh = limits.Weigh<false>(TK::Value(bestKey), p.Shift, nullptr);
    weigh.Rate = limits.Greedy() ? 0 : weigh.Rate;
    double weight[P];
    uint64_t sum[P], all = 0, likely = 0, total = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const auto key = item[i].Key();
        const double w = weigh.Weight(weigh.Under(static_cast<T>(TK::Value(key))));
        weight[i] = key != 0 ? w : 0.0;
        const uint64_t whole = weigh.Whole(weight[i]);
        all += limits.TopK <= 0 || lane * P + i < static_cast<uint32_t>(limits.TopK) ? whole : 0;
        likely += weight[i] >= limits.MinP ? whole : 0;
        total += whole;
        sum[i] = total;
    }
    uint64_t before = total;
    if constexpr (LANES == 64) {
        before = SumUpTo(total);
        all = limits.TopK > 0 ? OfLane(SumUpTo(all), 63) : OfLane(before, 63);
        likely = OfLane(SumUpTo(likely), 63);
    } else {
#pragma unroll
        for (int d = 1; d < LANES; d *= 2) {
            const uint64_t other = __shfl_up(before, d, LANES);
            const uint64_t otherAll = __shfl_xor(all, d), otherLikely = __shfl_xor(likely, d);
            before += lane >= static_cast<uint32_t>(d) ? other : 0;
            all += otherAll;
            likely += otherLikely;
        }
    }
    before -= total;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        sum[i] += before;
    }
    // the value at the place that reaches a sum first
    const auto at = [&](uint64_t target, auto&& valueOf) {
        const uint64_t there = __ballot(before < target && sum[P - 1] >= target);
        auto value = valueOf(P - 1);
#pragma unroll
        for (int i = P - 2; i >= 0; --i) {
            value = sum[i] >= target ? valueOf(i) : value;
        }
        const uint64_t ofRow = LANES == 64 ? there : there >> base & ((uint64_t(1) << (LANES & 63)) - 1);
        return __shfl(value, base + (ofRow != 0 ? __ffsll(static_cast<unsigned long long>(ofRow)) - 1 : 0));
    };
    uint64_t kept = all < likely ? all : likely;
    if (p.Sampling.TopP != nullptr) {
        const uint64_t reached = at(limits.ShareOf(all), [&](int i) { return sum[i]; });
        kept = limits.TopP < 1 && reached < kept ? reached : kept;
    }
    const uint64_t target = limits.DrawOf(kept);
    const uint32_t index = at(target, [&](int i) { return item[i].Index(); });
    const double foundWeight = at(target, [&](int i) { return weight[i]; });
    if (mine && bestKey != 0 && !limits.Greedy()) {
        Answer<T>(p, r, static_cast<int32_t>(index), foundWeight * weigh.Unit / static_cast<double>(kept));
    }
}

// ---------------------------------------------------------------- a workgroup for a row ----

// Sums by a digit of BITS bits
template <int BITS>
struct TDigitSums {
    uint64_t Weights[1 << BITS];
    uint32_t Counts[1 << BITS];

    template <int THREADS>
    __device__ __forceinline__ void Clear() {
        for (uint32_t d = threadIdx.x; d < 1u << BITS; d += THREADS) {
            Weights[d] = 0;
            Counts[d] = 0;
        }
    }
    __device__ __forceinline__ void Add(uint32_t digit, uint64_t weight) {
        atomicAdd(reinterpret_cast<unsigned long long*>(&Weights[digit]), static_cast<unsigned long long>(weight));
        atomicAdd(&Counts[digit], 1u);
    }
};

// What the waves of a workgroup hand each other
template <int WAVES>
struct TShared {
    uint64_t Sums[WAVES];
    uint64_t Found[4];
    uint32_t Counted[WAVES];
    uint32_t Listed;
    double Powers[kPowers];
};

// Sums and maxima over a workgroup; every lane gets them
template <int WAVES>
__device__ __forceinline__ uint64_t SumOf(uint64_t v, TShared<WAVES>& shared) {
    v = SumUpTo(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) {
        shared.Sums[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        v += shared.Sums[w];
    }
    return v;
}
template <int WAVES, typename TKey>
__device__ __forceinline__ TKey MostOf(TKey v, TShared<WAVES>& shared) {
    v = MostOfWave(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        shared.Sums[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const TKey other = static_cast<TKey>(shared.Sums[w]);
        v = other > v ? other : v;
    }
    return v;
}
// The sums over the threads before this one
template <int WAVES>
__device__ __forceinline__ void SumBefore(uint64_t& weights, uint32_t& counts, TShared<WAVES>& shared) {
    const uint32_t wave = threadIdx.x >> 6;
    const uint64_t sum = SumUpTo(weights);
    const uint32_t counted = SumUpTo(counts);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) {
        shared.Sums[wave] = sum;
        shared.Counted[wave] = counted;
    }
    __syncthreads();
    weights = sum - weights;
    counts = counted - counts;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) {
        weights += w < wave ? shared.Sums[w] : 0;
        counts += w < wave ? shared.Counted[w] : 0;
    }
}

// f(score, class) for this thread's scores of a row, 16 bytes at a time, four of them on their way
template <typename T, int THREADS, typename F>
__device__ __forceinline__ void ForRow(const T* row, uint32_t classes, F&& f) {
    constexpr uint32_t N = 16 / sizeof(T);
    const uint32_t whole = classes / N;
    for (uint32_t c = threadIdx.x; c < whole; c += 4 * THREADS) {
        TValues<T, N> v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (behind the end the last ones again, so that no load waits in a branch)
            v[j] = TValues<T, N>::Load(row + (c + j * THREADS < whole ? c + j * THREADS : whole - 1) * N);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (c + j * THREADS < whole) {
#pragma unroll
                for (uint32_t i = 0; i < N; ++i) {
                    f(v[j].V[i], (c + j * THREADS) * N + i);
                }
            }
        }
    }
    for (uint32_t c = whole * N + threadIdx.x; c < classes; c += THREADS) {
        f(row[c], c);
    }
}

// The same one after the other, for what is rarely done: it takes few registers from the rest of a kernel
template <typename T, int THREADS, typename F>
__device__ __forceinline__ void ForRowSlowly(const T* row, uint32_t classes, F&& f) {
#pragma unroll 1
    for (uint32_t c = threadIdx.x; c < classes; c += THREADS) {
        f(row[c], c);
    }
}

// A position in a row's order: the key there, how many classes and which weights are before those of that key, how many have it
template <typename TKey>
struct TPosition {
    TKey Key;
    uint32_t Before, Alike;
    uint64_t WeightBefore;
};

// The position in sums by digits where the count or the weights reach `target`, which they do in one of them; the digit's class counts
// and weights are added to what `at` has before it
template <int BITS, int THREADS, typename TKey>
__device__ __forceinline__ uint32_t ReachDigit(const TDigitSums<BITS>& sums, bool byCount, uint64_t target, TPosition<TKey>& at, TShared<THREADS / 64>& shared) {
    constexpr uint32_t kMine = (1u << BITS) / THREADS;
    uint64_t weights = 0;
    uint32_t counts = 0;
    const uint32_t begin = threadIdx.x * kMine;
#pragma unroll
    for (uint32_t d = 0; d < kMine; ++d) {
        weights += sums.Weights[begin + d];
        counts += sums.Counts[begin + d];
    }
    uint64_t weightBefore = weights;
    uint32_t countBefore = counts;
    SumBefore(weightBefore, countBefore, shared);
    weightBefore += at.WeightBefore;
    countBefore += at.Before;
    const auto reached = [&](uint64_t weight, uint32_t count) { return byCount ? countBefore + uint64_t(count) >= target : weightBefore + weight >= target; };
    if (!reached(0, 0) && reached(weights, counts)) {
        uint32_t d = begin;
        for (; d + 1 < begin + kMine; ++d) {
            if (reached(sums.Weights[d], sums.Counts[d])) {
                break;
            }
            weightBefore += sums.Weights[d];
            countBefore += sums.Counts[d];
        }
        shared.Found[0] = d;
        shared.Found[1] = weightBefore;
        shared.Found[2] = countBefore;
        shared.Found[3] = sums.Counts[d];
    }
    __syncthreads();
    at.WeightBefore = shared.Found[1];
    at.Before = static_cast<uint32_t>(shared.Found[2]);
    at.Alike = static_cast<uint32_t>(shared.Found[3]);
    return static_cast<uint32_t>(shared.Found[0]);
}

// The (nth + 1)-th class with this key
template <typename T, int THREADS>
__device__ int32_t ClassOf(const T* row, uint32_t classes, typename TKeys<T>::TKey key, uint32_t nth, TShared<THREADS / 64>& shared) {
    using TK = TKeys<T>;
    constexpr uint32_t kWaves = THREADS / 64;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // which wave's part of the row has it, then which thread's part of that
    const uint32_t part = (classes + kWaves - 1) / kWaves;
    uint32_t begin = wave * part, end = begin + part < classes ? begin + part : classes, n = 0;
    for (uint32_t c = begin + lane; c < end; c += 64) {
        n += TK::Of(row[c]) == key;
    }
    n = SumUpTo(n);
    __syncthreads();
    if (lane == 63) {
        shared.Counted[wave] = n;
    }
    __syncthreads();
    uint32_t w = 0;
    while (w + 1 < kWaves && nth >= shared.Counted[w]) {
        nth -= shared.Counted[w++];
    }
    begin = w * part;
    end = begin + part < classes ? begin + part : classes;
    const uint32_t each = (part + THREADS - 1) / THREADS;
    const uint32_t mine = begin + threadIdx.x * each, last = mine + each < end ? mine + each : end;
    n = 0;
    for (uint32_t c = mine; c < last; ++c) {
        n += TK::Of(row[c]) == key;
    }
    uint64_t none = 0;
    uint32_t before = n;
    SumBefore(none, before, shared);
    if (nth >= before && nth < before + n) {
        for (uint32_t c = mine; c < last; ++c) {
            if (TK::Of(row[c]) == key && before++ == nth) {
                shared.Found[0] = c;
            }
        }
    }
    __syncthreads();
    return static_cast<int32_t>(shared.Found[0]);
}

// From sums up to positions: the row's limits, then its class. reach(byCount, target) -> TPosition, where the count or the weights from
// the front of the order, its own among them, reach `target`; classAt(position, nth) -> class. `all`: every weight's sum, `likely`: of
// those that MinP leaves, `there`: how many classes take part
template <typename T, typename TReach, typename TClass>
__device__ __forceinline__ void DrawFrom(const TSampleArguments& p, size_t r, const TLimits& limits, const TWeigh<true>& weigh, uint64_t all, uint64_t likely,
                                         uint64_t there, TReach&& reach, TClass&& classAt) {
    using TK = TKeys<T>;
    const auto wholeOf = [&](typename TK::TKey key) { return weigh.WholeOf(static_cast<T>(TK::Value(key))); };
    if (limits.TopK > 0 && static_cast<uint64_t>(limits.TopK) < there) {
        const auto at = reach(true, static_cast<uint64_t>(limits.TopK));
        all = at.WeightBefore + (static_cast<uint32_t>(limits.TopK) - at.Before) * wholeOf(at.Key);
    }
    uint64_t kept = all < likely ? all : likely;
    if (limits.TopP < 1) {
        const uint64_t target = limits.ShareOf(all);
        const auto at = reach(false, target);
        const uint64_t whole = wholeOf(at.Key);
        const uint64_t sum = at.WeightBefore + ((target - at.WeightBefore + whole - 1) / whole) * whole;
        kept = sum < kept ? sum : kept;
    }
    const uint64_t target = limits.DrawOf(kept);
    const auto at = reach(false, target);
    const double weight = weigh.Weight(weigh.Under(static_cast<T>(TK::Value(at.Key))));
    const int32_t index = classAt(at, static_cast<uint32_t>((target - 1 - at.WeightBefore) / weigh.Whole(weight)));
    if (threadIdx.x == 0) {
        Answer<T>(p, r, index, weight * weigh.Unit / static_cast<double>(kept));
    }
}

// Positions by the digits of how far a key is under the best one, with a pass over the row for each digit but the first: what takes
// any row, however many of its classes are alike
template <typename T, int THREADS, int BITS>
__device__ void DrawByDigits(const T* row, const TSampleArguments& p, size_t r, const TLimits& limits, const TWeigh<true>& weigh, typename TKeys<T>::TKey most,
                             uint64_t all, uint64_t likely, uint64_t there, TDigitSums<BITS>& sums, TShared<THREADS / 64>& shared) {
    using TK = TKeys<T>;
    using TKey = typename TK::TKey;
    constexpr int kLevels = (TK::kBits + BITS - 1) / BITS;
    const auto reach = [&](bool byCount, uint64_t target) {
        TPosition<TKey> at{0, 0, 0, 0};
        TKey prefix = 0;  // the digits so far
        for (int level = kLevels - 1; level >= 0; --level) {
            const uint32_t shift = level * BITS;
            __syncthreads();
            sums.template Clear<THREADS>();
            __syncthreads();
            ForRowSlowly<T, THREADS>(row, p.Classes, [&](T x, uint32_t) {
                const TKey key = TK::Of(x), under = most - key;
                if (key != 0 && (level == kLevels - 1 || under >> (shift + BITS) == prefix)) {
                    sums.Add(static_cast<uint32_t>(under >> shift) & ((1u << BITS) - 1), weigh.WholeOf(x));
                }
            });
            __syncthreads();
            prefix = prefix << BITS | ReachDigit<BITS, THREADS>(sums, byCount, target, at, shared);
        }
        at.Key = most - prefix;
        return at;
    };
    DrawFrom<T>(p, r, limits, weigh, all, likely, there, reach,
                [&](const TPosition<TKey>& at, uint32_t nth) { return ClassOf<T, THREADS>(row, p.Classes, at.Key, nth, shared); });
}

// The same from nothing but the best key
template <typename T, int THREADS, int BITS>
__device__ void DrawAny(const T* row, const TSampleArguments& p, size_t r, const TLimits& limits, TWeigh<true> weigh, typename TKeys<T>::TKey most,
                        TDigitSums<BITS>& sums, TShared<THREADS / 64>& shared) {
    uint64_t all, likely, there;
    for (uint32_t more = 0;;) {
        all = likely = there = 0;
        ForRowSlowly<T, THREADS>(row, p.Classes, [&](T x, uint32_t) {
            if (TKeys<T>::Of(x) != 0) {
                const double weight = weigh.Weight(weigh.Under(x));
                ++there;
                all += weigh.Whole(weight);
                likely += weight >= limits.MinP ? weigh.Whole(weight) : 0;
            }
        });
        all = SumOf(all, shared);
        likely = SumOf(likely, shared);
        there = SumOf(there, shared);
        if (more != 0 || (more = p.MoreBits(all)) == 0) {
            break;
        }
        weigh.Unit = ldexp(weigh.Unit, static_cast<int>(more));
    }
    DrawByDigits<T, THREADS, BITS>(row, p, r, limits, weigh, most, all, likely, there, sums, shared);
}

// Positions by t first, in steps of 56 / 2^BITS of a power of two. The classes of the step where a position is are listed, their keys
// told apart digit by digit, from the list. Weights, most of the work, are computed for classes up to the step of rank TopK. Scores are
// compared as they are, with bounds a little wider than a step's, before anything is computed for them.
template <typename T, int THREADS, int BITS, int LIST>
__global__ void __launch_bounds__(THREADS) SampleRowKernel(const T* scores, TSampleArguments p) {
    using TK = TKeys<T>;
    using TKey = typename TK::TKey;
    using A = TAcc<T>;
    constexpr uint32_t kDigits = 1u << BITS;
    constexpr double kStep = 56.0 / kDigits;
    constexpr A kNone = -std::numeric_limits<A>::infinity();
    __shared__ TDigitSums<BITS> first, later;
    __shared__ TShared<THREADS / 64> shared;
    __shared__ TKey keys[LIST];
    __shared__ uint32_t listed[LIST];

    const size_t r = p.First + blockIdx.x;
    const T* row = scores + r * p.Stride;
    FillPowers(shared.Powers);
    first.template Clear<THREADS>();
    A best = kNone;
    ForRow<T, THREADS>(row, p.Classes, [&](T x, uint32_t) { best = fmax(best, static_cast<A>(x)); });  // (NaN is passed over)
    const TKey most = MostOf(TK::Of(static_cast<T>(best)), shared);
    if (most == 0) {
        if (threadIdx.x == 0) {
            Answer<T>(p, r, -1, 0);
        }
        return;
    }
    const TLimits limits(p, r);
    if (limits.Greedy()) {
        const int32_t index = ClassOf<T, THREADS>(row, p.Classes, most, 0, shared);
        if (threadIdx.x == 0) {
            Answer<T>(p, r, index, 1);
        }
        return;
    }
    auto weigh = limits.Weigh<true>(TK::Value(most), p.Shift, shared.Powers);
    if (weigh.Best == __builtin_inf()) {
        return DrawAny<T, THREADS, BITS>(row, p, r, limits, weigh, most, later, shared);
    }
    // as Under, for a finite best score
    const auto underOf = [&](A x) {
        double under = weigh.Best - static_cast<double>(x);
        if constexpr (std::is_same_v<T, double>) {
            under = fmin(under, 1.7976931348623157e308);
        }
        return fmin(under * weigh.Rate, 4096.0);
    };
    const auto stepOf = [&](double under) {
        const uint32_t step = static_cast<uint32_t>(under * (1 / kStep));
        return step < kDigits ? step : kDigits - 1;
    };
    // A bound of the scores that are `under` or less; and more, on the side of `away`
    const auto boundOf = [&](double under, double away) {
        const double apart = under / weigh.Rate, bound = weigh.Best - apart;
        return static_cast<A>(bound + away * 1e-6 * (fabs(bound) + fabs(apart) + 1e-30));
    };
    // the last step of the classes that count: what is in the very last one weighs nothing
    uint32_t lastStep = kDigits - 1;
    uint64_t there = 0;
    if (limits.TopK > 0) {
        ForRow<T, THREADS>(row, p.Classes, [&](T x, uint32_t) {
            if (static_cast<A>(x) > kNone) {
                atomicAdd(&first.Counts[stepOf(underOf(static_cast<A>(x)))], 1u);
            }
        });
        __syncthreads();
        for (uint32_t d = threadIdx.x; d < kDigits; d += THREADS) {
            there += first.Counts[d];
        }
        there = SumOf(there, shared);
        if (static_cast<uint64_t>(limits.TopK) < there) {
            TPosition<TKey> at{0, 0, 0, 0};
            lastStep = ReachDigit<BITS, THREADS>(first, true, static_cast<uint64_t>(limits.TopK), at, shared);
        }
        there = lastStep < kDigits - 1 ? there : 0;  // no class that weighs anything is left out by its rank
        __syncthreads();
    }
    const A lowest = lastStep < kDigits - 1 ? boundOf((lastStep + 1) * kStep, -1) : kNone;
    uint64_t all, likely;
    const bool atLeast = limits.MinP > 0;
    for (uint32_t more = 0;;) {
        all = likely = 0;
        ForRow<T, THREADS>(row, p.Classes, [&](T x, uint32_t) {
            const A score = static_cast<A>(x);
            if (score >= lowest && score > kNone) {
                const double under = underOf(score), weight = weigh.Weight(under);
                const uint32_t step = stepOf(under);
                const uint64_t whole = weigh.Whole(weight);
                if (step <= lastStep) {
                    atomicAdd(reinterpret_cast<unsigned long long*>(&first.Weights[step]), static_cast<unsigned long long>(whole));
                    if (atLeast) {
                        likely += weight >= limits.MinP ? whole : 0;
                    }
                }
            }
        });
        __syncthreads();
        for (uint32_t d = threadIdx.x; d < kDigits; d += THREADS) {
            all += first.Weights[d];
        }
        all = SumOf(all, shared);
        likely = atLeast ? SumOf(likely, shared) : all;
        if (more != 0 || (more = p.MoreBits(all)) == 0) {
            break;
        }
        weigh.Unit = ldexp(weigh.Unit, static_cast<int>(more));
        for (uint32_t d = threadIdx.x; d < kDigits; d += THREADS) {
            first.Weights[d] = 0;
        }
        __syncthreads();
    }
    uint32_t listedStep = kDigits;
    const auto reach = [&](bool byCount, uint64_t target) {
        TPosition<TKey> at{0, 0, 0, 0};
        const uint32_t step = ReachDigit<BITS, THREADS>(first, byCount, target, at, shared);
        const A low = boundOf((step + 1) * kStep, -1), high = step > 0 ? boundOf(step * kStep, 1) : static_cast<A>(weigh.Best);
        const auto forStep = [&](auto&& f) {
            ForRow<T, THREADS>(row, p.Classes, [&](T x, uint32_t c) {
                const A score = static_cast<A>(x);
                if (score >= low && score <= high && score > kNone && stepOf(underOf(score)) == step) {
                    f(TK::Of(x), c);
                }
            });
        };
        __syncthreads();
        if (step != listedStep) {
            if (threadIdx.x == 0) {
                shared.Listed = 0;
            }
            __syncthreads();
            forStep([&](TKey key, uint32_t c) {
                const uint32_t place = atomicAdd(&shared.Listed, 1u);
                if (place < LIST) {
                    keys[place] = key;
                    listed[place] = c;
                }
            });
            listedStep = step;
            __syncthreads();
        }
        const uint32_t n = shared.Listed;
        const auto forKeys = [&](auto&& f) {
            if (n <= LIST) {
                for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
                    f(keys[i]);
                }
            } else {
                // a step of more classes than the list holds
                forStep([&](TKey key, uint32_t) { f(key); });
            }
        };
        TKey most = 0, least = 0;  // least: of the complement
        forKeys([&](TKey key) {
            const TKey other = ~key;
            most = key > most ? key : most;
            least = other > least ? other : least;
        });
        most = MostOf(most, shared);
        least = ~MostOf(least, shared);
        int bits = 0;
        while (bits < TK::kBits && (most - least) >> bits != 0) {
            ++bits;
        }
        TKey prefix = 0;
        at.Alike = n;
        for (int level = (bits + BITS - 1) / BITS - 1; level >= 0; --level) {
            const uint32_t shift = level * BITS;
            __syncthreads();
            later.template Clear<THREADS>();
            __syncthreads();
            forKeys([&](TKey key) {
                const TKey under = most - key;
                if (shift + BITS >= static_cast<uint32_t>(TK::kBits) || under >> (shift + BITS) == prefix) {
                    later.Add(static_cast<uint32_t>(under >> shift) & (kDigits - 1), weigh.WholeOf(static_cast<T>(TK::Value(key))));
                }
            });
            __syncthreads();
            prefix = prefix << BITS | ReachDigit<BITS, THREADS>(later, byCount, target, at, shared);
        }
        at.Key = most - prefix;
        return at;
    };
    DrawFrom<T>(p, r, limits, weigh, all, likely, there, reach, [&](const TPosition<TKey>& at, uint32_t nth) {
        const uint32_t n = shared.Listed;
        if (n > LIST) {
            return ClassOf<T, THREADS>(row, p.Classes, at.Key, nth, shared);
        }
        // the last position's list has them all, in no order
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
            if (keys[i] == at.Key) {
                uint32_t before = 0;
                for (uint32_t j = 0; j < n && at.Alike > 1; ++j) {
                    before += keys[j] == at.Key && listed[j] < listed[i];
                }
                if (before == nth) {
                    shared.Found[0] = listed[i];
                }
            }
        }
        __syncthreads();
        return static_cast<int32_t>(shared.Found[0]);
    });
}

// 16-bit scores: how often each key comes, counted in 16 bits in LDS, says everything. A weight is computed for each key that there is
// instead of each class, and only up to the one of rank TopK. A key that more than 65535 classes have shows in the counts' sum; such a row
// is done by digits.
template <typename T>
__global__ void __launch_bounds__(1024) SampleCountedKernel(const T* scores, TSampleArguments p) {
    using TK = TKeys<T>;
    using TPair = __attribute__((ext_vector_type(2))) uint16_t;
    using TSignedPair = __attribute__((ext_vector_type(2))) int16_t;
    constexpr int kThreads = 1024, kWaves = 16;
    constexpr uint32_t kWords = 32768;  // two counts in each
    constexpr uint32_t kInfinity = std::is_same_v<T, _Float16> ? 0x7c00 : 0x7f80;
    constexpr uint32_t kHighest = 0x8000 | kInfinity, kLowest = 0x7fff ^ kInfinity;  // keys here: of plus and minus infinity
    __shared__ union {
        uint32_t Counts[kWords];
        TDigitSums<11> Sums;
    } lds;
    __shared__ TShared<kWaves> shared;
    __shared__ TDigitSums<8> segments;

    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t r = p.First + blockIdx.x;
    const T* row = scores + r * p.Stride;
    // A wave's part of the row's whole 16 bytes is contiguous, in pieces of 64 times as many; up to seven classes behind them are the first
    // threads' own. Keys grow with the scores, the zeros have one, NaN are at both ends.
    const uint32_t whole = p.Classes & ~7u;
    const uint32_t pieces = (p.Classes + kWaves * 512 - 1) / (kWaves * 512);
    const uint32_t begin = wave * pieces * 512 + lane * 8;
    struct TKeysOfEight {
        TPair V[4];
    };
    const auto keysAt = [&](uint32_t piece) {
        const uint32_t c = begin + piece * 512;
        TValues<uint32_t, 4> words = TValues<uint32_t, 4>::Load(row + (c < whole ? c : 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            words.V[j] = c < whole ? words.V[j] : 0x10001u * (0x8000 | kInfinity);
        }
        return words;
    };
    const auto keysOfWords = [](const TValues<uint32_t, 4>& words) {
        TKeysOfEight keys;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const TSignedPair sign = __builtin_bit_cast(TSignedPair, words.V[j]) >> TSignedPair{15, 15};
            const TPair key = __builtin_bit_cast(TPair, words.V[j]) ^ (__builtin_bit_cast(TPair, sign) | TPair{0x8000, 0x8000});
            // minus zero's, 0x7fff, becomes zero's
            keys.V[j] = key + (TPair{1, 1} - __builtin_elementwise_min(key ^ TPair{0x7fff, 0x7fff}, TPair{1, 1}));
        }
        return keys;
    };
    // f(keys of a thread's eight classes of a piece in pairs, the piece)
    constexpr uint32_t kAtOnce = 8;
    TKeysOfEight held[kAtOnce];
    const auto load = [&](uint32_t first) {
        TValues<uint32_t, 4> words[kAtOnce];
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j) {
            // (the last piece again behind the end: no load waits in a branch)
            words[j] = keysAt(first + j < pieces ? first + j : pieces - 1);
        }
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j) {
            held[j] = keysOfWords(words[j]);
        }
    };
    const auto forPieces = [&](auto&& f) {
        for (uint32_t first = 0; first < pieces; first += kAtOnce) {
            load(first);
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j) {
                if (first + j < pieces) {
                    f(held[j], first + j);
                }
            }
        }
    };
    uint32_t ownKey = kLowest;
    if (whole + threadIdx.x < p.Classes) {
        const TValues<uint32_t, 4> word = {{__builtin_bit_cast(uint16_t, row[whole + threadIdx.x]), 0, 0, 0}};
        ownKey = keysOfWords(word).V[0][0];
    }
    FillPowers(shared.Powers);
#pragma unroll
    for (uint32_t i = 0; i < kWords / 4 / kThreads; ++i) {
        reinterpret_cast<uint4*>(lds.Counts)[threadIdx.x + i * kThreads] = uint4{0, 0, 0, 0};
    }
    TPair mosts = {static_cast<uint16_t>(ownKey), 0};
    forPieces([&](const TKeysOfEight& keys, uint32_t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mosts = __builtin_elementwise_max(mosts, keys.V[j]);
        }
    });
    uint32_t most = MostOf<kWaves>(static_cast<uint32_t>(mosts[0] > mosts[1] ? mosts[0] : mosts[1]), shared);
    if (most > kHighest) {
        // there are NaN over plus infinity (those do not take part: they are over the best key, which counts as far under it)
        most = ownKey <= kHighest ? ownKey : 0;
        forPieces([&](const TKeysOfEight& keys, uint32_t) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t key = keys.V[j / 2][j % 2];
                most = key <= kHighest && key > most ? key : most;
            }
        });
        most = MostOf<kWaves>(most, shared);
    }
    if (most <= kLowest) {
        if (threadIdx.x == 0) {
            Answer<T>(p, r, -1, 0);
        }
        return;
    }
    const TLimits limits(p, r);
    const auto sharedKey = [](uint32_t key) { return key - kLowest - (key >> 15); };  // as TKeys has it, with one key for both zeros
    // the (nth + 1)-th class with this key
    const auto classOf = [&](uint32_t key, uint32_t nth) {
        const TPair wanted = {static_cast<uint16_t>(key), static_cast<uint16_t>(key)};
        // 1 where a key is another one
        const auto other = [&](TPair keys) { return __builtin_elementwise_min(keys ^ wanted, TPair{1, 1}); };
        // how many of them the pieces have, 256 parts of the row that hold some in a row each: of each part first, then in its pieces
        const uint32_t each = (pieces + 15) / 16;  // pieces of a part
        __syncthreads();
        if (threadIdx.x < 256) {
            segments.Counts[threadIdx.x] = 0;
        }
        __syncthreads();
        forPieces([&](const TKeysOfEight& keys, uint32_t piece) {
            const TPair others = (other(keys.V[0]) + other(keys.V[1])) + (other(keys.V[2]) + other(keys.V[3]));
            const uint32_t n = 8 - others[0] - others[1];
            if (n != 0) {
                atomicAdd(&segments.Counts[wave * 16 + piece / each], n);
            }
        });
        __syncthreads();
        uint32_t counts[4], sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            counts[j] = segments.Counts[lane * 4 + j];
            sum += counts[j];
        }
        uint32_t before = SumUpTo(sum) - sum, part = lane * 4;
        const int from = __ffsll(static_cast<unsigned long long>(__ballot(nth < before + sum))) - 1;
        const uint32_t inPieces = OfLane(before + sum, 63);
#pragma unroll
        for (uint32_t j = 0; j < 3; ++j) {
            const uint32_t n = counts[j];
            const bool past = part == lane * 4 + j && nth >= before + n;
            before += past ? n : 0;
            part += past ? 1 : 0;
        }
        before = OfLane(before, from < 0 ? 0 : from);
        part = OfLane(part, from < 0 ? 0 : from);
        if (from < 0) {
            // behind the whole 16 bytes
            const uint64_t own = __ballot(ownKey == key);
            if (wave == 0 && ownKey == key && inPieces + __popcll(own & ((uint64_t(1) << lane) - 1)) == nth) {
                shared.Found[0] = whole + lane;
            }
        } else if (part / 16 == wave) {
            for (uint32_t piece = part % 16 * each; piece < (part % 16 + 1) * each && piece < pieces; ++piece) {
                const TKeysOfEight keys = keysOfWords(keysAt(piece));
                uint32_t mine = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    mine += keys.V[j / 2][j % 2] == key;
                }
                const uint32_t upTo = before + SumUpTo(mine);
                uint32_t place = upTo - mine;
                if (nth >= place && nth < upTo) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (keys.V[j / 2][j % 2] == key && place++ == nth) {
                            shared.Found[0] = begin + piece * 512 + j;
                        }
                    }
                }
                before = OfLane(upTo, 63);
            }
        }
        __syncthreads();
        return static_cast<int32_t>(shared.Found[0]);
    };
    if (limits.Greedy()) {
        const int32_t index = classOf(most, 0);
        if (threadIdx.x == 0) {
            Answer<T>(p, r, index, 1);
        }
        return;
    }
    auto weigh = limits.Weigh<true>(TK::Value(sharedKey(most)), p.Shift, shared.Powers);
    const uint32_t keys = most - kLowest;  // from the best one down to the last over minus infinity
    uint32_t mine = 0;
    if (most - ownKey < keys) {
        ++mine;
        atomicAdd(&lds.Counts[(most - ownKey) >> 1], 1u << ((most - ownKey) << 4 & 31));
    }
    const TPair best = {static_cast<uint16_t>(most), static_cast<uint16_t>(most)};
    forPieces([&](const TKeysOfEight& keysOfEight, uint32_t) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (keys over the best one, of NaN, come out at `most` at least)
            const TPair pair = best - keysOfEight.V[j];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t under = pair[k];
                if (under < keys) {
                    ++mine;
                    atomicAdd(&lds.Counts[under >> 1], 1u << (under << 4 & 31));
                }
            }
        }
    });
    const uint64_t there = SumOf(mine, shared);
    __syncthreads();
    // Sums of 256 keys in a row, four for a lane; a wave has every sixteenth of them, since the keys that there are lie together
    const auto weightOf = [&](uint32_t under) { return weigh.Weight(weigh.Under(static_cast<T>(TK::Value(sharedKey(most - under))))); };
    struct TOfLane {
        uint64_t Weights[4];
        uint32_t Counts[4];
    };
    const auto keysOf = [&](uint32_t segment, uint64_t* atLeast) {
        const uint2 words = reinterpret_cast<const uint2*>(lds.Counts)[segment * 64 + lane];
        TOfLane v = {{0, 0, 0, 0}, {words.x & 0xffff, words.x >> 16, words.y & 0xffff, words.y >> 16}};
        if (__ballot((words.x | words.y) != 0) != 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double weight = weightOf(segment * 256 + lane * 4 + j);
                v.Weights[j] = v.Counts[j] != 0 ? weigh.Whole(weight) * v.Counts[j] : 0;
                if (atLeast != nullptr) {
                    *atLeast += weight >= limits.MinP ? v.Weights[j] : 0;
                }
            }
        }
        return v;
    };
    uint64_t counts = 0;
    for (uint32_t segment = wave; segment < 256; segment += kWaves) {
        const uint2 words = reinterpret_cast<const uint2*>(lds.Counts)[segment * 64 + lane];
        const uint32_t count = (words.x & 0xffff) + (words.x >> 16) + (words.y & 0xffff) + (words.y >> 16);
        const uint32_t sum = SumUpTo(count);
        counts += count;
        if (lane == 63) {
            segments.Counts[segment] = sum;
            segments.Weights[segment] = 0;
        }
    }
    if (SumOf(counts, shared) != there) {
        return DrawAny<T, kThreads, 11>(row, p, r, limits, weigh, sharedKey(most), lds.Sums, shared);
    }
    // the last segment whose weights are asked for
    uint32_t lastSegment = 255;
    if (limits.TopK > 0 && static_cast<uint64_t>(limits.TopK) < there) {
        uint32_t sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sum += segments.Counts[lane * 4 + j];
        }
        const uint64_t reached = __ballot(SumUpTo(sum) >= static_cast<uint32_t>(limits.TopK));
        lastSegment = (__ffsll(static_cast<unsigned long long>(reached)) - 1) * 4 + 3;
    }
    uint64_t likely, all;
    for (uint32_t more = 0;;) {
        likely = all = 0;
        for (uint32_t segment = wave; segment <= lastSegment; segment += kWaves) {
            if (segments.Counts[segment] != 0) {
                const TOfLane v = keysOf(segment, &likely);
                const uint64_t weight = SumUpTo((v.Weights[0] + v.Weights[1]) + (v.Weights[2] + v.Weights[3]));
                if (lane == 63) {
                    segments.Weights[segment] = weight;
                    all += weight;
                }
            }
        }
        all = SumOf(all, shared);
        likely = SumOf(likely, shared);
        if (more != 0 || (more = p.MoreBits(all)) == 0) {
            break;
        }
        weigh.Unit = ldexp(weigh.Unit, static_cast<int>(more));
    }
    // every wave for itself: the segment, then the key in it
    const auto reach = [&](bool byCount, uint64_t target) {
        uint64_t weight = 0;
        uint32_t count = 0;
        const auto place = [&](const TOfLane& v) {
            uint64_t weights = (v.Weights[0] + v.Weights[1]) + (v.Weights[2] + v.Weights[3]);
            uint32_t counted = (v.Counts[0] + v.Counts[1]) + (v.Counts[2] + v.Counts[3]);
            const uint64_t mine = weights;
            const uint32_t mineCounted = counted;
            weights = SumUpTo(weights);
            counted = SumUpTo(counted);
            weights += weight;
            counted += count;
            const uint64_t reached = __ballot(byCount ? counted >= target : weights >= target);
            const int from = __ffsll(static_cast<unsigned long long>(reached)) - 1;
            weight = weights - mine;
            count = counted - mineCounted;
            uint32_t place = lane * 4, of = v.Counts[3];
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                const uint64_t w = v.Weights[j];
                const uint32_t c = v.Counts[j];
                const bool past = place == lane * 4 + j && (byCount ? count + c < target : weight + w < target);
                of = place == lane * 4 + j && !past ? c : of;
                weight += past ? w : 0;
                count += past ? c : 0;
                place += past ? 1 : 0;
            }
            weight = OfLane(weight, from);
            count = OfLane(count, from);
            struct TFound {
                uint32_t Place, Counts;
            };
            return TFound{OfLane(place, from), OfLane(of, from)};
        };
        TOfLane v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v.Weights[j] = segments.Weights[lane * 4 + j];
            v.Counts[j] = segments.Counts[lane * 4 + j];
        }
        const uint32_t segment = place(v).Place;
        const auto found = place(keysOf(segment, nullptr));
        return TPosition<typename TK::TKey>{sharedKey(most - (segment * 256 + found.Place)), count, found.Counts, weight};
    };
    DrawFrom<T>(p, r, limits, weigh, all, likely, there, reach,
                [&](const TPosition<typename TK::TKey>& at, uint32_t nth) { return classOf(at.Key + kLowest + (at.Key >= kInfinity ? 1 : 0), nth); });
}

}  // namespace op

using namespace op;

namespace {

constexpr size_t kMostClassesToSample = size_t(1) << 24;
constexpr size_t kMostGroupsToSample = size_t(1) << 21;

// f(integral_constant) for the n of 1 to MOST that `n` is
template <int MOST, typename F>
void WithNumber(size_t n, F&& f) {
    if constexpr (MOST > 1) {
        if (n < MOST) {
            return WithNumber<MOST - 1>(n, f);
        }
    }
    f(std::integral_constant<int, MOST>());
}

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
    p.Shift = kMostBits;
    while ((size_t(1) << (63 - p.Shift)) <= classes) {
        --p.Shift;
    }
    p.Stride = scoreStride;
    p.Sampling = sampling;
    p.Uniform = uniform;
    p.Indexes = indexes;
    p.Weights = weights;
    const auto launch = [&](auto kernel, const auto* from, uint32_t threads, size_t rowsOfGroup) {
        for (p.First = 0; p.First < rows; p.First += kMostGroupsToSample * rowsOfGroup) {
            p.Rows = std::min(rows - p.First, kMostGroupsToSample * rowsOfGroup);
            call.Launch(kernel, (p.Rows + rowsOfGroup - 1) / rowsOfGroup, threads, 0, from, p);
        }
    };
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        const T* from = static_cast<const T*>(scores);
        // (2M x 10 f64 58 us, 1M x 16 f32 58; 250000 x 64 f64 206; 16000 x 1000 f64 238, 258 with a workgroup each, 100 rows of it 30 and 26)
        if (classes <= 16) {
            return WithNumber<16>(classes, [&](auto n) { launch(SampleOfFewKernel<T, decltype(n)::value>, from, 256, 256); });
        }
        if (classes <= 32) {
            return launch(SampleByLanesKernel<T, 32, 1>, from, 256, 8);
        }
        if (classes <= 64) {
            return launch(SampleByLanesKernel<T, 64, 1>, from, 256, 4);
        }
        if (classes <= 128) {
            return launch(SampleByLanesKernel<T, 64, 2>, from, 256, 4);
        }
        if (classes <= 256) {
            return launch(SampleByLanesKernel<T, 64, 4>, from, 256, 4);
        }
        if (classes <= 512) {
            return launch(SampleByLanesKernel<T, 64, 8>, from, 256, 4);
        }
        if (classes <= 1024) {
            return launch(SampleByLanesKernel<T, 64, 16>, from, 256, 4);
        }
        if (classes <= 4096) {
            return launch(SampleRowKernel<T, 256, 9, 1024>, from, 256, 1);
        }
        if constexpr (sizeof(T) == 2) {
            // (64 x 131000 bf16 46 us, 359 with weights of each class)
            launch(SampleCountedKernel<T>, from, 1024, 1);
        } else {
            // two workgroups for a compute unit where rows are more than those (with a share of 0.95, 384 x 100003 f32 151 us, 164 with 1024 threads each;
            // 2000 x 10000 107 and 182; 257 x 100003 126 and 131; 256 x 100003 112 and 89, 32 x 100003 92 and 72)
            constexpr int kList = 2048;
            rows > 256 ? launch(SampleRowKernel<T, 512, 11, kList>, from, 512, 1) : launch(SampleRowKernel<T, 1024, 11, kList>, from, 1024, 1);
        }
    });
}

}  // namespace cbamd
