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
    size_t Rows, FirstTile;
    uint32_t Classes, Slices, SliceClasses;       // of AdjustSliceKernel
    uint32_t RowsPerTile, Pieces, PiecesInverse, RowLanesLog2;  // of AdjustRowsKernel
    CbHipScoreAdjustment A;
};

__device__ __forceinline__ int64_t Clamped(int64_t at, size_t count) {
    return at < 0 ? 0 : at > static_cast<int64_t>(count) ? static_cast<int64_t>(count) : at;
}

// The mask that a row has, -1: none
__device__ __forceinline__ int64_t MaskOf(const CbHipScoreAdjustment& p, size_t row) {
    const int64_t mask = p.AllowedRows != nullptr ? static_cast<int64_t>(p.AllowedRows[row]) : static_cast<int64_t>(row);
    return mask >= 0 && static_cast<size_t>(mask) < p.AllowedCount ? mask : -1;
}

// A row's penalties. A part that a call leaves out has the value that changes nothing: a repetition penalty of 1, a frequency
// and a presence penalty of 0
struct TPenalties {
    float Repetition, Frequency, Presence, Unused;

    __device__ __forceinline__ static TPenalties Of(const CbHipScoreAdjustment& p, size_t row) {
        return {p.Repetition != nullptr ? p.Repetition[row] : 1.f, p.Frequency != nullptr ? p.Frequency[row] : 0.f,
                p.Presence != nullptr ? p.Presence[row] : 0.f, 0.f};
    }
};

// A tile's table in LDS has a word for each of its scores that counts the row's history: 1 for a class that was given, 2
// for each time that it was generated, so that a word is 0 exactly for the classes outside the history. The row's biases have
// the table afterwards. Both are made by integer atomics, whose order does not show.
__device__ __forceinline__ void CountEntry(uint32_t* word, bool given) {
    if (given) {
        atomicOr(word, 1u);
    } else {
        atomicAdd(word, 2u);
    }
}

// The N words of a piece in a table, which begins at a multiple of 16 bytes, and whether any is not 0
template <int N>
struct TWords : TValues<uint32_t, N> {
    uint32_t Any = 0;
    static constexpr int Alignment = N * 4 < 16 ? N * 4 : 16;

    __device__ __forceinline__ TWords() {}
    __device__ __forceinline__ explicit TWords(const uint32_t* words) {
        __builtin_memcpy(this->V, __builtin_assume_aligned(words, Alignment), sizeof(this->V));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            Any |= this->V[i];
        }
    }
    __device__ __forceinline__ static void Clear(uint32_t* words) {
        const TValues<uint32_t, N> none{};
        __builtin_memcpy(__builtin_assume_aligned(words, Alignment), &none, sizeof(none));
    }
};

// Four entries of a list of `count` from entry e on
__device__ __forceinline__ TValues<int32_t, 4> LoadEntries(const int32_t* list, int64_t e, size_t count) {
    return LoadUpTo<int32_t, 4>(list + e, count - static_cast<size_t>(e));
}

// A row of up to this many biases needs no table of them: the word of a class that has one names it in its upper bits, if the
// history is short enough for its counts to leave those free (64 x 131000 16-bit scores with 3000 entries and 20 biases a row 15.1 us, with a
// table 16.5; 2M x 10 32-bit ones with two of each 95 and 108)
constexpr uint32_t kNamedBiases = 1024, kNameShift = 21;
constexpr int64_t kNamedHistory = int64_t(1) << (kNameShift - 2);

// The bits of -0, which changes no score when it is added (0 would make a score of -0 a 0)
constexpr uint32_t kNoBias = 0x80000000u;

// 16 bytes of scores as they are in memory. (As single 16-bit values they would take a register each.)
using TRaw = TValues<uint32_t, 4>;

// A piece's scores on their way
template <typename T>
struct TPiece {
    using A = TAcc<T>;
    static constexpr int N = 16 / sizeof(T);
    A X[N];

    __device__ __forceinline__ void From(const TRaw& raw) {
        TValues<T, N> v;
        __builtin_memcpy(&v, &raw, 16);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            X[i] = static_cast<A>(v.V[i]);
        }
    }
    // (`counts`: the bits of a word that count)
    __device__ __forceinline__ void Penalize(const TValues<uint32_t, N>& words, const TPenalties& penalties, uint32_t counts = ~0u) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t w = words.V[i] & counts;
            if (w != 0) {
                const A repetition = penalties.Repetition;
                X[i] = X[i] > 0 ? X[i] / repetition : X[i] * repetition;
            }
            if (w > 1) {
                X[i] -= static_cast<A>(penalties.Frequency) * static_cast<A>(w >> 1);
                X[i] -= static_cast<A>(penalties.Presence);
            }
        }
    }
    __device__ __forceinline__ void Add(const TValues<float, N>& bias) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            X[i] += bias.V[i];
        }
    }
    __device__ __forceinline__ void AddNamed(const TValues<uint32_t, N>& words, const float* biasValues) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (words.V[i] >> 31 != 0) {
                X[i] += biasValues[words.V[i] >> kNameShift & (kNamedBiases - 1)];
            }
        }
    }
    // (from a table, see MakeBiases)
    __device__ __forceinline__ void Add(const uint32_t* words) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            X[i] += __uint_as_float(words[i] ^ kNoBias);
        }
    }
    // a bit of `allowed` for each of them
    __device__ __forceinline__ TRaw Rounded(uint32_t allowed) const {
        TValues<T, N> v;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v.V[i] = static_cast<T>((allowed >> i & 1) != 0 ? X[i] : -std::numeric_limits<A>::infinity());
        }
        TRaw raw;
        __builtin_memcpy(&raw, &v, 16);
        return raw;
    }
};

// The first n values of a piece (a row's last piece may have less than N)
template <typename T>
__device__ __forceinline__ TRaw LoadPiece(const T* at, uint32_t n) {
    const TValues<T, 16 / sizeof(T)> v = LoadUpTo<T, 16 / sizeof(T)>(at, n);
    TRaw raw;
    __builtin_memcpy(&raw, &v, 16);
    return raw;
}
// The same in a row of at least N values, without branches: the load ends with the row, the values are shifted into place
template <typename T>
__device__ __forceinline__ TRaw LoadShifted(const T* at, uint32_t n) {
    constexpr uint32_t N = 16 / sizeof(T);
    const uint32_t back = n < N ? N - n : 0;
    unsigned __int128 bits;
    __builtin_memcpy(&bits, at - back, 16);
    bits >>= back * (8 * sizeof(T));
    TRaw raw;
    __builtin_memcpy(&raw, &bits, 16);
    return raw;
}
template <typename T>
__device__ __forceinline__ void StorePiece(const TRaw& raw, T* at, uint32_t n) {
    TValues<T, 16 / sizeof(T)> v;
    __builtin_memcpy(&v, &raw, 16);
    StoreUpTo<T, 16 / sizeof(T)>(v, at, n);
}

// The table of biases: the last entry of each class, counted from 1, and then its value's bits in its place, with the sign
// the other way around, so that 0, the word of a class without an entry, stands for -0. Entries are taken `threads` at a time,
// so that an entry looks whether it is the last one before any of the same class writes: the ones after it are in its own
// batch or a later one. `word(i, entry)`: the word of entry i's class, null outside of the tile
template <typename F>
__device__ __forceinline__ void MakeBiases(uint32_t threads, uint32_t count, const int32_t* classes, const float* values, int32_t firstClass, float firstValue, F&& word) {
    for (uint32_t i = threadIdx.x; i < count; i += threads) {
        uint32_t* at = word(i, i == threadIdx.x ? firstClass : classes[i]);
        if (at != nullptr) {
            atomicMax(at, i + 1);
        }
    }
    __syncthreads();
    for (uint32_t begin = 0; begin < count; begin += threads) {
        const uint32_t i = begin + threadIdx.x;
        uint32_t* at = nullptr;
        float value = firstValue;
        if (i < count) {
            at = word(i, begin == 0 ? firstClass : classes[i]);
            value = begin == 0 ? firstValue : values[i];
        }
        const bool isLast = at != nullptr && *at == i + 1;
        __syncthreads();
        if (isLast) {
            *at = __float_as_uint(value) ^ kNoBias;
        }
    }
    __syncthreads();
}

// A workgroup for a slice of one row, at most P pieces for each of its threads. What it reads is requested at once, as far as its place is
// known, and without branches, which would wait for one load after the other: the scores, the mask's words, the first
// entries of the lists; the table is made while they are on their way. Its words count the history and name the biases' classes;
// where that does not fit, the table of the biases has its place afterwards. Two workgroups fit a compute unit either way. Every slice
// of a row looks through the row's whole history; slices of a row are alike in length. Memory bounds it when there is much: 384 x
// 100003 32-bit scores with 12000 entries a row take 80 us (4.1 TB/s); 64 x 131000 of 16 bits with 3000 entries, biases and masks 15,
// where the steps wait for each other.
template <typename T, int P, bool BIASES>
__global__ void __launch_bounds__(1024) AdjustSliceKernel(TAdjustArgs a) {
    const uint32_t threads = blockDim.x;
    constexpr int N = 16 / sizeof(T);
    extern __shared__ uint4 tables[];
    const CbHipScoreAdjustment& p = a.A;
    const bool history = p.HistoryOffsets != nullptr;
    uint32_t* words = reinterpret_cast<uint32_t*>(tables);
    float* biasValues = reinterpret_cast<float*>(words + a.SliceClasses);
    const auto clear = [&] {
        for (uint32_t i = threadIdx.x; i < a.SliceClasses / 4; i += threads) {
            tables[i] = uint4{0, 0, 0, 0};
        }
        __syncthreads();
    };
    const size_t tile = a.FirstTile + blockIdx.x;
    const size_t row = tile / a.Slices;
    const uint32_t c0 = static_cast<uint32_t>(tile - row * a.Slices) * a.SliceClasses;
    const uint32_t width = min(a.SliceClasses, a.Classes - c0);
    int64_t begin = 0, end = 0, given = 0, firstBias = 0, endBias = 0;
    TPenalties penalties{1, 0, 0, 0};
    if (history) {
        given = p.HistoryOffsets[row];
        begin = Clamped(given, p.HistoryCount);
        end = Clamped(p.HistoryOffsets[row + 1], p.HistoryCount);
        given += p.PromptLengths != nullptr ? p.PromptLengths[row] : 0;
        penalties = TPenalties::Of(p, row);
    }
    if (BIASES) {
        firstBias = Clamped(p.BiasOffsets[row], p.BiasCount);
        endBias = max(firstBias, Clamped(p.BiasOffsets[row + 1], p.BiasCount));
    }
    const int64_t mask = p.AllowedCount != 0 ? MaskOf(p, row) : -1;
    const T* from = static_cast<const T*>(a.Scores) + row * a.ScoreStride + c0;
    const bool whole = width % N == 0;  // only a row's last slice may end inside a piece
    TRaw raw[P];
    uint32_t allowed[P];
    if (whole) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            raw[j] = TRaw::Load(from + min((j * threads + threadIdx.x) * N, width - N));
        }
    } else {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint32_t c = (j * threads + threadIdx.x) * N;
            if (c < width) {
                raw[j] = LoadPiece<T>(from + c, width - c);
            }
        }
    }
    if (mask >= 0) {
        const uint32_t* bits = p.Allowed + static_cast<size_t>(mask) * p.AllowedStride;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            // (N classes from a multiple of N on are in one word)
            allowed[j] = bits[(c0 + min((j * threads + threadIdx.x) * N, width - 1)) >> 5];
        }
    }
    int32_t biasClass = 0;
    float biasValue = 0;
    if (firstBias + threadIdx.x < endBias) {
        biasClass = p.BiasClasses[firstBias + threadIdx.x];
        biasValue = p.BiasValues[firstBias + threadIdx.x];
    }
    const bool few = BIASES && endBias - firstBias <= kNamedBiases && end - begin < kNamedHistory;
    const uint32_t named = few ? static_cast<uint32_t>(endBias - firstBias) : 0;
    const bool table = history || named > 0;
    if (table) {
        int64_t e = begin + threadIdx.x * 4;
        TValues<int32_t, 4> entries{};
        if (e < end) {
            entries = LoadEntries(p.History, e, p.HistoryCount);
        }
        clear();
        if (named > 0) {
            for (uint32_t i = threadIdx.x; i < named; i += threads) {
                const bool first = i == threadIdx.x;
                const uint32_t c = static_cast<uint32_t>(first ? biasClass : p.BiasClasses[firstBias + i]) - c0;
                if (c < width) {
                    atomicMax(&words[c], 1u << 31 | i << kNameShift);  // the last one of a class stays
                }
                biasValues[i] = first ? biasValue : p.BiasValues[firstBias + i];
            }
            __syncthreads();
        }
        while (e < end) {
            const int64_t next = e + threads * 4;
            TValues<int32_t, 4> more{};
            if (next < end) {
                more = LoadEntries(p.History, next, p.HistoryCount);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t c = static_cast<uint32_t>(entries.V[i]) - c0;  // outside of the slice: large
                if (c < width && e + i < end) {
                    CountEntry(&words[c], e + i < given);
                }
            }
            entries = more;
            e = next;
        }
        __syncthreads();
    }
    TValues<float, N> classBias[P];
    if (p.ClassBias != nullptr) {
        const float* bias = p.ClassBias + row * p.ClassBiasStride + c0;
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint32_t c = (j * threads + threadIdx.x) * N;
            if (whole) {
                classBias[j] = TValues<float, N>::Load(bias + min(c, width - N));
            } else if (c < width) {
                classBias[j] = LoadUpTo<float, N>(bias + c, width - c);
            }
        }
    }
    T* to = static_cast<T*>(a.Result) + row * a.ResultStride + c0;
    const auto store = [&](int j, const TPiece<T>& x) {
        const uint32_t c = (j * threads + threadIdx.x) * N;
        if (c < width) {
            const TRaw out = x.Rounded(mask >= 0 ? allowed[j] >> (c & 31) : ~0u);
            if (whole) {
                out.Store(to + c);
            } else {
                StorePiece<T>(out, to + c, width - c);
            }
        }
    };
    TPiece<T> x[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const uint32_t c = (j * threads + threadIdx.x) * N;
        x[j].From(raw[j]);
        TWords<N> w;
        if (table && c < width) {
            w = TWords<N>(words + c);
            if (w.Any != 0) {
                x[j].Penalize(w, penalties, few ? (1u << kNameShift) - 1 : ~0u);
            }
        }
        if (p.ClassBias != nullptr) {
            x[j].Add(classBias[j]);
        }
        if (BIASES && named > 0 && w.Any >> 31 != 0) {
            x[j].AddNamed(w, biasValues);
        }
        if (!BIASES || few) {
            store(j, x[j]);
        }
    }
    if (BIASES && !few) {
        if (history) {
            __syncthreads();  // the history's words are read
        }
        clear();
        MakeBiases(threads, static_cast<uint32_t>(endBias - firstBias), p.BiasClasses + firstBias, p.BiasValues + firstBias, biasClass, biasValue,
                            [&](uint32_t, int32_t entry) {
                                const uint32_t c = static_cast<uint32_t>(entry) - c0;
                                return c < width ? &words[c] : nullptr;
                            });
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint32_t c = (j * threads + threadIdx.x) * N;
            if (c < width) {
                x[j].Add(words + c);
                store(j, x[j]);
            }
        }
    }
}

// The row that entry `e` of a list with these offsets belongs to: the last one that begins at or before it
template <typename TOffset>
__device__ __forceinline__ uint32_t RowOfEntry(const TOffset* offsets, uint32_t rows, TOffset e) {
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

// f(entry, row, class) for the entries of a tile's rows. A thread takes four entries at a time: it searches for the row of
// the first and goes on from there. `entries`: its first four
template <typename F>
__device__ __forceinline__ void ForEntries(const int64_t* offsets, uint32_t rows, int64_t begin, int64_t end, const int32_t* list, size_t count,
                                           TValues<int32_t, 4> entries, F&& f) {
    for (int64_t e = begin + threadIdx.x * 4; e < end;) {
        const int64_t next = e + 256 * 4;
        TValues<int32_t, 4> more{};
        if (next < end) {
            more = LoadEntries(list, next, count);
        }
        uint32_t r = RowOfEntry(offsets, rows, e);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (e + i < end) {
                while (r + 1 < rows && offsets[r + 1] <= e + i) {
                    ++r;
                }
                f(e + i, r, static_cast<uint32_t>(entries.V[i]));
            }
        }
        entries = more;
        e = next;
    }
}

// Rows that are shorter than a slice: a workgroup for RowsPerTile of them, P pieces for a thread. Pieces are taken in the
// order in which they are in memory, whatever the rows' length, so that a wave's stores fill whole lines (a thread for a
// row, at ten 64-bit values each, wrote 413 MB for 160). What is read is requested first, as in the kernel above. A row's first entries
// are counted by lanes of its own, which know whose they are; a search for the row of each (all threads of the tile, as for what is
// left of long histories) took 73 us for 2M x 10 32-bit scores where these took 65 (60 with smaller tables). Memory bounds it: 2M x 10 64-bit scores with histories,
// biases of classes and masks take 83 us (4.8 TB/s).
template <typename T>
constexpr int kPiecesPerThread = sizeof(T) == 2 ? 2 : 4;  // 16 scores on their way, 8 of 64 bits

enum ERests {
    kNoRests,       // rows are whole pieces
    kRests,         // a row's last piece may have less than N values
    kLessThanOne,   // the only piece of a row has
};

// (Eight waves a SIMD, seven where the 64 registers of those would spill: 2M x 10 32-bit scores 60 us, with eight 12 more. Kernels with and
// without histories: 2M x 10 64-bit scores without one 60 us, 74 by a kernel of both.)
template <typename T, int RESTS, bool HISTORY, bool BIASES>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(sizeof(T) > 2 && HISTORY ? 7 : 8))) AdjustRowsKernel(TAdjustArgs a) {
    constexpr int N = 16 / sizeof(T), P = kPiecesPerThread<T>;
    extern __shared__ uint4 tables[];
    const CbHipScoreAdjustment& p = a.A;
    constexpr bool history = HISTORY;
    const uint32_t pitch = a.Pieces * N;
    // (in the order of their alignments: a piece's words, 8 bytes, 4)
    uint32_t* words = reinterpret_cast<uint32_t*>(tables);
    TPenalties* penalties = reinterpret_cast<TPenalties*>(words + a.RowsPerTile * pitch);
    int64_t* offsets = reinterpret_cast<int64_t*>(penalties + (history ? a.RowsPerTile : 0));
    int32_t* given = reinterpret_cast<int32_t*>(offsets + (history ? a.RowsPerTile : 0));  // how many of a row's entries are
    uint32_t* biasOffsets = reinterpret_cast<uint32_t*>(given + (history ? a.RowsPerTile : 0));  // from the tile's first on
    float* biasValues = reinterpret_cast<float*>(biasOffsets + (BIASES ? a.RowsPerTile : 0));
    uint32_t* more = reinterpret_cast<uint32_t*>(biasValues + (BIASES ? kNamedBiases : 0));  // a row has a longer history
    const auto rowOf = [&](uint32_t q) { return a.PiecesInverse != 0 ? __umulhi(q, a.PiecesInverse) : q; };
    const size_t tile = a.FirstTile + blockIdx.x;
    const size_t r0 = tile * a.RowsPerTile;
    const uint32_t rows = static_cast<uint32_t>(a.Rows - r0 < a.RowsPerTile ? a.Rows - r0 : a.RowsPerTile);
    const auto clear = [&] {
        for (uint32_t i = threadIdx.x; i < rows * a.Pieces; i += 256) {
            TWords<N>::Clear(words + i * N);
        }
    };
    int64_t begin = 0, end = 0, firstBias = 0, endBias = 0;
    // a row's first entries are counted by lanes of its own, which know whose they are: this thread's row, where its history begins, how long it
    // is and how much of it is given
    const uint32_t rowLanes = 1u << a.RowLanesLog2, myRow = threadIdx.x >> a.RowLanesLog2, myLane = threadIdx.x & (rowLanes - 1);
    int64_t myBegin = 0;
    int32_t myLength = 0, myGiven = 0;
    const auto loadOffsets = [&](uint32_t i) {
        const size_t r = r0 + min(i, rows - 1);
        const int64_t first = p.HistoryOffsets[r];
        myBegin = Clamped(first, p.HistoryCount);
        myLength = static_cast<int32_t>(Clamped(p.HistoryOffsets[r + 1], p.HistoryCount) - myBegin);
        const int64_t end = first + (p.PromptLengths != nullptr ? p.PromptLengths[r] : 0);
        myGiven = static_cast<int32_t>(max(min(end - myBegin, int64_t(0x7fffffff)), int64_t(0)));
        if (myLane == 0 && i < rows) {
            offsets[i] = myBegin;
            given[i] = myGiven;
            penalties[i] = TPenalties::Of(p, r);
        }
    };
    if (history) {
        begin = Clamped(p.HistoryOffsets[r0], p.HistoryCount);
        end = Clamped(p.HistoryOffsets[r0 + rows], p.HistoryCount);
    }
    if (BIASES) {
        firstBias = Clamped(p.BiasOffsets[r0], p.BiasCount);
        endBias = max(firstBias, Clamped(p.BiasOffsets[r0 + rows], p.BiasCount));
    }
    // a thread whose pieces are behind the tile's last row reads that row's instead
    int32_t mask[P];
    uint32_t allowed[P];
    TRaw raw[P];
    if (p.AllowedRows != nullptr) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            mask[j] = p.AllowedRows[r0 + min(rowOf(j * 256 + threadIdx.x), rows - 1)];
        }
    }
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const uint32_t q = j * 256 + threadIdx.x, r = rowOf(q), c = (q - r * a.Pieces) * N;
        const T* from = static_cast<const T*>(a.Scores) + (r0 + min(r, rows - 1)) * a.ScoreStride + c;
        raw[j] = RESTS == kNoRests ? TRaw::Load(from)
            : RESTS == kRests ? LoadShifted<T>(from, a.Classes - c) : LoadPiece<T>(from, a.Classes - c);
    }
    if (p.AllowedCount != 0) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint32_t q = j * 256 + threadIdx.x, r = rowOf(q), c = (q - r * a.Pieces) * N;
            size_t m = r0 + min(r, rows - 1);
            if (p.AllowedRows != nullptr) {
                const bool some = mask[j] >= 0 && static_cast<size_t>(mask[j]) < p.AllowedCount;
                m = some ? mask[j] : 0;
                mask[j] = some;
            }
            allowed[j] = p.Allowed[m * p.AllowedStride + (c >> 5)];
        }
    }
    int32_t biasClass = 0;
    float biasValue = 0;
    if (firstBias + threadIdx.x < endBias) {
        biasClass = p.BiasClasses[firstBias + threadIdx.x];
        biasValue = p.BiasValues[firstBias + threadIdx.x];
    }
    const auto loadBiasOffsets = [&] {
        for (uint32_t i = threadIdx.x; i < rows; i += 256) {
            biasOffsets[i] = static_cast<uint32_t>(max(Clamped(p.BiasOffsets[r0 + i], p.BiasCount) - firstBias, int64_t(0)));
        }
    };
    const bool few = BIASES && endBias - firstBias <= kNamedBiases && end - begin < kNamedHistory;
    const uint32_t named = few ? static_cast<uint32_t>(endBias - firstBias) : 0;
    const bool table = history || named > 0;
    if (table) {
        TValues<int32_t, 4> entries{};
        const auto loadEntries = [&](uint32_t i) {
            if (i < rows && static_cast<int32_t>(myLane * 4) < myLength) {
                entries = LoadEntries(p.History, myBegin + myLane * 4, p.HistoryCount);
            }
        };
        if (history) {
            loadOffsets(myRow);
            loadEntries(myRow);
        }
        clear();
        if (threadIdx.x == 0) {
            *more = 0;
        }
        if (BIASES) {
            loadBiasOffsets();
        }
        __syncthreads();
        if (named > 0) {
            for (uint32_t i = threadIdx.x; i < named; i += 256) {
                const bool first = i == threadIdx.x;
                const uint32_t c = static_cast<uint32_t>(first ? biasClass : p.BiasClasses[firstBias + i]);
                if (c < a.Classes) {
                    // the last one of a class stays
                    atomicMax(&words[RowOfEntry(biasOffsets, rows, i) * pitch + c], 1u << 31 | i << kNameShift);
                }
                biasValues[i] = first ? biasValue : p.BiasValues[firstBias + i];
            }
            __syncthreads();
        }
        if (history) {
            for (uint32_t i = myRow; i < rows; i += 256 >> a.RowLanesLog2) {
                if (i != myRow) {
                    loadOffsets(i);
                    loadEntries(i);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int32_t e = myLane * 4 + k;
                    const uint32_t c = static_cast<uint32_t>(entries.V[k]);
                    if (e < myLength && c < a.Classes) {
                        CountEntry(&words[i * pitch + c], e < myGiven);
                    }
                }
                if (myLength > static_cast<int32_t>(4 * rowLanes)) {
                    *more = 1;
                }
            }
            __syncthreads();
            if (*more != 0) {
                // the others by all threads
                TValues<int32_t, 4> four{};
                if (begin + threadIdx.x * 4 < end) {
                    four = LoadEntries(p.History, begin + threadIdx.x * 4, p.HistoryCount);
                }
                ForEntries(offsets, rows, begin, end, p.History, p.HistoryCount, four, [&](int64_t e, uint32_t i, uint32_t c) {
                    if (c < a.Classes && e - offsets[i] >= 4 * rowLanes) {
                        CountEntry(&words[i * pitch + c], e - offsets[i] < given[i]);
                    }
                });
                __syncthreads();
            }
        }
    }
    TValues<float, N> classBias[P];
    if (p.ClassBias != nullptr) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint32_t q = j * 256 + threadIdx.x, r = rowOf(q), c = (q - r * a.Pieces) * N;
            const float* bias = p.ClassBias + (r0 + min(r, rows - 1)) * p.ClassBiasStride;
            classBias[j] = RESTS == kNoRests ? TValues<float, N>::Load(bias + c) : LoadUpTo<float, N>(bias + c, a.Classes - c);
        }
    }
    const auto store = [&](int j, const TPiece<T>& x) {
        const uint32_t q = j * 256 + threadIdx.x, r = rowOf(q), c = (q - r * a.Pieces) * N;
        if (r < rows) {
            const bool masked = p.AllowedCount != 0 && (p.AllowedRows == nullptr || mask[j] != 0);
            const TRaw out = x.Rounded(masked ? allowed[j] >> (c & 31) : ~0u);
            T* to = static_cast<T*>(a.Result) + (r0 + r) * a.ResultStride + c;
            if (RESTS == kNoRests) {
                out.Store(to);
            } else {
                StorePiece<T>(out, to, a.Classes - c);
            }
        }
    };
    TPiece<T> x[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
        const uint32_t q = j * 256 + threadIdx.x, r = rowOf(q);
        x[j].From(raw[j]);
        TWords<N> w;
        if (table && r < rows) {
            w = TWords<N>(words + q * N);
            if (history && w.Any != 0) {
                x[j].Penalize(w, penalties[r], few ? (1u << kNameShift) - 1 : ~0u);
            }
        }
        if (p.ClassBias != nullptr) {
            x[j].Add(classBias[j]);
        }
        if (BIASES && named > 0 && w.Any >> 31 != 0) {
            x[j].AddNamed(w, biasValues);
        }
        if (!BIASES || few) {
            store(j, x[j]);
        }
    }
    if (BIASES && !few) {
        if (history) {
            __syncthreads();  // the history's words are read
        } else {
            loadBiasOffsets();
        }
        clear();
        __syncthreads();
        MakeBiases(256, static_cast<uint32_t>(endBias - firstBias), p.BiasClasses + firstBias, p.BiasValues + firstBias, biasClass, biasValue,
                        [&](uint32_t i, int32_t entry) {
                            const uint32_t c = static_cast<uint32_t>(entry);
                            return c < a.Classes ? &words[RowOfEntry(biasOffsets, rows, i) * pitch + c] : nullptr;
                        });
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const uint32_t q = j * 256 + threadIdx.x;
            if (rowOf(q) < rows) {
                x[j].Add(words + q * N);
                store(j, x[j]);
            }
        }
    }
}

// ---------------------------------------------------------------- the best classes ----

// A score with its class as one value that orders them: larger scores first, of equal ones the lower class first. What is
// never selected (minus infinity, NaN) comes behind all others. 16-bit scores and their class fit 32 bits, 32-bit ones 64.
template <typename T>
struct TRanked;

template <>
struct TRanked<float> {
    uint64_t K;

    __device__ __forceinline__ static TRanked None() { return {0}; }
    __device__ __forceinline__ static TRanked Of(float x, uint32_t c) {
        uint32_t bits = __float_as_uint(x + 0.f);  // zeros of both signs are equal
        bits ^= static_cast<uint32_t>(static_cast<int32_t>(bits) >> 31) | 0x80000000u;
        return {x > -std::numeric_limits<float>::infinity() ? static_cast<uint64_t>(bits) << 32 | ~c : 0};
    }
    __device__ __forceinline__ bool IsNone() const { return K == 0; }
    __device__ __forceinline__ uint32_t Class() const { return ~static_cast<uint32_t>(K); }
    __device__ __forceinline__ float Score() const {
        const uint32_t bits = static_cast<uint32_t>(K >> 32);
        return IsNone() ? -std::numeric_limits<float>::infinity() : __uint_as_float(bits ^ (static_cast<uint32_t>(static_cast<int32_t>(~bits) >> 31) | 0x80000000u));
    }
    __device__ __forceinline__ TRanked Better(const TRanked& other) const { return {other.K > K ? other.K : K}; }
    // the same for an `other` whose class is the higher one
    __device__ __forceinline__ TRanked BetterLater(const TRanked& other) const { return Better(other); }
    __device__ __forceinline__ TRanked Without(const TRanked& other) const { return {K == other.K ? 0 : K}; }
    __device__ __forceinline__ TRanked Or(const TRanked& other, bool take) const { return {take ? other.K : K}; }
};

// The upper half: the score as a number that has its order and is 0 for minus infinity. It is made of the magnitude with the
// sign (zeros of both signs are equal), from which that of minus infinity is taken with a stop at 0, for two scores at a time.
template <typename T>
struct TRanked16 {
    static constexpr uint32_t kInfinity = std::is_same_v<T, _Float16> ? 0x7c00 : 0x7f80;
    uint32_t K;

    __device__ __forceinline__ static TRanked16 None() { return {0}; }
    __device__ __forceinline__ static TRanked16 Of(T x, uint32_t c) {
        const uint32_t bits = __builtin_bit_cast(uint16_t, x), magnitude = bits & 0x7fff;
        const uint32_t order = (bits & 0x8000) != 0 ? kInfinity - min(magnitude, kInfinity) : kInfinity + magnitude;
        return {magnitude > kInfinity || order == 0 ? 0 : order << 16 | (~c & 0xffff)};
    }
    __device__ __forceinline__ bool IsNone() const { return K < 0x10000; }
    __device__ __forceinline__ uint32_t Class() const { return ~K & 0xffff; }
    __device__ __forceinline__ float Score() const {
        const int32_t order = static_cast<int32_t>(K >> 16) - static_cast<int32_t>(kInfinity);
        const uint16_t bits = order < 0 ? static_cast<uint16_t>(0x8000 - order) : static_cast<uint16_t>(order);
        return static_cast<float>(__builtin_bit_cast(T, bits));
    }
    __device__ __forceinline__ TRanked16 Better(const TRanked16& other) const { return {max(K, other.K)}; }
    __device__ __forceinline__ TRanked16 BetterLater(const TRanked16& other) const { return Better(other); }
    __device__ __forceinline__ TRanked16 Without(const TRanked16& other) const { return {K == other.K ? 0 : K}; }
    __device__ __forceinline__ TRanked16 Or(const TRanked16& other, bool take) const { return {take ? other.K : K}; }
};
template <>
struct TRanked<_Float16> : TRanked16<_Float16> {
    __device__ __forceinline__ TRanked() {}
    __device__ __forceinline__ TRanked(const TRanked16<_Float16>& x) : TRanked16<_Float16>(x) {}
};
template <>
struct TRanked<__bf16> : TRanked16<__bf16> {
    __device__ __forceinline__ TRanked() {}
    __device__ __forceinline__ TRanked(const TRanked16<__bf16>& x) : TRanked16<__bf16>(x) {}
};

// A lane's V scores from class c on, of which those before `classes` count (all of every lane's, if `full`)
// (Those of 16 bits in pairs as they are in memory: single ones would take a register each.)
template <typename T, int V>
using TLaneScores = std::conditional_t<sizeof(T) == 2 && V % 2 == 0, TValues<uint32_t, (V + 1) / 2>, TValues<T, V>>;

template <typename T, int V>
__device__ __forceinline__ TLaneScores<T, V> LoadLane(const T* at, uint32_t c, uint32_t classes, bool full) {
    TLaneScores<T, V> raw{};
    if (full) {
        __builtin_memcpy(&raw, at + c, sizeof(raw));
    } else if (c < classes) {
        const TValues<T, V> v = LoadUpTo<T, V>(at + c, classes - c);
        __builtin_memcpy(&raw, &v, sizeof(raw));
    }
    return raw;
}

template <typename T, int V>
__device__ __forceinline__ void Rank(const TLaneScores<T, V>& v, uint32_t c, uint32_t classes, bool full, TRanked<T> (&ranked)[V]) {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
        using TPair = uint16_t __attribute__((ext_vector_type(2)));
        constexpr uint16_t infinity = TRanked<T>::kInfinity;
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const uint32_t bits = v.V[j / 2];
            const TPair sign = __builtin_bit_cast(TPair, bits) >> uint16_t(15);                       // 0 or 1
            const uint32_t negative = __builtin_bit_cast(uint32_t, static_cast<TPair>(TPair(0) - sign));  // 0 or all bits
            const TPair magnitude = __builtin_bit_cast(TPair, (bits & 0x7fff7fffu) ^ negative) + sign;
            // from minus the largest magnitude on up, and then from minus infinity
            const TPair order = __builtin_elementwise_sub_sat(static_cast<TPair>(magnitude + uint16_t(0x8000)), TPair(uint16_t(0x8000 - infinity)));
            const uint32_t both = __builtin_bit_cast(uint32_t, order);
            ranked[j].K = both << 16 | (~(c + j) & 0xffff);
            ranked[j + 1].K = (both & 0xffff0000u) | (~(c + j + 1) & 0xffff);
            most = max(most, max(ranked[j].K, ranked[j + 1].K));
        }
        if (!full) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ranked[j].K = c + j < classes ? ranked[j].K : 0;
            }
        }
        if (most >> 16 > 2 * uint32_t(infinity)) {  // NaN of the sign that comes behind infinity
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ranked[j].K = ranked[j].K >> 16 > 2 * uint32_t(infinity) ? 0 : ranked[j].K;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            ranked[j] = c + j < classes ? TRanked<T>::Of(v.V[j], c + j) : TRanked<T>::None();
        }
    }
}

// Larger keys first, by exchanges in a fixed order
template <typename R>
__device__ __forceinline__ void Sort8(R (&r)[8]) {
    constexpr int pairs[19][2] = {{0, 1}, {2, 3}, {4, 5}, {6, 7}, {0, 2}, {1, 3}, {4, 6}, {5, 7}, {1, 2}, {5, 6},
                                  {0, 4}, {1, 5}, {2, 6}, {3, 7}, {2, 4}, {3, 5}, {1, 2}, {3, 4}, {5, 6}};
#pragma unroll
    for (int i = 0; i < 19; ++i) {
        const uint32_t x = r[pairs[i][0]].K, y = r[pairs[i][1]].K;
        r[pairs[i][0]].K = max(x, y);
        r[pairs[i][1]].K = min(x, y);
    }
}

template <>
struct TRanked<double> {
    uint32_t Words[2];  // of the score (with a double here, the padding behind C kept arrays of these out of registers)
    uint32_t C;

    __device__ __forceinline__ TRanked() {}
    __device__ __forceinline__ TRanked(double x, uint32_t c)
        : C(c)
    {
        __builtin_memcpy(Words, &x, 8);
    }
    __device__ __forceinline__ static TRanked None() { return {-std::numeric_limits<double>::infinity(), ~0u}; }
    __device__ __forceinline__ static TRanked Of(double x, uint32_t c) {
        const bool usable = x > -std::numeric_limits<double>::infinity();
        return {usable ? x : -std::numeric_limits<double>::infinity(), usable ? c : ~0u};
    }
    __device__ __forceinline__ bool IsNone() const { return C == ~0u; }
    __device__ __forceinline__ uint32_t Class() const { return C; }
    __device__ __forceinline__ double Score() const {
        double x;
        __builtin_memcpy(&x, Words, 8);
        return x;
    }
    __device__ __forceinline__ TRanked Or(const TRanked& other, bool take) const { return {take ? other.Score() : Score(), take ? other.C : C}; }
    __device__ __forceinline__ TRanked Better(const TRanked& other) const {
        return Or(other, other.Score() > Score() || (other.Score() == Score() && other.C < C));
    }
    __device__ __forceinline__ TRanked BetterLater(const TRanked& other) const { return Or(other, other.Score() > Score()); }
    __device__ __forceinline__ TRanked Without(const TRanked& other) const { return Or(None(), C == other.C); }
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
// lane's own, then over the group; whoever has it takes it out. Lane k % G keeps what round k finds. Arithmetic bounds it: 131072
// rows, 8 of 128 16-bit classes take 15 us, for 42 MB.
template <typename T, int G, int V>
__global__ void __launch_bounds__(256) SelectTopKernel(TTopArgs<T> a, int32_t* indexes, TAcc<T>* weights) {
    using A = TAcc<T>;
    using R = TRanked<T>;
    constexpr int kept = 32 / G > 0 ? 32 / G : 1;
    const uint32_t lane = threadIdx.x & (G - 1);
    const size_t row = size_t(blockIdx.x) * (256 / G) + threadIdx.x / G;
    if (row >= a.Rows) {
        return;
    }
    const uint32_t c = lane * V;
    const bool full = a.Classes == G * V;
    R left[V];
    Rank<T, V>(LoadLane<T, V>(a.Scores + row * a.Stride, c, a.Classes, full), c, a.Classes, full, left);
    // eight 32-bit keys of a lane are sorted first: a round's best is then the first, and taking it out moves the others up
    constexpr bool sorted = sizeof(T) == 2 && V == 8;
    if constexpr (sorted) {
        Sort8(left);
    }
    R mine[kept];
#pragma unroll
    for (int i = 0; i < kept; ++i) {
        mine[i] = R::None();
    }
    A most = 0, total = 0;
    // `keys`: of a lane's sorted ones, how many later rounds may ask for
    const auto round = [&](uint32_t k, int keys) {
        R best = left[0];
        if constexpr (!sorted) {
#pragma unroll
            for (int j = 1; j < V; ++j) {
                best = best.BetterLater(left[j]);
            }
        }
        best = OverGroup<G>(best, [](const R& x, const R& y) { return x.Better(y); });
        if (k == 0) {
            most = best.Score();
            if (!a.Among) {
                // (what is never selected has a weight of 0; where nothing else is there the sum is not used)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    total += WeightOf(left[j].Score(), most);
                }
            }
        }
        if constexpr (sorted) {
            const bool taken = left[0].K == best.K;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (j < keys) {
                    left[j] = j + 1 < V ? left[j].Or(left[j + 1 < V ? j + 1 : 0], taken) : left[j].Or(R::None(), taken);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                left[j] = left[j].Without(best);
            }
        }
#pragma unroll
        for (int i = 0; i < kept; ++i) {
            if (i * G < a.Count) {
                mine[i] = mine[i].Or(best, k == lane + i * G);
            }
        }
    };
    if (sorted && a.Count <= V) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (static_cast<uint32_t>(k) < a.Count) {
                round(k, V - 1 - k);
            }
        }
    } else {
        for (uint32_t k = 0; k < a.Count; ++k) {
            round(k, V);
        }
    }
    A e[kept];
#pragma unroll
    for (int i = 0; i < kept; ++i) {
        e[i] = 0;
        if (i * G < a.Count) {
            e[i] = mine[i].IsNone() ? A(0) : WeightOf(mine[i].Score(), most);
            total += a.Among ? e[i] : A(0);
        }
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

// Rows of C classes, a thread for each. What is stored goes through LDS, so that a wave's stores fill whole lines. Memory bounds it:
// 2M rows, 3 of 10 64-bit classes take 54 us (4.3 TB/s).
template <typename T, int C>
__global__ void __launch_bounds__(256) SelectTopOfFewKernel(TTopArgs<T> a, int32_t* indexes, TAcc<T>* weights) {
    using A = TAcc<T>;
    using R = TRanked<T>;
    extern __shared__ uint4 tables[];
    A* outWeights = reinterpret_cast<A*>(tables);
    int32_t* outIndexes = reinterpret_cast<int32_t*>(outWeights + 256 * a.Count);
    const size_t r0 = size_t(blockIdx.x) * 256;
    const uint32_t rows = static_cast<uint32_t>(a.Rows - r0 < 256 ? a.Rows - r0 : 256);
    if (threadIdx.x < rows) {
        R left[C];
        Rank<T, C>(LoadLane<T, C>(a.Scores + (r0 + threadIdx.x) * a.Stride, 0, C, true), 0, C, true, left);
        A* myWeights = outWeights + threadIdx.x * a.Count;
        int32_t* myIndexes = outIndexes + threadIdx.x * a.Count;
        R first = left[0];
#pragma unroll
        for (int j = 1; j < C; ++j) {
            first = first.BetterLater(left[j]);
        }
        const A most = first.Score();
        A total = 0;
        if (!a.Among) {
            // (what is never selected has a weight of 0; where nothing else is there the sum is not used)
#pragma unroll
            for (int j = 0; j < C; ++j) {
                total += WeightOf(left[j].Score(), most);
            }
        }
        for (uint32_t k = 0; k < a.Count; ++k) {
            R best = left[0];
#pragma unroll
            for (int j = 1; j < C; ++j) {
                best = best.BetterLater(left[j]);
            }
#pragma unroll
            for (int j = 0; j < C; ++j) {
                left[j] = left[j].Without(best);
            }
            const A e = best.IsNone() ? A(0) : k == 0 ? A(1) : WeightOf(best.Score(), most);
            myIndexes[k] = best.IsNone() ? -1 : static_cast<int32_t>(best.Class());
            myWeights[k] = e;
            total += a.Among ? e : A(0);
        }
        for (uint32_t k = 0; k < a.Count; ++k) {
            myWeights[k] = myIndexes[k] < 0 ? A(0) : myWeights[k] / total;
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < rows * a.Count; i += 256) {
        indexes[r0 * a.Count + i] = outIndexes[i];
        weights[r0 * a.Count + i] = outWeights[i];
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
// G lanes for a row, which take its pieces of 16 bytes in turn, V classes each in all (V next to each other instead took 43 us for
// 131072 rows of 256 32-bit classes, and these 20). The gradients are put together in LDS, where the selected classes' lanes add
// their parts. Memory bounds it: 8 of 128 16-bit classes 9.5 us for 46 MB, which the caches still have in part.
template <typename T, int G, int V>
__global__ void __launch_bounds__(256) SelectTopBackwardKernel(TTopArgs<T> a, TTopGradientArgs<T> b) {
    using A = TAcc<T>;
    constexpr int kept = 32 / G > 0 ? 32 / G : 1;
    constexpr int N = V * sizeof(T) <= 16 ? V : 16 / sizeof(T), P = V / N;
    __shared__ __align__(16) A sums[256 * V];
    const uint32_t lane = threadIdx.x & (G - 1);
    A* mySums = sums + threadIdx.x / G * (G * V);
    const size_t row = size_t(blockIdx.x) * (256 / G) + threadIdx.x / G;
    if (row >= a.Rows) {
        return;
    }
    const auto classOf = [&](int i) { return (i * G + lane) * N; };
    const bool full = a.Classes == G * V;
    TValues<T, N> v[P]{};
    if (!a.Among) {
        const T* scores = a.Scores + row * a.Stride;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (full) {
                v[i] = TValues<T, N>::Load(scores + classOf(i));
            } else if (classOf(i) < a.Classes) {
                v[i] = LoadUpTo<T, N>(scores + classOf(i), a.Classes - classOf(i));
            }
        }
    }
    // (a lane without a slot reads the last one's, so that no load waits for another)
    int32_t index[kept];
    A w[kept], g[kept], part[kept], mean = 0;
#pragma unroll
    for (int i = 0; i < kept; ++i) {
        const size_t at = row * a.Count + min(lane + i * G, a.Count - 1);
        index[i] = b.Indexes[at];
        w[i] = b.Weights[at];
        g[i] = b.WeightGradients[at];
    }
#pragma unroll
    for (int i = 0; i < kept; ++i) {
        index[i] = lane + i * G < a.Count ? index[i] : -1;
        mean += index[i] >= 0 ? w[i] * g[i] : A(0);
    }
    mean = GroupSum<G>(mean);
#pragma unroll
    for (int i = 0; i < kept; ++i) {
        part[i] = a.Among ? w[i] * (g[i] - mean) : w[i] * g[i];
    }
    TValues<A, N> x[P]{};
    if (!a.Among) {
        A most = -std::numeric_limits<A>::infinity();
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const A s = static_cast<A>(v[i].V[j]);
                x[i].V[j] = classOf(i) + j < a.Classes && s == s ? s : -std::numeric_limits<A>::infinity();
                most = x[i].V[j] > most ? x[i].V[j] : most;
            }
        }
        most = OverGroup<G>(most, [](A y, A z) { return z > y ? z : y; });
        A total = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[i].V[j] = x[i].V[j] > -std::numeric_limits<A>::infinity() ? WeightOf(x[i].V[j], most) : A(0);
                total += x[i].V[j];
            }
        }
        total = GroupSum<G>(total);
#pragma unroll
        for (int i = 0; i < P; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                x[i].V[j] = total > 0 ? -(x[i].V[j] / total) * mean : A(0);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
        x[i].Store(mySums + classOf(i));
    }
    WaveHandover();  // a row's lanes are of one wave
#pragma unroll
    for (int i = 0; i < kept; ++i) {
        if (static_cast<uint32_t>(index[i]) < a.Classes) {
            mySums[index[i]] += part[i];
        }
    }
    WaveHandover();
    T* gradients = b.Gradients + row * b.GradientStride;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        x[i] = TValues<A, N>::Load(mySums + classOf(i));
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[i].V[j] = static_cast<T>(x[i].V[j]);
        }
        if (full) {
            v[i].Store(gradients + classOf(i));
        } else if (classOf(i) < a.Classes) {
            StoreUpTo<T, N>(v[i], gradients + classOf(i), a.Classes - classOf(i));
        }
    }
}

// Rows of C classes, a thread for each. What is loaded and stored goes through LDS (a thread that loaded its own row's selected
// classes, one after the other, took 76 us for 262144 rows, 8 of 16 64-bit classes selected). Memory bounds it: 2M rows, 3 of 10 64-bit
// classes over all take 86 us (5.1 TB/s).
template <typename T, int C>
__global__ void __launch_bounds__(256) SelectTopOfFewBackwardKernel(TTopArgs<T> a, TTopGradientArgs<T> b) {
    using A = TAcc<T>;
    extern __shared__ uint4 tables[];
    const size_t r0 = size_t(blockIdx.x) * 256;
    const uint32_t rows = static_cast<uint32_t>(a.Rows - r0 < 256 ? a.Rows - r0 : 256);
    const bool there = threadIdx.x < rows;
    TValues<T, C> v{};
    if (!a.Among) {
        v = TValues<T, C>::Load(a.Scores + (r0 + min(threadIdx.x, rows - 1)) * a.Stride);
    }
    A* weights = reinterpret_cast<A*>(tables);
    A* gradients = weights + 256 * a.Count;
    int32_t* indexes = reinterpret_cast<int32_t*>(gradients + 256 * a.Count);
    for (uint32_t i = threadIdx.x; i < rows * a.Count; i += 256) {
        weights[i] = b.Weights[r0 * a.Count + i];
        gradients[i] = b.WeightGradients[r0 * a.Count + i];
        indexes[i] = b.Indexes[r0 * a.Count + i];
    }
    __syncthreads();
    A x[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
        x[j] = 0;
    }
    if (there) {
        const uint32_t first = threadIdx.x * a.Count;
        A mean = 0;
        for (uint32_t k = first; k < first + a.Count; ++k) {
            mean += indexes[k] >= 0 ? weights[k] * gradients[k] : A(0);
        }
        if (!a.Among) {
            A most = -std::numeric_limits<A>::infinity(), total = 0;
#pragma unroll
            for (int j = 0; j < C; ++j) {
                const A s = static_cast<A>(v.V[j]);
                x[j] = s == s ? s : -std::numeric_limits<A>::infinity();
                most = x[j] > most ? x[j] : most;
            }
#pragma unroll
            for (int j = 0; j < C; ++j) {
                x[j] = WeightOf(x[j], most);
                total += x[j];
            }
            const bool some = most > -std::numeric_limits<A>::infinity();
#pragma unroll
            for (int j = 0; j < C; ++j) {
                x[j] = some ? -(x[j] / total) * mean : A(0);
            }
        }
        for (uint32_t k = first; k < first + a.Count; ++k) {
            const int32_t index = indexes[k];
            const A part = index >= 0 ? weights[k] * (a.Among ? gradients[k] - mean : gradients[k]) : A(0);
#pragma unroll
            for (int j = 0; j < C; ++j) {
                x[j] += index == j ? part : A(0);
            }
        }
    }
    __syncthreads();  // what was loaded is read: the gradients have its place
    T* out = reinterpret_cast<T*>(tables);
    if (there) {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            out[threadIdx.x * C + j] = static_cast<T>(x[j]);
        }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < rows * C; i += 256) {
        const uint32_t r = i / C;
        b.Gradients[(r0 + r) * b.GradientStride + (i - r * C)] = out[i];
    }
}

}  // namespace op

using namespace op;

namespace {

// One for each compute unit (64 x 50021 32-bit scores 8.1 us, 9.5 where two were wanted; 512 x 2000: 4.4, 5.9 where half were)
constexpr size_t kWorkgroupsWanted = 256;
constexpr size_t kTilesPerLaunch = 1u << 21;  // 2^31 threads

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
    if (p.Allowed == nullptr) {
        a.A.AllowedCount = 0;
    }
    const TCallDevice call(result, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        constexpr uint32_t N = 16 / sizeof(T);
        // a workgroup has one tile: a loop over tiles in the kernels kept their arguments in registers all along
        const auto launchTiles = [&](auto kernel, size_t tiles, uint32_t threads, size_t lds) {
            for (a.FirstTile = 0; a.FirstTile < tiles; a.FirstTile += kTilesPerLaunch) {
                call.Launch(kernel, std::min(tiles - a.FirstTile, kTilesPerLaunch), threads, lds, a);
            }
        };
        const uint32_t pieces = (a.Classes + N - 1) / N;
        constexpr uint32_t tilePieces = kPiecesPerThread<T> * 256;
        // rows that a tile holds eight of (48000 x 1000 16-bit scores: 54 us as a slice for each, 72 in tiles of 4 rows; 160000 x 300: 97 in tiles of
        // 13, as slices the same)
        if (pieces <= tilePieces / 8) {
            a.Pieces = pieces;
            a.RowsPerTile = static_cast<uint32_t>(std::min<size_t>(tilePieces / pieces, rows));
            // floor(q / pieces) = floor(q m / 2^32) with m = floor(2^32 / pieces) + 1: q m / 2^32 is over q / pieces by q / 2^32 at most, and
            // q / pieces is under the next integer by 1 / pieces at least, which is more for the q and pieces under 2^11 here
            a.PiecesInverse = pieces > 1 ? static_cast<uint32_t>((uint64_t(1) << 32) / pieces + 1) : 0;
            const size_t tiles = (rows + a.RowsPerTile - 1) / a.RowsPerTile;
            const size_t perRow = (history ? sizeof(TPenalties) + 12 : 0) + (biases ? 4 : 0) + (history || biases ? size_t(pieces) * N * 4 : 0);
            const size_t lds = history || biases ? a.RowsPerTile * perRow + 4 + (biases ? kNamedBiases * 4 : 0) : 0;
            a.RowLanesLog2 = 0;
            while ((a.RowsPerTile << (a.RowLanesLog2 + 1)) <= 256) {
                ++a.RowLanesLog2;
            }
            const auto launch = [&](auto kernel) {
                call.AllowLds(reinterpret_cast<const void*>(kernel), lds);
                launchTiles(kernel, tiles, 256, lds);
            };
            const auto withBiases = [&](auto rests) {
                constexpr int RESTS = decltype(rests)::value;
                if (history) {
                    biases ? launch(AdjustRowsKernel<T, RESTS, true, true>) : launch(AdjustRowsKernel<T, RESTS, true, false>);
                } else {
                    biases ? launch(AdjustRowsKernel<T, RESTS, false, true>) : launch(AdjustRowsKernel<T, RESTS, false, false>);
                }
            };
            if (a.Classes % N == 0) {
                withBiases(std::integral_constant<int, kNoRests>());
            } else if (a.Classes > N) {
                withBiases(std::integral_constant<int, kRests>());
            } else {
                withBiases(std::integral_constant<int, kLessThanOne>());
            }
            return;
        }
        const auto slices = [&](uint32_t size) { return (a.Classes + size - 1) / size; };
        const auto launch = [&](uint32_t size, auto perThread) {
            constexpr int P = decltype(perThread)::value;
            a.Slices = slices(size);
            a.SliceClasses = ((a.Classes + a.Slices - 1) / a.Slices + 31) / 32 * 32;  // masks begin with a word
            a.Slices = slices(a.SliceClasses);
            // as many threads as a slice has work for, more where long histories are looked through (384 rows of 100003 with 12000 entries:
            // 85 us with 1024 threads, 89 with 896; 1411 of 17000 with 50: 48 with 1024, 44 with 576)
            const bool longHistory = history && p.HistoryCount / rows > a.SliceClasses / 2;
            const uint32_t threads = longHistory ? size / (P * N) : ((a.SliceClasses + P * N - 1) / (P * N) + 63) / 64 * 64;
            const size_t lds = (history || biases ? a.SliceClasses * 4 : 0) + (biases ? kNamedBiases * 4 : 0);
            const auto launchSlices = [&](auto kernel) {
                call.AllowLds(reinterpret_cast<const void*>(kernel), lds);
                launchTiles(kernel, rows * a.Slices, threads, lds);
            };
            if (biases) {
                launchSlices(AdjustSliceKernel<T, P, true>);
            } else {
                launchSlices(AdjustSliceKernel<T, P, false>);
            }
        };
        // the longest slices that a row fills at least half of one of and of which there are workgroups enough
        const auto suits = [&](uint32_t size) {
            return a.Classes > size / 2 && rows >= (kWorkgroupsWanted + slices(size) - 1) / slices(size);
        };
        using std::integral_constant;
        // Slices of 16384 look through a history least often; the tables of two workgroups of 1024 threads fit a compute unit (and their
        // registers: 64-bit scores would not). Where there are slices in plenty and histories are not long, smaller workgroups with as many
        // pieces for a thread as it can hold are the better ones, of which more are at different steps at a time (256 x 50021 32-bit scores:
        // 22.6 us in slices of 8192, 26.4 in slices of 16384; 256 x 131000 of 16 bits with 3000 entries a row: 46 us in slices of 8192, 50 in slices of 16384; with 12000 entries 61 and 60; 64 rows 18 and 17. 9600 x 5000:
        // 64 us in two slices with two pieces for a thread, 103 in one with one).
        const bool plenty = rows >= (4 * kWorkgroupsWanted + slices(8192) - 1) / slices(8192) && (!history || p.HistoryCount / rows <= 4096);
        constexpr int most = kPiecesPerThread<T>;
        if (plenty) {
            launch(a.Classes > 4096 ? 8192 : a.Classes > 2048 ? 4096 : 2048, integral_constant<int, most>());
        } else if (sizeof(T) < 8 && suits(16384)) {
            launch(16384, integral_constant<int, sizeof(T) < 8 ? 16 / N : 1>());
        } else if (suits(8192)) {
            launch(8192, integral_constant<int, 8 / N>());
        } else if (suits(4096)) {
            launch(4096, integral_constant<int, N >= 4 ? 1 : 4 / N>());
        } else {
            launch(2048, integral_constant<int, N >= 2 ? 1 : 2 / N>());
        }
    });
}

namespace {

constexpr size_t kMaxTopClasses = 1024;
constexpr int32_t kMaxTopCount = 32;
constexpr int kClassesForThreads = 16;
struct TForThreads {
    size_t Rows;
    int32_t Count;
};
// (16384 rows of 16 32-bit classes, 8 of them selected: 6.3 us by threads, 4.4 by lanes; 65536: 6.8 and 10.1; a million, 2 of 10: 11.4 and 50)
constexpr TForThreads kForwardByThreads{32768, 8};
// (65536 rows, 2 of 10 32-bit classes: 4.2 us by threads, 3.5 by lanes; 262144: 6.3 and 8.7; 8 of 10: 12.2 and 9.7)
constexpr TForThreads kBackwardByThreads{131072, 4};

void CheckTop(size_t rows, size_t classes, int32_t count) {
    CBAMD_ENSURE(classes <= kMaxTopClasses, "too many classes to select from: " + std::to_string(classes) + ", at most " + std::to_string(kMaxTopClasses));
    CBAMD_ENSURE(count >= 1 && count <= kMaxTopCount, "selected classes per row: " + std::to_string(count) + ", 1 to " + std::to_string(kMaxTopCount) + " are supported");
    CBAMD_ENSURE(classes > 0 || rows == 0, "no classes to select from");
    CBAMD_ENSURE(rows <= size_t(1) << 48, "too many rows");
}

template <typename F, int... C>
bool WithExactClasses(size_t classes, F&& f, std::integer_sequence<int, C...>) {
    return ((classes == C + 1 && (f(std::integral_constant<int, 1>(), std::integral_constant<int, C + 1>()), true)) || ...);
}

// f(lanes of a row, classes of a lane). 1 lane: a thread has a row of exactly so many classes to itself, without branches for
// others. That reads each line of memory once as long as a row is short, and needs rows enough to fill the chip with threads. 16 lanes
// as long as their registers hold the row: sums and best ones of a group cost the same for four rows of a wave as for one (131072 rows
// of 256 32-bit classes, 2 of them selected: 25 us, 42 with 64 lanes; of 64 classes 12 and 33).
template <typename F>
void WithShape(size_t classes, size_t rows, int32_t count, const TForThreads& threads, F&& f) {
    using std::integral_constant;
    if (rows >= threads.Rows && count <= threads.Count && WithExactClasses(classes, f, std::make_integer_sequence<int, kClassesForThreads>())) {
        return;
    }
    const integral_constant<int, 16> sixteen;
    const integral_constant<int, 64> wave;
    return classes <= 16 ? f(sixteen, integral_constant<int, 1>()) : classes <= 32 ? f(sixteen, integral_constant<int, 2>())
        : classes <= 64 ? f(sixteen, integral_constant<int, 4>()) : classes <= 128 ? f(sixteen, integral_constant<int, 8>())
        : classes <= 256 ? f(sixteen, integral_constant<int, 16>()) : classes <= 512 ? f(wave, integral_constant<int, 8>())
        : f(wave, integral_constant<int, 16>());
}

// f(first row, rows) for rows that one launch takes (a workgroup has one tile of them)
template <typename F>
void ForLaunches(size_t rows, F&& f) {
    constexpr size_t most = size_t(1) << 24;
    for (size_t first = 0; first < rows; first += most) {
        f(first, std::min(rows - first, most));
    }
}

size_t GroupsOf(size_t rows, int lanes) {
    const size_t rowsPerGroup = 256 / lanes;
    return (rows + rowsPerGroup - 1) / rowsPerGroup;
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
        WithShape(classes, rows, count, kForwardByThreads, [&](auto lanes, auto perLane) {
            constexpr int G = decltype(lanes)::value, V = decltype(perLane)::value;
            ForLaunches(rows, [&](size_t first, size_t n) {
                const TTopArgs<T> a{static_cast<const T*>(scores) + first * scoreStride, scoreStride, n, static_cast<uint32_t>(classes),
                                    static_cast<uint32_t>(count), amongSelected};
                int32_t* theIndexes = indexes + first * count;
                TAcc<T>* theWeights = static_cast<TAcc<T>*>(weights) + first * count;
                if constexpr (G == 1) {
                    call.Launch(SelectTopOfFewKernel<T, V>, GroupsOf(n, G), 256, size_t(256) * count * (sizeof(TAcc<T>) + 4), a, theIndexes, theWeights);
                } else {
                    call.Launch(SelectTopKernel<T, G, V>, GroupsOf(n, G), 256, 0, a, theIndexes, theWeights);
                }
            });
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
        WithShape(classes, rows, count, kBackwardByThreads, [&](auto lanes, auto perLane) {
            constexpr int G = decltype(lanes)::value, V = decltype(perLane)::value;
            ForLaunches(rows, [&](size_t first, size_t n) {
                const TTopArgs<T> a{static_cast<const T*>(scores) + (amongSelected ? 0 : first * scoreStride), scoreStride, n,
                                    static_cast<uint32_t>(classes), static_cast<uint32_t>(count), amongSelected};
                const TTopGradientArgs<T> b{indexes + first * count, static_cast<const TAcc<T>*>(weights) + first * count,
                                            static_cast<const TAcc<T>*>(weightGradients) + first * count,
                                            static_cast<T*>(scoreGradients) + first * gradientStride, gradientStride};
                if constexpr (G == 1) {
                    const size_t lds = 256 * std::max(count * (2 * sizeof(TAcc<T>) + 4), V * sizeof(T));
                    call.Launch(SelectTopOfFewBackwardKernel<T, V>, GroupsOf(n, G), 256, lds, a, b);
                } else {
                    call.Launch(SelectTopBackwardKernel<T, G, V>, GroupsOf(n, G), 256, 0, a, b);
                }
            });
        });
    });
}

}  // namespace cbamd
