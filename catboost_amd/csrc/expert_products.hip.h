// The experts' products on rows sorted by expert: gated projections and plain ones, with their gradients.
//
// Three forms of one product, out[m][n] = sum over k of a(m, k) * b(n, k), for every expert with rows:
//   rows      out = x W^T:    m a row of the expert, n an output, k an input; both operands have k in a row in memory
//   inputs    dx = dy W:      m a row, n an input, k an output; the weights have n in a row in memory
//   weights   dW = dy^T x:    m an output, n an input, k a row of the expert; both operands have k across their rows
#pragma once

#include "operator_common.hip.h"

#include <algorithm>
#include <type_traits>

namespace cbamd {
namespace op {

constexpr int32_t kMostExperts = 1024;

using TFloat4 = __attribute__((ext_vector_type(4))) float;
using TDouble4 = __attribute__((ext_vector_type(4))) double;
using THalf8 = __attribute__((ext_vector_type(8))) _Float16;
using TBFloat8 = __attribute__((ext_vector_type(8))) __bf16;
using TShort4 = __attribute__((ext_vector_type(4))) short;

// ---------------------------------------------------------------- what differs by type ----

// A fragment is 16 bytes of a lane: its row's (or column's) values k = N * (lane / 16) + i, i < N, of 64 bytes of k. Step:
// out[n][m] += over those 64 bytes; the operand of n comes first, so that a lane ends up with four n of one m.
template <typename T>
struct TMatrix;
template <>
struct TMatrix<_Float16> {
    using TOut = TFloat4;
    __device__ __forceinline__ static TOut Step(uint4 n, uint4 m, TOut out) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(THalf8, n), __builtin_bit_cast(THalf8, m), out, 0, 0, 0);
    }
};
template <>
struct TMatrix<__bf16> {
    using TOut = TFloat4;
    __device__ __forceinline__ static TOut Step(uint4 n, uint4 m, TOut out) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(TBFloat8, n), __builtin_bit_cast(TBFloat8, m), out, 0, 0, 0);
    }
};
template <>
struct TMatrix<float> {
    using TOut = TFloat4;
    __device__ __forceinline__ static TOut Step(uint4 n, uint4 m, TOut out) {
        const TFloat4 a = __builtin_bit_cast(TFloat4, n), b = __builtin_bit_cast(TFloat4, m);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            out = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], out, 0, 0, 0);
        }
        return out;
    }
};
template <>
struct TMatrix<double> {
    using TOut = TDouble4;
    __device__ __forceinline__ static TOut Step(uint4 n, uint4 m, TOut out) {
        struct TPair {
            double V[2];
        };
        const TPair a = __builtin_bit_cast(TPair, n), b = __builtin_bit_cast(TPair, m);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            out = __builtin_amdgcn_mfma_f64_16x16x4f64(a.V[i], b.V[i], out, 0, 0, 0);
        }
        return out;
    }
};

// Which n of a 16 x 16 product a lane's value r is
template <typename T>
__device__ __forceinline__ uint32_t OutputOf(uint32_t lane, int r) {
    return std::is_same_v<T, double> ? (lane >> 4) + 4 * r : 4 * (lane >> 4) + r;
}

// act(x) and its derivative, in the type that sums are held in
template <typename A>
struct TActivated {
    A Value, Slope;
};
__device__ __forceinline__ float ExpOf(float x) {
    return expf(x);
}
__device__ __forceinline__ double ExpOf(double x) {
    return exp(x);
}
template <typename A>
__device__ __forceinline__ TActivated<A> Activate(int activation, A x) {
    switch (activation) {
        case CBHIP_SILU: {
            // (a negative exponent alone: nothing overflows)
            const A e = ExpOf(x < 0 ? x : -x), y = (x < 0 ? e : A(1)) / (1 + e), rest = (x < 0 ? A(1) : e) / (1 + e);
            // (the limits at both infinities)
            const A low = x < A(-1e6) ? A(0) : x, near = x > A(1e6) || x < A(-1e6) ? A(0) : x;
            return {low * y, y * (1 + near * rest)};
        }
        case CBHIP_GELU: {
            A y;
            if constexpr (std::is_same_v<A, double>) {
                y = A(0.5) * erfc(-x * A(0.70710678118654752440));
            } else {
                y = A(0.5) * erfcf(-x * A(0.70710678118654752440));
            }
            const A low = x < A(-1e6) ? A(0) : x, near = x > A(1e6) || x < A(-1e6) ? A(0) : x;
            return {low * y, y + near * ExpOf(A(-0.5) * near * near) * A(0.39894228040143267794)};
        }
        case CBHIP_GELU_TANH: {
            // 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z)); past |x| = 100 both are 0 or 1 to the last bit
            const A c = A(0.79788456080286535588), q = A(0.044715);
            const A near = x > A(100) ? A(100) : x < A(-100) ? A(-100) : x;
            const A z = 2 * c * (near + q * near * near * near);
            const A e = ExpOf(z < 0 ? z : -z), y = (z < 0 ? e : A(1)) / (1 + e), rest = (z < 0 ? A(1) : e) / (1 + e);
            const A low = x < A(-100) ? A(0) : x;
            return {low * y, y + near * y * rest * 2 * c * (1 + 3 * q * near * near)};
        }
        default: return {x > 0 ? x : x <= 0 ? A(0) : x, x > 0 ? A(1) : x <= 0 ? A(0) : x};
    }
}

// ---------------------------------------------------------------- rows of an expert ----

struct TSegments {
    const int32_t* Offsets;  // nullptr: one expert has all rows
    uint32_t Rows;
    uint32_t Experts;

    // The rows of expert e, whatever the offsets say inside [0, Rows]
    __device__ __forceinline__ void Get(uint32_t e, uint32_t& begin, uint32_t& end) const {
        if (Offsets == nullptr) {
            begin = 0;
            end = Rows;
            return;
        }
        const int32_t b = Offsets[e], n = Offsets[e + 1];
        begin = b < 0 ? 0 : static_cast<uint32_t>(b) > Rows ? Rows : static_cast<uint32_t>(b);
        end = n < 0 ? 0 : static_cast<uint32_t>(n) > Rows ? Rows : static_cast<uint32_t>(n);
        end = end < begin ? begin : end;
    }

    // The expert that has tile `tile` of all experts' tiles of `size` rows, and the tile's rows; false behind the last one.
    // Every lane of the wave takes part.
    __device__ __forceinline__ bool Find(uint64_t tile, uint32_t size, uint32_t& expert, uint32_t& begin, uint32_t& end) const {
        if (Offsets == nullptr) {
            const uint64_t at = tile * size;
            if (at >= Rows) {
                return false;
            }
            expert = 0;
            begin = static_cast<uint32_t>(at);
            end = Rows - begin > size ? begin + size : Rows;
            return true;
        }
        const uint32_t lane = threadIdx.x & 63;
        for (uint32_t first = 0; first < Experts; first += 64) {
            uint32_t b = 0, n = 0;
            if (first + lane < Experts) {
                Get(first + lane, b, n);
            }
            const uint32_t tiles = (n - b) / size + ((n - b) % size != 0);
            uint64_t sum = tiles;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const uint64_t other = __shfl_up(sum, d);
                sum += lane >= static_cast<uint32_t>(d) ? other : 0;
            }
            const uint64_t before = sum - tiles;
            const uint64_t found = __ballot(tile >= before && tile < sum);
            if (found != 0) {
                const int from = __ffsll(static_cast<unsigned long long>(found)) - 1;
                expert = __builtin_amdgcn_readlane(static_cast<int>(first + lane), from);
                const uint32_t at = b + static_cast<uint32_t>(tile - before) * size;
                begin = __builtin_amdgcn_readlane(static_cast<int>(at), from);
                const uint32_t last = __builtin_amdgcn_readlane(static_cast<int>(n), from);
                end = last - begin > size ? begin + size : last;
                return true;
            }
            tile -= __shfl(sum, 63);
        }
        return false;
    }
};

// Workgroups go to the eight XCDs in turn, each with an L2 and 32 compute units of its own: 256 of them have eight times 32 tiles in a
// row, the last ones, fewer than 256, one each
__device__ __forceinline__ uint64_t TileOfGroup(uint32_t group, uint32_t groups) {
    return (group | 255) < groups ? (group & ~255u) | (group & 7) << 5 | (group >> 3 & 31) : group;
}

// ---------------------------------------------------------------- tiles through LDS ----

enum EForm { kRows = 0, kInputs = 1, kWeights = 2 };

// One operand of a product. Its values lie N = 16 bytes' worth at a time along `k` (LINE_IS_K) or along its own rows; a tile of it
// in LDS is laid out the same way, with some bytes behind each line that keep what 16 lanes read at a time on banks of their own.
template <typename T, int SIZE, int KBYTES, bool LINE_IS_K, int THREADS>
struct TOperand {
    static constexpr int N = 16 / sizeof(T);
    static constexpr int K = KBYTES / sizeof(T);
    static constexpr int kLines = LINE_IS_K ? SIZE : K;
    static constexpr int kLineChunks = (LINE_IS_K ? K : SIZE) / N;
    static constexpr int kPad = LINE_IS_K ? 16 : sizeof(T) == 2 ? 32 : sizeof(T) == 4 ? 16 : 64;
    static constexpr int kLineBytes = kLineChunks * 16 + kPad;
    static constexpr int kBytes = kLines * kLineBytes;
    static constexpr int kChunks = (kLines * kLineChunks + THREADS - 1) / THREADS;
    static constexpr bool kWhole = kLines * kLineChunks % THREADS == 0;
    using TChunk = TValues<T, N>;

    // 16-bit lines of k are stored so that the eight lines which 32 lanes read at a time follow each other
    __device__ __forceinline__ static uint32_t Place(uint32_t line) {
        if constexpr (!LINE_IS_K && sizeof(T) == 2) {
            return (line & ~31u) + ((line >> 2 & 1) << 4) + ((line >> 3 & 3) << 2) + (line & 3);
        }
        return line;
    }
    __device__ __forceinline__ static bool Mine(uint32_t thread, int i) {
        return kWhole || thread + i * THREADS < kLines * kLineChunks;
    }
    __device__ __forceinline__ static void Put(char* lds, uint32_t thread, const TChunk* held) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = thread + i * THREADS;
            if (Mine(thread, i)) {
                *reinterpret_cast<uint4*>(lds + Place(c / kLineChunks) * kLineBytes + c % kLineChunks * 16) = __builtin_bit_cast(uint4, held[i]);
            }
        }
    }
    // The fragment of own rows row to row + 15 and 64 bytes of k from `part` on
    __device__ __forceinline__ static uint4 Get(const char* lds, uint32_t row, uint32_t part, uint32_t lane) {
        if constexpr (LINE_IS_K) {
            return *reinterpret_cast<const uint4*>(lds + (row + (lane & 15)) * kLineBytes + part * 64 + (lane >> 4) * 16);
        } else if constexpr (sizeof(T) == 2) {
            // 16 lanes read four lines of 16 values and get four values of one column each
            struct TParts {
                TShort4 V[2];
            } r;
            const uint32_t line = part * 32 + (lane >> 4) * 4 + (lane >> 2 & 3);
            const char* at = lds + line * kLineBytes + (row + (lane & 3) * 4) * 2;
            using TLds = __attribute__((address_space(3))) TShort4;
            r.V[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TLds*)at);
            r.V[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TLds*)(at + 16 * kLineBytes));
            return __builtin_bit_cast(uint4, r);
        } else {
            struct TParts {
                T V[N];
            } r;
            const char* at = lds + (part * 4 * N + (lane >> 4) * N) * kLineBytes + (row + (lane & 15)) * sizeof(T);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                r.V[i] = *reinterpret_cast<const T*>(at + i * kLineBytes);
            }
            return __builtin_bit_cast(uint4, r);
        }
    }
};

// What a workgroup of a product works on. Matrices are T's rows `stride` values apart.
template <typename T>
struct TProduct {
    TSegments Segments;
    const T* Source;        // kRows: x; kInputs: dy (of the two projections side by side); kWeights: dy
    uint64_t SourceStride;
    const T* Other[2];      // kRows, kInputs: the weights of the first expert, of each projection; kWeights: x
    uint64_t OtherStride;   // kWeights: of x; else values from one expert's weights to the next's
    uint32_t M, N, K;       // kRows, kInputs: N and K, of one projection; kWeights: M (of one projection) and N
    T* Result[2];
    uint64_t ResultStride;  // of a row; kWeights: values from one expert's weights to the next's
    TAcc<T>* Kept;          // the gate and up values of a row side by side, or nullptr
    int Activation;
    uint64_t Tiles, First;  // of all launches, and the first of this one
    uint32_t TilesN, Together;
};

// Which tile of a product a workgroup has. kWeights: rows FirstRow on of the weights of one projection, from the expert's rows
// Begin to End; else rows Begin to End. Every lane of the wave takes part.
struct TTileOfProduct {
    bool There = true;
    uint32_t Expert = 0, Begin = 0, End = 0, FirstRow = 0, FirstColumn = 0, Projection = 0;

    template <typename T>
    __device__ __forceinline__ TTileOfProduct(const TProduct<T>& p, uint32_t tileM, uint32_t columns, int form, uint32_t projections) {
        const uint64_t id = p.First + TileOfGroup(blockIdx.x, gridDim.x);
        if (form == kWeights) {
            // an expert's tiles in a row, those of the same columns of x together
            const uint32_t tilesM = (p.M + tileM - 1) / tileM;
            uint64_t rest = id;
            FirstRow = static_cast<uint32_t>(rest % tilesM) * tileM;
            rest /= tilesM;
            Projection = static_cast<uint32_t>(rest % projections);
            rest /= projections;
            FirstColumn = static_cast<uint32_t>(rest % p.TilesN) * columns;
            Expert = static_cast<uint32_t>(rest / p.TilesN);
            p.Segments.Get(Expert, Begin, End);
        } else {
            // up to four tiles of rows with the same weights follow each other
            const uint64_t block = static_cast<uint64_t>(p.Together) * p.TilesN;
            const uint32_t within = static_cast<uint32_t>(id % block);
            FirstColumn = within / p.Together * columns;
            There = p.Segments.Find(id / block * p.Together + within % p.Together, tileM, Expert, Begin, End);
        }
    }
};

// A wave's part of a tile, from its row waveM and column waveN on
template <typename T, int TILES_M, int TILES_N, int FORM, int PROJECTIONS>
__device__ __forceinline__ void StoreProduct(const TProduct<T>& p, const TTileOfProduct& t, uint32_t waveM, uint32_t waveN, uint32_t lane,
                                             const typename TMatrix<T>::TOut (&out)[TILES_M][TILES_N]) {
    using A = TAcc<T>;
    constexpr bool kGated = FORM == kRows && PROJECTIONS == 2;
    constexpr int kTilesM = TILES_M, kTilesN = TILES_N;
    // four columns of a row at a time; 64-bit ones are four apart
    const auto store = [&](auto* row, uint32_t n, uint32_t most, const A(&v)[4]) {
        using TTo = std::remove_pointer_t<decltype(row)>;
        if constexpr (std::is_same_v<T, double>) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (n + 4 * r < most) {
                    row[n + 4 * r] = v[r];
                }
            }
        } else {
            if (n < most) {
                TValues<TTo, 4> rounded;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    rounded.V[r] = static_cast<TTo>(v[r]);
                }
                StoreUpTo(rounded, row + n, most - n);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < kTilesM; ++i) {
        const uint32_t m = waveM + i * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < kTilesN; j += kGated ? 2 : 1) {
            const uint32_t n = t.FirstColumn + (kGated ? (waveN + j * 16) / 2 : waveN + j * 16) + OutputOf<T>(lane, 0);
            A v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v[r] = out[i][j][r];
            }
            if constexpr (FORM == kWeights) {
                if (t.FirstRow + m < p.M) {
                    store(p.Result[t.Projection] + t.Expert * p.ResultStride + static_cast<uint64_t>(t.FirstRow + m) * p.N, n, p.N, v);
                }
            } else {
                if (t.Begin + m < t.End) {
                    const uint64_t row = t.Begin + m;
                    if constexpr (kGated) {
                        A u[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            u[r] = out[i][j + 1][r];
                        }
                        if (p.Kept != nullptr) {
                            A* kept = p.Kept + row * 2 * p.N;
                            store(kept, n, p.N, v);
                            store(kept + p.N, n, p.N, u);
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            v[r] = Activate(p.Activation, v[r]).Value * u[r];
                        }
                    }
                    store(p.Result[0] + row * p.ResultStride, n, p.N, v);
                }
            }
        }
    }
}

// WK: groups of WM * WN waves that share the steps of k in turns, where there are few tiles for many of those
template <typename T, int TM, int TN, int WM, int WN, int WK, int KBYTES, int FORM, int PROJECTIONS>
__global__ void __launch_bounds__(WM* WN* WK * 64) ProductKernel(const TProduct<T> p) {
    constexpr int kThreads = WM * WN * 64;  // of a group
    constexpr bool kGated = FORM == kRows && PROJECTIONS == 2;
    using TA = TOperand<T, TM, KBYTES, FORM != kWeights, kThreads>;
    using TB = TOperand<T, TN, KBYTES, FORM == kRows, kThreads>;
    using TOut = typename TMatrix<T>::TOut;
    constexpr int kValues = TA::N, kStepK = TA::K;
    constexpr int kColumns = kGated ? TN / 2 : TN;  // outputs of a tile
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const uint32_t group = WK == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
    const uint32_t thread = WK == 1 ? threadIdx.x : threadIdx.x % kThreads;
    const uint32_t lane = threadIdx.x & 63, wave = thread >> 6;
    const TTileOfProduct t(p, TM, kColumns, FORM, PROJECTIONS);
    if (!t.There) {
        return;
    }
    const uint32_t expert = t.Expert, begin = t.Begin, end = t.End, firstColumn = t.FirstColumn, projection = t.Projection;
    const uint32_t partK = FORM == kWeights ? end - begin : p.K;
    const uint32_t steps = (partK + kStepK - 1) / kStepK;
    const uint32_t allSteps = FORM == kInputs ? steps * PROJECTIONS : steps;

    // the chunks of 16 bytes that this thread loads for a step
    typename TA::TChunk heldA[TA::kChunks];
    typename TB::TChunk heldB[TB::kChunks];
    const auto load = [&](uint32_t step) {
        uint32_t part = 0;
        if constexpr (FORM == kInputs && PROJECTIONS == 2) {
            part = step >= steps;
            step -= part * steps;
        }
        const uint32_t k0 = step * kStepK;
        const bool whole = k0 + kStepK <= partK;
        constexpr bool kFitsA = FORM != kWeights;  // rows behind the last are read as the last one, and not stored
#pragma unroll
        for (int i = 0; i < TA::kChunks; ++i) {
            const uint32_t c = thread + i * kThreads;
            if (!TA::Mine(thread, i)) {
                continue;
            }
            const uint32_t line = c / TA::kLineChunks, at = c % TA::kLineChunks * kValues;
            if constexpr (kFitsA) {
                const uint32_t row = begin + line < end ? begin + line : end - 1;
                const T* from = p.Source + row * p.SourceStride + part * static_cast<uint64_t>(p.K) + k0 + at;
                heldA[i] = whole ? TA::TChunk::Load(from) : LoadUpTo<T, kValues>(k0 + at < partK ? from : p.Source, k0 + at < partK ? partK - k0 - at : 0);
            } else {
                const uint32_t m = t.FirstRow + at, k = k0 + line;
                const size_t left = k < partK && m < p.M ? p.M - m : 0;
                const T* from = left ? p.Source + (begin + k) * p.SourceStride + projection * static_cast<uint64_t>(p.M) + m : p.Source;
                heldA[i] = LoadUpTo<T, kValues>(from, left);
            }
        }
#pragma unroll
        for (int i = 0; i < TB::kChunks; ++i) {
            const uint32_t c = thread + i * kThreads;
            if (!TB::Mine(thread, i)) {
                continue;
            }
            const uint32_t line = c / TB::kLineChunks, at = c % TB::kLineChunks * kValues;
            if constexpr (FORM == kRows) {
                // gate and up values take turns by 16 columns, so that a wave has both of a column
                const uint32_t which = kGated ? line >> 4 & 1 : 0;
                uint32_t n = firstColumn + (kGated ? (line >> 5 << 4) + (line & 15) : line);
                n = n < p.N ? n : p.N - 1;
                const T* from = p.Other[which] + expert * p.OtherStride + static_cast<uint64_t>(n) * p.K + k0 + at;
                heldB[i] = whole ? TB::TChunk::Load(from) : LoadUpTo<T, kValues>(k0 + at < partK ? from : p.Other[0], k0 + at < partK ? partK - k0 - at : 0);
            } else {
                const uint32_t n = firstColumn + at, k = k0 + line;
                const size_t left = k < partK && n < p.N ? p.N - n : 0;
                const T* base = FORM == kInputs ? p.Other[part] + expert * p.OtherStride + static_cast<uint64_t>(k) * p.N : p.Other[0] + (begin + k) * p.OtherStride;
                heldB[i] = LoadUpTo<T, kValues>(left ? base + n : p.Other[0], left);
            }
        }
    };

    constexpr int kTilesM = TM / WM / 16, kTilesN = TN / WN / 16;
    const uint32_t waveM = wave % WM * (TM / WM), waveN = wave / WM * (TN / WN);
    TOut out[kTilesM][kTilesN] = {};
    constexpr int kStage = TA::kBytes + TB::kBytes;
    char* const mine = lds + group * 2 * kStage;
    if (group < allSteps) {
        load(group);
        TA::Put(mine, thread, heldA);
        TB::Put(mine + TA::kBytes, thread, heldB);
    }
    for (uint32_t turn = 0; turn * WK < allSteps; ++turn) {
        __syncthreads();
        const uint32_t step = turn * WK + group;
        const char* now = mine + (turn & 1) * kStage;
        if (step + WK < allSteps) {
            load(step + WK);
        }
        if (WK > 1 && step >= allSteps) {
            continue;
        }
#pragma unroll
        for (int part = 0; part < KBYTES / 64; ++part) {
            uint4 a[kTilesM], b[kTilesN];
#pragma unroll
            for (int i = 0; i < kTilesM; ++i) {
                a[i] = TA::Get(now, waveM + i * 16, part, lane);
            }
#pragma unroll
            for (int j = 0; j < kTilesN; ++j) {
                b[j] = TB::Get(now + TA::kBytes, waveN + j * 16, part, lane);
            }
#pragma unroll
            for (int i = 0; i < kTilesM; ++i) {
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) {
                    out[i][j] = TMatrix<T>::Step(b[j], a[i], out[i][j]);
                }
            }
        }
        if (step + WK < allSteps) {
            char* next = mine + ((turn + 1) & 1) * kStage;
            TA::Put(next, thread, heldA);
            TB::Put(next + TA::kBytes, thread, heldB);
        }
    }
    if constexpr (WK > 1) {
        // the groups' sums, added in their order, by way of the same memory
        constexpr uint32_t kSums = kTilesM * kTilesN * kThreads * sizeof(TOut);
        static_assert((WK - 1) * kSums <= WK * 2 * kStage, "what the other groups hand over fits");
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kTilesM * kTilesN; ++i) {
            if (group > 0) {
                *reinterpret_cast<TOut*>(lds + (group - 1) * kSums + (i * kThreads + thread) * sizeof(TOut)) = out[i / kTilesN][i % kTilesN];
            }
        }
        __syncthreads();
        if (group > 0) {
            return;
        }
#pragma unroll
        for (int g = 0; g < WK - 1; ++g) {
#pragma unroll
            for (int i = 0; i < kTilesM * kTilesN; ++i) {
                out[i / kTilesN][i % kTilesN] += *reinterpret_cast<const TOut*>(lds + g * kSums + (i * kThreads + thread) * sizeof(TOut));
            }
        }
    }

    StoreProduct<T, kTilesM, kTilesN, FORM, PROJECTIONS>(p, t, waveM, waveN, lane, out);
}

// ---------------------------------------------------------------- large tiles of 16-bit values ----

// Bytes that stand for what lies behind the last k of a product
__device__ __attribute__((aligned(16))) const uint32_t gZeros[4] = {};


// 16 bytes of each lane from its address to LDS, 1 KB in a row for the wave, without a trip through registers
__device__ __forceinline__ void CopyToLds(const void* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// What every wave copied so far is in LDS for all
__device__ __forceinline__ void CopiesAreThere() {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): copies count as loads
    __syncthreads();
}

// One operand of a tile of K (32 or 64) k, as TOperand, but copied straight to LDS: lines without gaps, in which pieces of 16 bytes trade
// places, so that the lanes which read at a time meet different banks.
template <typename T, int SIZE, int K, bool LINE_IS_K, int THREADS>
struct TCopied {
    static constexpr uint32_t kK = K;
    static constexpr uint32_t kLineChunks = (LINE_IS_K ? kK : SIZE) / 8;
    static constexpr uint32_t kBytes = SIZE * kK * 2;
    static constexpr int kChunks = kBytes / 16 / THREADS;
    static_assert(kBytes % (16 * THREADS) == 0 && (LINE_IS_K || kLineChunks >= 8), "whole waves copy whole lines");

    // what a piece's place in its line is crossed with
    __device__ __forceinline__ static uint32_t Cross(uint32_t line) {
        return LINE_IS_K ? (K == 64 ? line & 7 : line >> 1 & 3) : ((line & 3) | (line >> 1 & 4)) << 1 & (kLineChunks - 1);
    }
    // The line, and the piece of it, that goes to this thread's i-th place
    __device__ __forceinline__ static uint32_t Line(uint32_t thread, int i) {
        return (thread + i * THREADS) / kLineChunks;
    }
    __device__ __forceinline__ static uint32_t Piece(uint32_t thread, int i) {
        return (thread + i * THREADS) % kLineChunks ^ Cross(Line(thread, i));
    }
    __device__ __forceinline__ static char* Place(char* lds, uint32_t thread, int i) {
        return lds + ((thread & ~63u) + i * THREADS) * 16;
    }
    __device__ __forceinline__ static uint4 Get(const char* lds, uint32_t row, uint32_t part, uint32_t lane) {
        if constexpr (LINE_IS_K) {
            const uint32_t line = row + (lane & 15);
            return *reinterpret_cast<const uint4*>(lds + line * (K * 2) + ((part * 4 + (lane >> 4)) ^ Cross(lane)) * 16);  // (rows begin at multiples of 16)
        } else {
            struct TParts {
                TShort4 V[2];
            } r;
            using TLds = __attribute__((address_space(3))) TShort4;
            const uint32_t line = part * 32 + (lane >> 4) * 8 + (lane >> 2 & 3);
            const char* at = lds + line * (SIZE * 2) + ((row / 8 + (lane >> 1 & 1)) ^ Cross(line)) * 16 + (lane & 1) * 8;
            r.V[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TLds*)at);
            r.V[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TLds*)(at + 4 * SIZE * 2));  // (crossed alike)
            return __builtin_bit_cast(uint4, r);
        }
    }
};

// WK: groups of WM * WN waves that share the steps of k in turns, where there are few tiles for many of those
template <typename T, int TM, int TN, int WM, int WN, int WK, int K, int FORM, int PROJECTIONS>
__global__ void __launch_bounds__(WM* WN* WK * 64) LargeProductKernel(const TProduct<T> p) {
    constexpr int kThreads = WM * WN * 64;  // of a group
    constexpr bool kGated = FORM == kRows && PROJECTIONS == 2;
    using TA = TCopied<T, TM, K, FORM != kWeights, kThreads>;
    using TB = TCopied<T, TN, K, FORM == kRows, kThreads>;
    constexpr uint32_t kStepK = K;
    constexpr int kColumns = kGated ? TN / 2 : TN;
    constexpr uint32_t kStage = TA::kBytes + TB::kBytes;
    __shared__ __attribute__((aligned(16))) char even[WK * kStage];
    __shared__ __attribute__((aligned(16))) char odd[WK * kStage];

    const uint32_t group = WK == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
    const uint32_t thread = WK == 1 ? threadIdx.x : threadIdx.x % kThreads;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const TTileOfProduct t(p, TM, kGated ? TN / 2 : TN, FORM, PROJECTIONS);
    if (!t.There) {
        return;
    }
    const uint32_t partK = FORM == kWeights ? t.End - t.Begin : p.K;
    const uint32_t steps = (partK + kStepK - 1) / kStepK;
    const uint32_t allSteps = FORM == kInputs ? steps * PROJECTIONS : steps;

    // where this thread's pieces of a step lie behind the step's first value, in bytes
    uint32_t offsetA[TA::kChunks], offsetB[TB::kChunks];
#pragma unroll
    for (int i = 0; i < TA::kChunks; ++i) {
        const uint32_t line = TA::Line(thread, i), at = TA::Piece(thread, i) * 8;
        if constexpr (FORM != kWeights) {
            const uint32_t rows = t.End - t.Begin;
            offsetA[i] = (line < rows ? line : rows - 1) * static_cast<uint32_t>(p.SourceStride) * 2 + at * 2;
        } else {
            const uint32_t left = p.M - t.FirstRow;  // at least 8
            offsetA[i] = line * static_cast<uint32_t>(p.SourceStride) * 2 + (at < left ? at : left - 8) * 2;
        }
    }
    const T* gateOrUp[2] = {p.Other[0], p.Other[PROJECTIONS - 1]};
    bool isUp[TB::kChunks];
#pragma unroll
    for (int i = 0; i < TB::kChunks; ++i) {
        const uint32_t line = TB::Line(thread, i), at = TB::Piece(thread, i) * 8;
        isUp[i] = kGated && (line >> 4 & 1);
        if constexpr (FORM == kRows) {
            const uint32_t left = p.N - t.FirstColumn, n = kGated ? (line >> 5 << 4) + (line & 15) : line;
            offsetB[i] = (n < left ? n : left - 1) * p.K * 2 + at * 2;
        } else {
            const uint32_t left = p.N - t.FirstColumn;
            offsetB[i] = line * static_cast<uint32_t>(FORM == kInputs ? p.N : p.OtherStride) * 2 + (at < left ? at : left - 8) * 2;
        }
    }
    const auto copy = [&](uint32_t step, char* lds) {
        uint32_t part = 0;
        if constexpr (FORM == kInputs && PROJECTIONS == 2) {
            part = step >= steps;
            step -= part * steps;
        }
        const uint32_t k0 = step * kStepK;
        const char* a;
        const char* b[2];
        if constexpr (FORM == kRows) {
            a = reinterpret_cast<const char*>(p.Source + t.Begin * p.SourceStride + k0);
            const uint64_t at = t.Expert * p.OtherStride + static_cast<uint64_t>(t.FirstColumn) * p.K + k0;
            b[0] = reinterpret_cast<const char*>(gateOrUp[0] + at);
            b[1] = reinterpret_cast<const char*>(gateOrUp[1] + at);
        } else if constexpr (FORM == kInputs) {
            a = reinterpret_cast<const char*>(p.Source + t.Begin * p.SourceStride + part * static_cast<uint64_t>(p.K) + k0);
            b[0] = b[1] = reinterpret_cast<const char*>(gateOrUp[part] + t.Expert * p.OtherStride + static_cast<uint64_t>(k0) * p.N + t.FirstColumn);
        } else {
            a = reinterpret_cast<const char*>(p.Source + (t.Begin + k0) * p.SourceStride + t.Projection * static_cast<uint64_t>(p.M) + t.FirstRow);
            b[0] = b[1] = reinterpret_cast<const char*>(p.Other[0] + (t.Begin + k0) * p.OtherStride + t.FirstColumn);
        }
        if (k0 + kStepK <= partK) {
#pragma unroll
            for (int i = 0; i < TA::kChunks; ++i) {
                CopyToLds(a + offsetA[i], TA::Place(lds, thread, i));
            }
#pragma unroll
            for (int i = 0; i < TB::kChunks; ++i) {
                CopyToLds((isUp[i] ? b[1] : b[0]) + offsetB[i], TB::Place(lds + TA::kBytes, thread, i));
            }
        } else {
            const uint32_t left = partK - k0;
            const char* zeros = reinterpret_cast<const char*>(gZeros);
#pragma unroll
            for (int i = 0; i < TA::kChunks; ++i) {
                const uint32_t k = FORM != kWeights ? TA::Piece(thread, i) * 8 : TA::Line(thread, i);
                CopyToLds(k < left ? a + offsetA[i] : zeros, TA::Place(lds, thread, i));
            }
#pragma unroll
            for (int i = 0; i < TB::kChunks; ++i) {
                const uint32_t k = FORM == kRows ? TB::Piece(thread, i) * 8 : TB::Line(thread, i);
                CopyToLds(k < left ? (isUp[i] ? b[1] : b[0]) + offsetB[i] : zeros, TB::Place(lds + TA::kBytes, thread, i));
            }
        }
    };

    constexpr int kTilesM = TM / WM / 16, kTilesN = TN / WN / 16;
    // waves of the same columns share a SIMD, so that the last rows' waves, which do less, leave it to the others
    const uint32_t waveM = wave / WN * (TM / WM), waveN = wave % WN * (TN / WN);
    const uint32_t tileRows = FORM == kWeights ? p.M - t.FirstRow : t.End - t.Begin;
    const bool busy = waveM < tileRows && waveN / (kGated ? 2 : 1) < p.N - t.FirstColumn;
    TFloat4 out[kTilesM][kTilesN] = {};
    const auto multiply = [&](const char* now) {
        if (!busy) {
            return;
        }
#pragma unroll
        for (int part = 0; part < K / 32; ++part) {
            uint4 a[kTilesM], b[kTilesN];
#pragma unroll
            for (int j = 0; j < kTilesN; ++j) {
                b[j] = TB::Get(now + TA::kBytes, waveN + j * 16, part, lane);
            }
#pragma unroll
            for (int i = 0; i < kTilesM; ++i) {
                a[i] = TA::Get(now, waveM + i * 16, part, lane);
            }
#pragma unroll
            for (int i = 0; i < kTilesM; ++i) {
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) {
                    out[i][j] = TMatrix<T>::Step(b[j], a[i], out[i][j]);
                }
            }
        }
        if constexpr (FORM == kRows && kTilesM == 8 && kTilesN == 4) {
            // the first part's twelve fragments, then one of the second part's after every other product (without it the compiler waits for
            // each two fragments: 8192 rows 8192 to 4096 421 us, 405 with it; the other forms' fragments are two reads each, and it costs them)
            __builtin_amdgcn_sched_group_barrier(0x100, 12, 0);
#pragma unroll
            for (int i = 0; i < 12; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, 40, 0);
        }
    };
    char* const myEven = even + group * kStage;
    char* const myOdd = odd + group * kStage;
    if (group < allSteps) {
        copy(group, myEven);
    }
    for (uint32_t step = group; step - group < allSteps; step += 2 * WK) {
        CopiesAreThere();  // of this step; and what those to come overwrite has been read
        if (step + WK < allSteps) {
            copy(step + WK, myOdd);
        }
        if (WK == 1 || step < allSteps) {
            multiply(myEven);
        }
        if (step - group + WK < allSteps) {
            CopiesAreThere();
            if (step + 2 * WK < allSteps) {
                copy(step + 2 * WK, myEven);
            }
            if (WK == 1 || step + WK < allSteps) {
                multiply(myOdd);
            }
        }
    }
    if constexpr (WK > 1) {
        // the groups' sums, added in their order
        constexpr uint32_t kSums = kTilesM * kTilesN * kThreads * 16;
        static_assert((WK - 1) * kSums <= WK * kStage, "what the other groups hand over fits");
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kTilesM * kTilesN; ++i) {
            if (group > 0) {
                *reinterpret_cast<TFloat4*>(even + (group - 1) * kSums + (i * kThreads + thread) * 16) = out[i / kTilesN][i % kTilesN];
            }
        }
        __syncthreads();
        if (group == 0) {
#pragma unroll
            for (int g = 0; g < WK - 1; ++g) {
#pragma unroll
                for (int i = 0; i < kTilesM * kTilesN; ++i) {
                    out[i / kTilesN][i % kTilesN] += *reinterpret_cast<const TFloat4*>(even + g * kSums + (i * kThreads + thread) * 16);
                }
            }
        }
    }

    // The tile goes to memory by way of LDS, so that lanes in a row store a row's pieces of 16 bytes: from the products' own layout, 32
    // bytes of 16 rows at a time, stores came to 1.3 TB/s
    // (all rows at a time, or those of the waves of the same columns one after the other, where LDS does not hold more)
    constexpr int kRounds = TM / 2 * kColumns * (kGated ? 4 : 2) <= kStage ? 1 : WM;
    constexpr uint32_t kRoundRows = TM / kRounds, kHalf = kRoundRows / 2;
    static_assert(kHalf * kColumns * (kGated ? 4 : 2) <= kStage, "half of a round's rows fit in each part of LDS");
    const auto store = [&](auto type, auto&& valueOf, auto* to, uint64_t stride, uint32_t rows, uint32_t columns) {
        using TTo = decltype(type);
        constexpr uint32_t kValues = 16 / sizeof(TTo), kPieces = kColumns / kValues;
        const auto at = [&](uint32_t row, uint32_t piece) {
            return (row < kHalf ? even : odd) + ((row & (kHalf - 1)) * kPieces + (piece ^ (row & 15 & (kPieces - 1)))) * 16;
        };
#pragma unroll
        for (int round = 0; round < kRounds; ++round) {
            __syncthreads();
            if (group == 0 && (kRounds == 1 || waveM == round * kRoundRows)) {
#pragma unroll
                for (int i = 0; i < kTilesM; ++i) {
#pragma unroll
                    for (int j = 0; j < kTilesN; j += kGated ? 2 : 1) {
                        TValues<TTo, 4> v;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            v.V[r] = static_cast<TTo>(valueOf(i, j, r));
                        }
                        const uint32_t n = (kGated ? (waveN + j * 16) / 2 : waveN + j * 16) + 4 * (lane >> 4);
                        using TWords = std::conditional_t<sizeof(TTo) == 2, uint2, uint4>;
                        *reinterpret_cast<TWords*>(at(waveM - round * kRoundRows + i * 16 + (lane & 15), n / kValues) + n % kValues * sizeof(TTo)) =
                            __builtin_bit_cast(TWords, v);
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < (kRoundRows * kPieces + WK * kThreads - 1) / (WK * kThreads); ++i) {
                const uint32_t row = (threadIdx.x + i * WK * kThreads) / kPieces, piece = (threadIdx.x + i * WK * kThreads) % kPieces;
                if (row >= kRoundRows) {
                    break;
                }
                const auto v = __builtin_bit_cast(TValues<TTo, kValues>, *reinterpret_cast<const uint4*>(at(row, piece)));
                const uint32_t m = round * kRoundRows + row;
                if (m < rows && piece * kValues < columns) {
                    StoreUpTo(v, to + m * stride + piece * kValues, columns - piece * kValues);
                }
            }
        }
    };
    if constexpr (FORM == kWeights) {
        store(T(), [&](int i, int j, int r) { return out[i][j][r]; },
              p.Result[t.Projection] + t.Expert * p.ResultStride + static_cast<uint64_t>(t.FirstRow) * p.N + t.FirstColumn, p.N, p.M - t.FirstRow, p.N - t.FirstColumn);
    } else {
        const uint64_t row = t.Begin;
        const uint32_t rows = t.End - t.Begin, columns = p.N - t.FirstColumn;
        if constexpr (kGated) {
            if (p.Kept != nullptr) {
                float* kept = p.Kept + row * 2 * p.N + t.FirstColumn;
                store(float(), [&](int i, int j, int r) { return out[i][j][r]; }, kept, uint64_t(2) * p.N, rows, columns);
                store(float(), [&](int i, int j, int r) { return out[i][j + 1][r]; }, kept + p.N, uint64_t(2) * p.N, rows, columns);
            }
            store(T(), [&](int i, int j, int r) { return Activate(p.Activation, out[i][j][r]).Value * out[i][j + 1][r]; },
                  p.Result[0] + row * p.ResultStride + t.FirstColumn, p.ResultStride, rows, columns);
        } else {
            store(T(), [&](int i, int j, int r) { return out[i][j][r]; }, p.Result[0] + row * p.ResultStride + t.FirstColumn, p.ResultStride, rows, columns);
        }
    }
}

// ---------------------------------------------------------------- few rows, few outputs ----

// out = x W^T where one operand is read once and little is done with it, so that it goes straight to registers, 64 bytes of 16 lines at
// a time; the other one comes from the caches. SPLIT: the four waves of a workgroup have the same 16 * MT rows, and share the line of
// k in turns of 64 * PARTS bytes (few rows: the weights are what is read). Else each has 16 * MT rows of its own (few outputs: the rows
// are). Operands at any alignment.
template <typename T, int MT, int NT, int PARTS, bool SPLIT, int PROJECTIONS>
__global__ void __launch_bounds__(256) StreamProductKernel(const TProduct<T> p) {
    constexpr int N = 16 / sizeof(T), kPart = 4 * N;
    constexpr uint32_t kRowsOfTile = SPLIT ? 16 * MT : 64 * MT, kColumns = 16 * NT / PROJECTIONS;
    using TOut = typename TMatrix<T>::TOut;
    using TChunk = TValues<T, N>;
    const TTileOfProduct t(p, kRowsOfTile, kColumns, kRows, PROJECTIONS);
    if (!t.There) {
        return;
    }
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t waveM = SPLIT ? 0 : wave * 16 * MT;
    const T* rows[MT];
    const T* columns[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const uint32_t m = t.Begin + waveM + i * 16 + (lane & 15);
        rows[i] = p.Source + (m < t.End ? m : t.End - 1) * p.SourceStride + (lane >> 4) * N;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const uint32_t n = t.FirstColumn + j / PROJECTIONS * 16 + (lane & 15);
        columns[j] = p.Other[j % PROJECTIONS] + t.Expert * p.OtherStride + static_cast<uint64_t>(n < p.N ? n : p.N - 1) * p.K + (lane >> 4) * N;
    }

    struct TParts {
        TChunk A[PARTS][MT], B[PARTS][NT];
    };
    constexpr uint32_t kTurn = kPart * PARTS, kStep = SPLIT ? 4 * kTurn : kTurn;
    const auto load = [&](TParts& to, uint32_t k0) {
        if (k0 + kTurn <= p.K) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    to.B[part][j] = TChunk::Load(columns[j] + k0 + part * kPart);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    to.A[part][i] = TChunk::Load(rows[i] + k0 + part * kPart);
                }
            }
        } else {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                const uint32_t k = k0 + part * kPart + (lane >> 4) * N;
                const size_t left = k < p.K ? p.K - k : 0;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    to.B[part][j] = LoadUpTo<T, N>(left ? columns[j] + k0 + part * kPart : columns[j], left);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    to.A[part][i] = LoadUpTo<T, N>(left ? rows[i] + k0 + part * kPart : rows[i], left);
                }
            }
        }
    };
    TOut out[MT][NT] = {};
    const auto multiply = [&](const TParts& from) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    out[i][j] = TMatrix<T>::Step(__builtin_bit_cast(uint4, from.B[part][j]), __builtin_bit_cast(uint4, from.A[part][i]), out[i][j]);
                }
            }
        }
    };
    // two turns under way at a time
    TParts even, odd;
    uint32_t k = SPLIT ? wave * kTurn : 0;
    if (k < p.K) {
        load(even, k);
    }
    while (k < p.K) {
        if (k + kStep < p.K) {
            load(odd, k + kStep);
        }
        multiply(even);
        k += kStep;
        if (k < p.K) {
            if (k + kStep < p.K) {
                load(even, k + kStep);
            }
            multiply(odd);
            k += kStep;
        }
    }
    if constexpr (SPLIT) {
        __shared__ TOut parts[3][MT * NT][64];
        if (wave != 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    parts[wave - 1][i * NT + j][lane] = out[i][j];
                }
            }
        }
        __syncthreads();
        if (wave != 0) {
            return;
        }
#pragma unroll
        for (int w = 0; w < 3; ++w) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    out[i][j] += parts[w][i * NT + j][lane];
                }
            }
        }
    }
    StoreProduct<T, MT, NT, kRows, PROJECTIONS>(p, t, waveM, 0, lane, out);
}

// ---------------------------------------------------------------- launches ----

constexpr uint64_t kMostGroups = uint64_t(1) << 21;  // of a launch, of up to 1024 threads

template <int FORM, int PROJECTIONS, typename T, int TM, int TN>
void SetTiles(TProduct<T>& p) {
    constexpr uint32_t kColumns = FORM == kRows && PROJECTIONS == 2 ? TN / 2 : TN;
    p.TilesN = (p.N + kColumns - 1) / kColumns;
    if constexpr (FORM == kWeights) {
        p.Tiles = static_cast<uint64_t>(p.Segments.Experts) * p.TilesN * PROJECTIONS * ((p.M + TM - 1) / TM);
    } else {
        // an expert's last tile may be a part of one
        const uint64_t tilesM = p.Segments.Offsets != nullptr ? p.Segments.Rows / TM + std::min(p.Segments.Experts, p.Segments.Rows) : (p.Segments.Rows + uint64_t(TM) - 1) / TM;
        p.Together = static_cast<uint32_t>(std::min<uint64_t>(tilesM, 4));
        p.Tiles = (tilesM + p.Together - 1) / p.Together * p.Together * p.TilesN;
    }
}

template <int FORM, int PROJECTIONS, typename T, int TM, int TN, int WM, int WN, int WK>
void LaunchProduct(const TCallDevice& call, TProduct<T> p) {
    constexpr int kThreads = WM * WN * 64;
    constexpr int KBYTES = WK > 1 && sizeof(T) > 2 ? 128 : 64;  // (as many as LDS holds, where a step is a wait for memory)
    constexpr size_t lds = WK * 2 * (TOperand<T, TM, KBYTES, FORM != kWeights, kThreads>::kBytes + TOperand<T, TN, KBYTES, FORM == kRows, kThreads>::kBytes);
    SetTiles<FORM, PROJECTIONS, T, TM, TN>(p);
    const auto kernel = ProductKernel<T, TM, TN, WM, WN, WK, KBYTES, FORM, PROJECTIONS>;
    call.AllowLds(reinterpret_cast<const void*>(kernel), lds);
    for (p.First = 0; p.First < p.Tiles; p.First += kMostGroups) {
        call.Launch(kernel, std::min(kMostGroups, p.Tiles - p.First), WK * kThreads, lds, p);
    }
}

template <int FORM, int PROJECTIONS, typename T, int TM, int TN, int WM, int WN, int WK, int K = 64>
void LaunchLarge(const TCallDevice& call, TProduct<T> p) {
    SetTiles<FORM, PROJECTIONS, T, TM, TN>(p);
    for (p.First = 0; p.First < p.Tiles; p.First += kMostGroups) {
        call.Launch(LargeProductKernel<T, TM, TN, WM, WN, WK, K, FORM, PROJECTIONS>, std::min(kMostGroups, p.Tiles - p.First), WM * WN * WK * 64, 0, p);
    }
}

template <int PROJECTIONS, typename T, int MT, int NT, int PARTS, bool SPLIT>
void LaunchStream(const TCallDevice& call, TProduct<T> p) {
    SetTiles<kRows, PROJECTIONS, T, SPLIT ? 16 * MT : 64 * MT, 16 * NT>(p);
    for (p.First = 0; p.First < p.Tiles; p.First += kMostGroups) {
        call.Launch(StreamProductKernel<T, MT, NT, PARTS, SPLIT, PROJECTIONS>, std::min(kMostGroups, p.Tiles - p.First), 256, 0, p);
    }
}

// Whether copies of 16 bytes can take every operand
template <int FORM, int PROJECTIONS, typename T>
bool TakesCopies(const TProduct<T>& p) {
    const auto whole = [](uint64_t v) { return v % 8 == 0; };
    const auto at = [](const void* v) { return reinterpret_cast<uintptr_t>(v) % 16 == 0; };
    constexpr uint64_t kMostStride = uint64_t(1) << 22;  // 256 rows of it are under 2^32 bytes
    return whole(FORM == kWeights ? p.M : p.K) && (FORM == kRows || whole(p.N)) && whole(p.SourceStride) && whole(p.OtherStride) && at(p.Source) &&
           at(p.Other[0]) && at(p.Other[PROJECTIONS == 2 && FORM != kWeights ? 1 : 0]) && p.SourceStride < kMostStride &&
           (FORM == kWeights ? p.OtherStride : FORM == kInputs ? p.N : p.K) < kMostStride;
}

// Which kernel. The host does not see the offsets: `each` is what an expert has on average (2048 x 4096 to 1024 of 128 experts 249 evenly; 178
// where four have all, by tiles of 16 rows that read their weights again and again. 16384 of 64 experts 246 and 162). Times are of bf16, in microseconds, x W^T of
// rows x inputs to outputs (and the same gated) unless said otherwise.
template <int FORM, int PROJECTIONS, typename T>
void MultiplyBy(const TCallDevice& call, const TProduct<T>& p) {
    const uint32_t used = std::max(1u, std::min(p.Segments.Experts, p.Segments.Rows)), each = p.Segments.Rows / used;
    // tiles of `size` that there are about
    const auto tiles = [&](uint64_t size) {
        const auto parts = [&](uint64_t n) { return (n + size - 1) / size; };
        const uint64_t of = parts(p.N) * PROJECTIONS;
        return FORM == kWeights ? p.Segments.Experts * parts(p.M) * of : FORM == kRows ? used * parts(each) * of : used * parts(each) * parts(p.N);
    };
    if constexpr (FORM == kRows) {
        // weights that are read for 16 rows (14 x 4096 to 1024 of 64 experts 24 and 44; 30 and 60 by tiles; one row to 131000 outputs 186, 201)
        if (each <= 16) {
            return LaunchStream<PROJECTIONS, T, 1, 2, 4, true>(call, p);
        }
    }
    if constexpr (sizeof(T) == 2) {
        if (TakesCopies<FORM, PROJECTIONS>(p)) {
            if constexpr (FORM == kWeights) {
                // (1024 x 4096 weights of 64 experts with 1000 rows each 759, 859 by the tiles below; of 64 rows each 224 and 233; 2048 x 2048 of 2048
                // rows, 64 tiles of 256, 69 and 39)
                if (tiles(256) >= 256) {
                    return LaunchLarge<FORM, PROJECTIONS, T, 128, 256, 2, 4, 1, 32>(call, p);
                }
                // few tiles with many rows to add over (512 x 512 of 65536 rows 347, 964 without sharing; 1024 x 1024 of 4096 rows 26 and 66; 256 tiles of
                // 2048 rows 56 and 39)
                if (tiles(128) <= 128) {
                    return LaunchLarge<FORM, PROJECTIONS, T, 64, 64, 2, 2, 4>(call, p);
                }
            } else {
                // not enough tiles for the chip: the steps of k are shared by four groups of waves, or two (256 x 4096 to 1024 of 4 experts 22 and
                // 26; 30 and 31 by two, 34 and 37 by one; 512 x 4096 to 1024 of 16 experts 29 and 62, 32 and 47, 36 and 57)
                if (tiles(64) <= 256) {
                    return LaunchLarge<FORM, PROJECTIONS, T, 64, 64, 2, 2, 4>(call, p);
                }
                if (tiles(64) <= 512) {
                    return LaunchLarge<FORM, PROJECTIONS, T, 64, 64, 2, 2, 2>(call, p);
                }
                if constexpr (FORM == kRows) {
                    // (64 x 4096 to 131000 220, 249 by the tiles below; 128 rows 282 and 263)
                    if (each <= 64) {
                        return LaunchLarge<FORM, PROJECTIONS, T, 64, 128, 1, 4, 1>(call, p);
                    }
                }
                if constexpr (FORM == kRows) {
                    // (64000 x 4096 to 1024 of 64 experts 601 and 1285, 661 and 1420 by the tiles below; 16384 rows of 64 experts 236, 229; 65536 x 1024 to
                    // 1024 of one expert gated 371 and 329)
                    if (each >= 512 && tiles(256) >= 1024 && (PROJECTIONS == 1 || p.K >= 2048)) {
                        return LaunchLarge<FORM, PROJECTIONS, T, 256, 256, 2, 4, 1>(call, p);
                    }
                } else if (tiles(128) >= 512) {
                    // (inputs' gradients of 64000 x 4096 by 1024 of 64 experts 773, 912 by the tiles below, 879 by tiles of 256; of 30000 x 1024 by 256 of 128
                    // experts 52, 56 and 61)
                    return LaunchLarge<FORM, PROJECTIONS, T, 128, 256, 2, 4, 1, 32>(call, p);
                }
            }
            // two workgroups of a compute unit, one of which loads or stores while the other one multiplies
            return LaunchLarge<FORM, PROJECTIONS, T, 128, 128, 2, 4, 1>(call, p);
        }
    }
    if constexpr (FORM == kRows) {
        if (each <= 32) {
            return LaunchStream<PROJECTIONS, T, 2, 2, 4, true>(call, p);
        }
        if constexpr (PROJECTIONS == 1) {
            // rows that are read for 16 outputs (500009 x 200 to 10 of 37 experts in 32 bits 97, 241 by tiles)
            if (p.N <= 16) {
                return LaunchStream<PROJECTIONS, T, 2, 1, 2, false>(call, p);
            }
        }
    }
    // (32 bits, 5003 x 1001 to 699 of 5 experts, 240 tiles: 100 and 152; 4096 x 4096 to 4096, 1024 tiles: 1315 and 1177)
    if constexpr (FORM == kWeights) {
        // few tiles with many rows to add over (32 bits, 1024 x 1024 of 60000 rows 2591 without sharing; 1024 x 1024 of 4096 rows 146; 512 x 512 of 2000
        // rows 73; with it 1288, 101 and 47)
        if (tiles(64) <= 512) {
            return LaunchProduct<FORM, PROJECTIONS, T, 64, 64, 2, 2, 4>(call, p);
        }
    }
    if (sizeof(T) == 8 || tiles(128) <= 384) {
        return LaunchProduct<FORM, PROJECTIONS, T, 64, 64, 2, 2, 1>(call, p);
    }
    if constexpr (sizeof(T) < 8) {
        LaunchProduct<FORM, PROJECTIONS, T, 128, 128, 2, 2, 1>(call, p);
    }
}

}  // namespace op
}  // namespace cbamd
