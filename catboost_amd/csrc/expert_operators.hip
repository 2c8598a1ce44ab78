// The experts' products on rows sorted by expert: gated projections and plain ones, with their gradients.
//
// Three forms of one product, out[m][n] = sum over k of a(m, k) * b(n, k), for every expert with rows:
//   rows      out = x W^T:    m a row of the expert, n an output, k an input; both operands have k in a row in memory
//   inputs    dx = dy W:      m a row, n an input, k an output; the weights have n in a row in memory
//   weights   dW = dy^T x:    m an output, n an input, k a row of the expert; both operands have k across their rows
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
    __device__ __forceinline__ static bool Mine(int i) {
        return kWhole || threadIdx.x + i * THREADS < kLines * kLineChunks;
    }
    __device__ __forceinline__ static void Put(char* lds, const TChunk* held) {
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const uint32_t c = threadIdx.x + i * THREADS;
            if (Mine(i)) {
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
    uint32_t TilesN;
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
            // four tiles of rows with the same weights follow each other
            constexpr uint32_t kTogether = 4;
            const uint64_t block = static_cast<uint64_t>(kTogether) * p.TilesN;
            const uint32_t within = static_cast<uint32_t>(id % block);
            FirstColumn = within / kTogether * columns;
            There = p.Segments.Find(id / block * kTogether + within % kTogether, tileM, Expert, Begin, End);
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

template <typename T, int TM, int TN, int WM, int WN, int KBYTES, int FORM, int PROJECTIONS>
__global__ void __launch_bounds__(WM* WN * 64) ProductKernel(const TProduct<T> p) {
    constexpr int kThreads = WM * WN * 64;
    constexpr bool kGated = FORM == kRows && PROJECTIONS == 2;
    using TA = TOperand<T, TM, KBYTES, FORM != kWeights, kThreads>;
    using TB = TOperand<T, TN, KBYTES, FORM == kRows, kThreads>;
    using TOut = typename TMatrix<T>::TOut;
    constexpr int kValues = TA::N, kStepK = TA::K;
    constexpr int kColumns = kGated ? TN / 2 : TN;  // outputs of a tile
    extern __shared__ __attribute__((aligned(16))) char lds[];

    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const TTileOfProduct t(p, TM, kColumns, FORM, PROJECTIONS);
    if (!t.There) {
        return;
    }
    const uint32_t expert = t.Expert, begin = t.Begin, end = t.End, firstColumn = t.FirstColumn, projection = t.Projection;
    const uint32_t partK = FORM == kWeights ? end - begin : p.K;
    const uint32_t steps = (partK + kStepK - 1) / kStepK;
    const uint32_t allSteps = FORM == kInputs ? steps * PROJECTIONS : steps;

    // f(i, line, chunk of the line) for the chunks of 16 bytes that this thread loads
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
            const uint32_t c = threadIdx.x + i * kThreads;
            if (!TA::Mine(i)) {
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
            const uint32_t c = threadIdx.x + i * kThreads;
            if (!TB::Mine(i)) {
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
    if (allSteps > 0) {
        load(0);
        TA::Put(lds, heldA);
        TB::Put(lds + TA::kBytes, heldB);
    }
    for (uint32_t step = 0; step < allSteps; ++step) {
        __syncthreads();
        const char* now = lds + (step & 1) * kStage;
        if (step + 1 < allSteps) {
            load(step + 1);
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
        if (step + 1 < allSteps) {
            char* next = lds + ((step + 1) & 1) * kStage;
            TA::Put(next, heldA);
            TB::Put(next + TA::kBytes, heldB);
        }
    }

    StoreProduct<T, kTilesM, kTilesN, FORM, PROJECTIONS>(p, t, waveM, waveN, lane, out);
}

// ---------------------------------------------------------------- large tiles of 16-bit values ----

// Bytes that stand for what lies behind the last k of a product
__device__ __attribute__((aligned(16))) const uint32_t gZeros[4] = {};

using TLdsBytes = __attribute__((address_space(3))) char;
using TGlobalBytes = const __attribute__((address_space(1))) char;

// 16 bytes of each lane from its address to LDS, 1 KB in a row for the wave, without a trip through registers
__device__ __forceinline__ void CopyToLds(const void* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// One operand of a tile of 64 k, as TOperand, but copied straight to LDS: lines without gaps, in which pieces of 16 bytes trade
// places, so that the lanes which read at a time meet different banks.
template <typename T, int SIZE, bool LINE_IS_K, int THREADS>
struct TCopied {
    static constexpr uint32_t kK = 64;
    static constexpr uint32_t kLineChunks = (LINE_IS_K ? kK : SIZE) / 8;
    static constexpr uint32_t kBytes = SIZE * kK * 2;
    static constexpr int kChunks = kBytes / 16 / THREADS;
    static_assert(kBytes % (16 * THREADS) == 0 && (LINE_IS_K || kLineChunks >= 16), "whole waves copy whole lines");

    // what a piece's place in its line is crossed with
    __device__ __forceinline__ static uint32_t Cross(uint32_t line) {
        return LINE_IS_K ? line & 7 : ((line & 3) | (line >> 1 & 4)) << 1;
    }
    // The line, and the piece of it, that goes to this thread's i-th place
    __device__ __forceinline__ static uint32_t Line(int i) {
        return (threadIdx.x + i * THREADS) / kLineChunks;
    }
    __device__ __forceinline__ static uint32_t Piece(int i) {
        return (threadIdx.x + i * THREADS) % kLineChunks ^ Cross(Line(i));
    }
    __device__ __forceinline__ static char* Place(char* lds, int i) {
        return lds + ((threadIdx.x & ~63u) + i * THREADS) * 16;
    }
    __device__ __forceinline__ static uint4 Get(const char* lds, uint32_t row, uint32_t part, uint32_t lane) {
        if constexpr (LINE_IS_K) {
            const uint32_t line = row + (lane & 15);
            return *reinterpret_cast<const uint4*>(lds + line * 128 + ((part * 4 + (lane >> 4)) ^ (lane & 7)) * 16);
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

template <typename T, int TM, int TN, int WM, int WN, int FORM, int PROJECTIONS>
__global__ void __launch_bounds__(WM* WN * 64) LargeProductKernel(const TProduct<T> p) {
    constexpr int kThreads = WM * WN * 64;
    constexpr bool kGated = FORM == kRows && PROJECTIONS == 2;
    using TA = TCopied<T, TM, FORM != kWeights, kThreads>;
    using TB = TCopied<T, TN, FORM == kRows, kThreads>;
    constexpr uint32_t kStepK = 64;
    constexpr int kColumns = kGated ? TN / 2 : TN;
    __shared__ __attribute__((aligned(16))) char even[TA::kBytes + TB::kBytes];
    __shared__ __attribute__((aligned(16))) char odd[TA::kBytes + TB::kBytes];

    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
        const uint32_t line = TA::Line(i), at = TA::Piece(i) * 8;
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
        const uint32_t line = TB::Line(i), at = TB::Piece(i) * 8;
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
                CopyToLds(a + offsetA[i], TA::Place(lds, i));
            }
#pragma unroll
            for (int i = 0; i < TB::kChunks; ++i) {
                CopyToLds((isUp[i] ? b[1] : b[0]) + offsetB[i], TB::Place(lds + TA::kBytes, i));
            }
        } else {
            const uint32_t left = partK - k0;
            const char* zeros = reinterpret_cast<const char*>(gZeros);
#pragma unroll
            for (int i = 0; i < TA::kChunks; ++i) {
                const uint32_t k = FORM != kWeights ? TA::Piece(i) * 8 : TA::Line(i);
                CopyToLds(k < left ? a + offsetA[i] : zeros, TA::Place(lds, i));
            }
#pragma unroll
            for (int i = 0; i < TB::kChunks; ++i) {
                const uint32_t k = FORM == kRows ? TB::Piece(i) * 8 : TB::Line(i);
                CopyToLds(k < left ? (isUp[i] ? b[1] : b[0]) + offsetB[i] : zeros, TB::Place(lds + TA::kBytes, i));
            }
        }
    };

    constexpr int kTilesM = TM / WM / 16, kTilesN = TN / WN / 16;
    const uint32_t waveM = wave % WM * (TM / WM), waveN = wave / WM * (TN / WN);
    TFloat4 out[kTilesM][kTilesN] = {};
    const auto multiply = [&](const char* now) {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
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
        if constexpr (FORM == kRows) {
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
    if (allSteps > 0) {
        copy(0, even);
    }
    for (uint32_t step = 0; step < allSteps; step += 2) {
        __syncthreads();  // the step's copies are there, what the ones to come overwrite has been read
        if (step + 1 < allSteps) {
            copy(step + 1, odd);
        }
        multiply(even);
        if (step + 1 < allSteps) {
            __syncthreads();
            if (step + 2 < allSteps) {
                copy(step + 2, even);
            }
            multiply(odd);
        }
    }

    // The tile goes to memory by way of LDS, so that lanes in a row store a row's pieces of 16 bytes: from the products' own layout, 32
    // bytes of 16 rows at a time, stores came to 1.3 TB/s
    constexpr uint32_t kHalf = TM / 2;
    static_assert(kHalf * kColumns * (kGated ? 4 : 2) <= TA::kBytes + TB::kBytes, "half of the rows fit in each part of LDS");
    const auto store = [&](auto type, auto&& valueOf, auto* to, uint64_t stride, uint32_t rows, uint32_t columns) {
        using TTo = decltype(type);
        constexpr uint32_t kValues = 16 / sizeof(TTo), kPieces = kColumns / kValues;
        const auto at = [&](uint32_t row, uint32_t piece) {
            return (row < kHalf ? even : odd) + ((row & (kHalf - 1)) * kPieces + (piece ^ (row & 15))) * 16;
        };
        __syncthreads();
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
                *reinterpret_cast<TWords*>(at(waveM + i * 16 + (lane & 15), n / kValues) + n % kValues * sizeof(TTo)) = __builtin_bit_cast(TWords, v);
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < TM * kPieces / kThreads; ++i) {
            const uint32_t row = (threadIdx.x + i * kThreads) / kPieces, piece = (threadIdx.x + i * kThreads) % kPieces;
            const auto v = __builtin_bit_cast(TValues<TTo, kValues>, *reinterpret_cast<const uint4*>(at(row, piece)));
            if (row < rows && piece * kValues < columns) {
                StoreUpTo(v, to + row * stride + piece * kValues, columns - piece * kValues);
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

// ---------------------------------------------------------------- gradients of gate and up values ----

// preGradients[r] = (dh * up * act'(gate), dh * act(gate)) of the rows that experts have; N columns for a thread. The kept values are
// in 32 bits: rounded to bf16 they made the gradients 0.0031 off (in the norm) where rounding the gradients alone makes 0.0024.
template <typename T, int N>
__global__ void __launch_bounds__(256) GateGradientsKernel(TSegments segments, uint64_t firstPiece, uint64_t pieces, uint32_t rowPieces, uint32_t hidden,
                                                           int activation, const T* gradients, uint64_t stride, const TAcc<T>* kept, T* preGradients) {
    using A = TAcc<T>;
    const uint64_t piece = firstPiece + static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (piece >= pieces) {
        return;
    }
    const uint64_t row = piece / rowPieces;
    const uint32_t at = static_cast<uint32_t>(piece - row * rowPieces) * N, left = hidden - at;
    const int32_t there = segments.Offsets != nullptr ? segments.Offsets[segments.Experts] : static_cast<int32_t>(segments.Rows);
    const int32_t first = segments.Offsets != nullptr ? segments.Offsets[0] : 0;
    if (static_cast<int64_t>(row) < first || static_cast<int64_t>(row) >= there) {
        return;
    }
    const uint64_t gate = row * 2 * hidden + at;
    const auto d = LoadUpTo<T, N>(gradients + row * stride + at, left);
    const auto g = LoadUpTo<A, N>(kept + gate, left), u = LoadUpTo<A, N>(kept + gate + hidden, left);
    TValues<T, N> dg, du;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const TActivated<A> a = Activate(activation, g.V[i]);
        dg.V[i] = static_cast<T>(static_cast<A>(d.V[i]) * u.V[i] * a.Slope);
        du.V[i] = static_cast<T>(static_cast<A>(d.V[i]) * a.Value);
    }
    StoreUpTo(dg, preGradients + gate, left);
    StoreUpTo(du, preGradients + gate + hidden, left);
}

}  // namespace op

using namespace op;

namespace {

constexpr uint64_t kMostGroups = uint64_t(1) << 22;  // of a launch

void CheckRouted(size_t rows, size_t width, size_t outputs, int32_t experts, const int32_t* offsets) {
    CBAMD_ENSURE(experts >= 1 && experts <= kMostExperts, "experts: " + std::to_string(experts) + ", 1 to " + std::to_string(kMostExperts) + " are supported");
    CBAMD_ENSURE(offsets != nullptr || experts == 1, "offsets pointer is null");
    CBAMD_ENSURE(rows <= 0x7fffffffu, "too many rows: " + std::to_string(rows));
    CBAMD_ENSURE(width < size_t(1) << 30, "rows are too wide: " + std::to_string(width));
    CBAMD_ENSURE(outputs < size_t(1) << 30, "too many outputs: " + std::to_string(outputs));
}

void CheckWeights(const char* name, const void* data, size_t outputs, size_t width, int32_t experts, size_t stride, size_t valueSize) {
    if (outputs == 0 || width == 0) {
        return;
    }
    CheckMatrix(name, data, outputs, width, width, valueSize);
    CBAMD_ENSURE(experts <= 1 || stride >= outputs * width, std::string(name) + ": a stride of " + std::to_string(stride) +
                                                               " values is shorter than an expert's " + std::to_string(outputs * width));
    CBAMD_ENSURE(experts <= 1 || stride <= (size_t(1) << 60) / valueSize / static_cast<size_t>(experts), std::string(name) + " is too large");
}

template <int FORM, int PROJECTIONS, typename T, int TM, int TN>
void SetTiles(TProduct<T>& p) {
    constexpr uint32_t kColumns = FORM == kRows && PROJECTIONS == 2 ? TN / 2 : TN;
    p.TilesN = (p.N + kColumns - 1) / kColumns;
    if constexpr (FORM == kWeights) {
        p.Tiles = static_cast<uint64_t>(p.Segments.Experts) * p.TilesN * PROJECTIONS * ((p.M + TM - 1) / TM);
    } else {
        // an expert's last tile may be a part of one; four tiles of rows at a time
        const uint64_t tilesM = p.Segments.Offsets != nullptr ? p.Segments.Rows / TM + std::min(p.Segments.Experts, p.Segments.Rows) : (p.Segments.Rows + uint64_t(TM) - 1) / TM;
        p.Tiles = (tilesM + 3) / 4 * 4 * p.TilesN;
    }
}

template <int FORM, int PROJECTIONS, typename T, int TM, int TN, int WM, int WN, int KBYTES>
void LaunchProduct(const TCallDevice& call, TProduct<T> p) {
    constexpr int kThreads = WM * WN * 64;
    constexpr size_t lds = 2 * (TOperand<T, TM, KBYTES, FORM != kWeights, kThreads>::kBytes + TOperand<T, TN, KBYTES, FORM == kRows, kThreads>::kBytes);
    SetTiles<FORM, PROJECTIONS, T, TM, TN>(p);
    const auto kernel = ProductKernel<T, TM, TN, WM, WN, KBYTES, FORM, PROJECTIONS>;
    call.AllowLds(reinterpret_cast<const void*>(kernel), lds);
    for (p.First = 0; p.First < p.Tiles; p.First += kMostGroups) {
        call.Launch(kernel, std::min(kMostGroups, p.Tiles - p.First), kThreads, lds, p);
    }
}

template <int FORM, int PROJECTIONS, typename T, int TM, int TN, int WM, int WN>
void LaunchLarge(const TCallDevice& call, TProduct<T> p) {
    SetTiles<FORM, PROJECTIONS, T, TM, TN>(p);
    for (p.First = 0; p.First < p.Tiles; p.First += kMostGroups) {
        call.Launch(LargeProductKernel<T, TM, TN, WM, WN, FORM, PROJECTIONS>, std::min(kMostGroups, p.Tiles - p.First), WM * WN * 64, 0, p);
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

template <int FORM, int PROJECTIONS, typename T>
void MultiplyBy(const TCallDevice& call, const TProduct<T>& p) {
    if constexpr (sizeof(T) == 2) {
        if (TakesCopies<FORM, PROJECTIONS>(p) && p.Segments.Rows >= 256) {
            return LaunchLarge<FORM, PROJECTIONS, T, 256, 256, 2, 4>(call, p);
        }
        LaunchProduct<FORM, PROJECTIONS, T, 128, 128, 2, 2, 64>(call, p);
    } else if constexpr (sizeof(T) == 4) {
        LaunchProduct<FORM, PROJECTIONS, T, 128, 128, 2, 2, 64>(call, p);
    } else {
        LaunchProduct<FORM, PROJECTIONS, T, 64, 64, 2, 2, 64>(call, p);
    }
}

template <typename T>
TProduct<T> ProductOf(size_t rows, int32_t experts, const int32_t* offsets) {
    TProduct<T> p{};
    p.Segments.Offsets = offsets;
    p.Segments.Rows = static_cast<uint32_t>(rows);
    p.Segments.Experts = static_cast<uint32_t>(experts);
    return p;
}

}  // namespace

void GatedRows(int valueType, int activation, size_t rows, size_t width, size_t hidden, int32_t experts, const int32_t* offsets, const void* source,
               size_t sourceStride, const void* gateWeights, const void* upWeights, size_t expertStride, void* result, size_t resultStride, void* kept,
               void* stream) {
    const size_t size = ValueSize(valueType);
    CBAMD_ENSURE(activation >= CBHIP_SILU && activation <= CBHIP_RELU, "unknown activation " + std::to_string(activation));
    CheckRouted(rows, width, hidden, experts, offsets);
    if (rows == 0 || hidden == 0) {
        return;
    }
    if (width > 0) {
        CheckMatrix("source", source, rows, width, sourceStride, size);
    }
    CheckWeights("gate weights", gateWeights, hidden, width, experts, expertStride, size);
    CheckWeights("up weights", upWeights, hidden, width, experts, expertStride, size);
    CheckMatrix("result", result, rows, hidden, resultStride, size);
    CBAMD_ENSURE(reinterpret_cast<uintptr_t>(kept) % std::max<size_t>(size, 4) == 0, "kept values pointer is not a multiple of the value size");
    const TCallDevice call(result, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        TProduct<T> p = ProductOf<T>(rows, experts, offsets);
        p.Source = static_cast<const T*>(source);
        p.SourceStride = sourceStride;
        p.Other[0] = static_cast<const T*>(gateWeights);
        p.Other[1] = static_cast<const T*>(upWeights);
        p.OtherStride = expertStride;
        p.N = static_cast<uint32_t>(hidden);
        p.K = static_cast<uint32_t>(width);
        p.Result[0] = static_cast<T*>(result);
        p.ResultStride = resultStride;
        p.Kept = static_cast<TAcc<T>*>(kept);
        p.Activation = activation;
        MultiplyBy<kRows, 2>(call, p);
    });
}

void GatedRowsBackward(int valueType, int activation, size_t rows, size_t width, size_t hidden, int32_t experts, const int32_t* offsets,
                       const void* resultGradients, size_t gradientStride, const void* source, size_t sourceStride, const void* gateWeights,
                       const void* upWeights, size_t expertStride, const void* kept, void* preGradients, void* sourceGradients,
                       size_t sourceGradientStride, void* gateGradients, void* upGradients, size_t expertGradientStride, void* stream) {
    const size_t size = ValueSize(valueType);
    CBAMD_ENSURE(activation >= CBHIP_SILU && activation <= CBHIP_RELU, "unknown activation " + std::to_string(activation));
    CheckRouted(rows, width, hidden, experts, offsets);
    CBAMD_ENSURE((gateGradients == nullptr) == (upGradients == nullptr), "gradients of one projection alone are not supported");
    const bool ofRows = rows > 0 && hidden > 0, ofSource = sourceGradients != nullptr && rows > 0 && width > 0;
    const bool ofWeights = gateGradients != nullptr && hidden > 0 && width > 0;
    if (!ofRows && !ofSource && !ofWeights) {
        return;
    }
    if (ofRows) {
        CheckMatrix("result gradients", resultGradients, rows, hidden, gradientStride, size);
        CheckMatrix("kept values", kept, rows, 2 * hidden, 2 * hidden, std::max<size_t>(size, 4));
        CheckMatrix("gate and up gradients", preGradients, rows, 2 * hidden, 2 * hidden, size);
        CBAMD_ENSURE(preGradients != kept || size >= 4, "gate and up gradients of 16-bit values need memory of their own");
    }
    if (ofSource) {
        CheckWeights("gate weights", gateWeights, hidden, width, experts, expertStride, size);
        CheckWeights("up weights", upWeights, hidden, width, experts, expertStride, size);
        CheckMatrix("source gradients", sourceGradients, rows, width, sourceGradientStride, size);
    }
    if (ofWeights) {
        if (rows > 0) {
            CheckMatrix("source", source, rows, width, sourceStride, size);
        }
        CheckWeights("gate weight gradients", gateGradients, hidden, width, experts, expertGradientStride, size);
        CheckWeights("up weight gradients", upGradients, hidden, width, experts, expertGradientStride, size);
    }
    const TCallDevice call(ofRows ? preGradients : ofSource ? sourceGradients : gateGradients, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        TProduct<T> p = ProductOf<T>(rows, experts, offsets);
        if (ofRows) {
            const auto launch = [&](auto values) {
                constexpr int N = decltype(values)::value;
                const uint32_t rowPieces = static_cast<uint32_t>((hidden + N - 1) / N);
                const uint64_t pieces = static_cast<uint64_t>(rows) * rowPieces;
                for (uint64_t first = 0; first < pieces; first += kMostGroups * 256) {
                    call.Launch(GateGradientsKernel<T, N>, std::min(kMostGroups, (pieces - first + 255) / 256), 256, 0, p.Segments, first, pieces, rowPieces,
                                static_cast<uint32_t>(hidden), activation, static_cast<const T*>(resultGradients), gradientStride, static_cast<const TAcc<T>*>(kept),
                                static_cast<T*>(preGradients));
                }
            };
            launch(std::integral_constant<int, 16 / sizeof(T)>());
        }
        p.Source = static_cast<const T*>(preGradients);
        p.SourceStride = 2 * hidden;
        if (ofSource) {
            p.Other[0] = static_cast<const T*>(gateWeights);
            p.Other[1] = static_cast<const T*>(upWeights);
            p.OtherStride = expertStride;
            p.N = static_cast<uint32_t>(width);
            p.K = static_cast<uint32_t>(hidden);
            p.Result[0] = static_cast<T*>(sourceGradients);
            p.ResultStride = sourceGradientStride;
            MultiplyBy<kInputs, 2>(call, p);
        }
        if (ofWeights) {
            p.Other[0] = static_cast<const T*>(source);
            p.OtherStride = sourceStride;
            p.M = static_cast<uint32_t>(hidden);
            p.N = static_cast<uint32_t>(width);
            p.Result[0] = static_cast<T*>(gateGradients);
            p.Result[1] = static_cast<T*>(upGradients);
            p.ResultStride = expertGradientStride;
            MultiplyBy<kWeights, 2>(call, p);
        }
    });
}

void MultiplyRows(int valueType, size_t rows, size_t width, size_t outputs, int32_t experts, const int32_t* offsets, const void* source,
                  size_t sourceStride, const void* weights, size_t expertStride, void* result, size_t resultStride, void* stream) {
    const size_t size = ValueSize(valueType);
    CheckRouted(rows, width, outputs, experts, offsets);
    if (rows == 0 || outputs == 0) {
        return;
    }
    if (width > 0) {
        CheckMatrix("source", source, rows, width, sourceStride, size);
    }
    CheckWeights("weights", weights, outputs, width, experts, expertStride, size);
    CheckMatrix("result", result, rows, outputs, resultStride, size);
    const TCallDevice call(result, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        TProduct<T> p = ProductOf<T>(rows, experts, offsets);
        p.Source = static_cast<const T*>(source);
        p.SourceStride = sourceStride;
        p.Other[0] = static_cast<const T*>(weights);
        p.OtherStride = expertStride;
        p.N = static_cast<uint32_t>(outputs);
        p.K = static_cast<uint32_t>(width);
        p.Result[0] = static_cast<T*>(result);
        p.ResultStride = resultStride;
        MultiplyBy<kRows, 1>(call, p);
    });
}

void MultiplyRowsBackward(int valueType, size_t rows, size_t width, size_t outputs, int32_t experts, const int32_t* offsets,
                          const void* resultGradients, size_t gradientStride, const void* source, size_t sourceStride, const void* weights,
                          size_t expertStride, void* sourceGradients, size_t sourceGradientStride, void* weightGradients,
                          size_t expertGradientStride, void* stream) {
    const size_t size = ValueSize(valueType);
    CheckRouted(rows, width, outputs, experts, offsets);
    const bool ofSource = sourceGradients != nullptr && rows > 0 && width > 0, ofWeights = weightGradients != nullptr && outputs > 0 && width > 0;
    if (!ofSource && !ofWeights) {
        return;
    }
    if (rows > 0 && outputs > 0) {
        CheckMatrix("result gradients", resultGradients, rows, outputs, gradientStride, size);
    }
    if (ofSource) {
        CheckWeights("weights", weights, outputs, width, experts, expertStride, size);
        CheckMatrix("source gradients", sourceGradients, rows, width, sourceGradientStride, size);
    }
    if (ofWeights) {
        if (rows > 0) {
            CheckMatrix("source", source, rows, width, sourceStride, size);
        }
        CheckWeights("weight gradients", weightGradients, outputs, width, experts, expertGradientStride, size);
    }
    const TCallDevice call(ofSource ? sourceGradients : weightGradients, stream);
    WithType(valueType, [&](auto value) {
        using T = decltype(value);
        TProduct<T> p = ProductOf<T>(rows, experts, offsets);
        p.Source = static_cast<const T*>(resultGradients);
        p.SourceStride = gradientStride;
        if (ofSource) {
            p.Other[0] = static_cast<const T*>(weights);
            p.OtherStride = expertStride;
            p.N = static_cast<uint32_t>(width);
            p.K = static_cast<uint32_t>(outputs);
            p.Result[0] = static_cast<T*>(sourceGradients);
            p.ResultStride = sourceGradientStride;
            MultiplyBy<kInputs, 1>(call, p);
        }
        if (ofWeights) {
            p.Other[0] = static_cast<const T*>(source);
            p.OtherStride = sourceStride;
            p.M = static_cast<uint32_t>(outputs);
            p.N = static_cast<uint32_t>(width);
            p.Result[0] = static_cast<T*>(weightGradients);
            p.ResultStride = expertGradientStride;
            MultiplyBy<kWeights, 1>(call, p);
        }
    });
}

}  // namespace cbamd
