// Experts' products on rows sorted by expert, and their gradients (include/cb_hip_evaluator.h): what a call is asked, and the gradients
// of gate and up values. The products' kernels are compiled for each type by itself.
#include "expert_products.hip.h"

namespace cbamd {
namespace op {

// ---------------------------------------------------------------- gradients of gate and up values ----

// preGradients[r] = (dh * up * act'(gate), dh * act(gate)) of the rows that experts have; N columns for a thread. The kept values are
// in 32 bits: rounded to bf16 they made the gradients 0.0031 off (in the norm) where rounding the gradients alone makes 0.0024. These are rounded to
// the value type, which the matrix cores multiply at 16 bits' rate: 0.0017 is the rounding of the results by itself, and what the rounding
// here takes away would be a second product for each of the four that follow.
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

// (compiled by expert_products_*.hip and expert_gradients_*.hip)
#define PRODUCTS_OF(T)                                                                        \
    extern template void MultiplyBy<kRows, 1, T>(const TCallDevice&, const TProduct<T>&);    \
    extern template void MultiplyBy<kRows, 2, T>(const TCallDevice&, const TProduct<T>&);    \
    extern template void MultiplyBy<kInputs, 1, T>(const TCallDevice&, const TProduct<T>&);  \
    extern template void MultiplyBy<kInputs, 2, T>(const TCallDevice&, const TProduct<T>&);  \
    extern template void MultiplyBy<kWeights, 1, T>(const TCallDevice&, const TProduct<T>&); \
    extern template void MultiplyBy<kWeights, 2, T>(const TCallDevice&, const TProduct<T>&);
PRODUCTS_OF(double)
PRODUCTS_OF(float)
PRODUCTS_OF(_Float16)
PRODUCTS_OF(__bf16)
#undef PRODUCTS_OF

}  // namespace op

using namespace op;

namespace {

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
