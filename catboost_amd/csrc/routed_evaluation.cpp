// Documents evaluated by models of their own: sorted by model, each model on its documents, raw values back and mixed.
#include "routed_evaluation.h"
#include "operators.h"

#include <algorithm>
#include <string>
#include <vector>

namespace cbamd {

namespace {

// What the call keeps in the caller's workspace, each part at a multiple of 256 bytes
struct TParts {
    size_t Width = 0, CatWidth = 0, Dimension = 0, SortBytes = 0, Bytes = 0;
    size_t Places = 0, Offsets = 0, Sort = 0, Floats = 0, Cats = 0, Results = 0;

    TParts(const std::vector<THipEvaluator*>& evaluators, int layout, size_t slots) {
        for (const THipEvaluator* e : evaluators) {
            const THipEvaluator::TRowSizes sizes = e->GetRowSizes();
            Width = std::max(Width, layout == TFeatureBatch::FlatRows ? sizes.Flat : sizes.Floats);
            CatWidth = std::max(CatWidth, layout == TFeatureBatch::FlatRows ? size_t(0) : sizes.Cats);
        }
        Dimension = static_cast<size_t>(evaluators[0]->GetApproxDimension());
        SortBytes = SortByExpertBytes(slots, static_cast<int32_t>(evaluators.size()));
        const auto take = [this](size_t bytes) {
            const size_t at = Bytes;
            Bytes += (bytes + 255) / 256 * 256;
            return at;
        };
        Places = take(slots * 4);
        Offsets = take((evaluators.size() + 1) * 4);
        Sort = take(SortBytes);
        Floats = take(slots * Width * 4);
        Cats = take(slots * CatWidth * 4);
        Results = take(slots * Dimension * 8);
    }
};

void Check(const std::vector<THipEvaluator*>& evaluators, int layout, size_t docCount, int32_t perDoc) {
    CBAMD_ENSURE(!evaluators.empty() && evaluators.size() <= 1024, "evaluators: " + std::to_string(evaluators.size()) + ", 1 to 1024 are supported");
    CBAMD_ENSURE(layout == TFeatureBatch::FlatRows || layout == TFeatureBatch::SplitRows, "documents that are routed have their features in rows");
    CBAMD_ENSURE(perDoc >= 1 && perDoc <= 64, "evaluators per document: " + std::to_string(perDoc) + ", 1 to 64 are supported");
    CBAMD_ENSURE(docCount <= 0x7fffffffu / static_cast<size_t>(perDoc), "too many documents to route: " + std::to_string(docCount));
    for (const THipEvaluator* e : evaluators) {
        CBAMD_ENSURE(e->GetApproxDimension() == evaluators[0]->GetApproxDimension(), "evaluators of different dimensions");
        CBAMD_ENSURE(e->GetDeviceId() == evaluators[0]->GetDeviceId(), "evaluators on different devices");
    }
}

}  // namespace

size_t EvalRoutedBytes(const std::vector<THipEvaluator*>& evaluators, int layout, size_t docCount, int32_t perDoc) {
    Check(evaluators, layout, docCount, perDoc);
    return TParts(evaluators, layout, docCount * perDoc).Bytes;
}

void EvalRouted(const std::vector<THipEvaluator*>& evaluators, const TFeatureBatch& batch, size_t docCount, int32_t perDoc,
                const int32_t* experts, const double* weights, double* results, void* workspace, size_t workspaceBytes, void* stream) {
    Check(evaluators, batch.Layout, docCount, perDoc);
    if (docCount == 0) {
        return;
    }
    const size_t slots = docCount * perDoc;
    const TParts parts(evaluators, batch.Layout, slots);
    CBAMD_ENSURE(experts != nullptr && results != nullptr, "evaluator indexes or results pointer is null");
    CBAMD_ENSURE(workspace != nullptr && workspaceBytes >= parts.Bytes,
                 "workspace of " + std::to_string(workspaceBytes) + " bytes, " + std::to_string(parts.Bytes) + " are needed");
    CBAMD_ENSURE(reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "workspace pointer is not a multiple of 8");
    for (const THipEvaluator* e : evaluators) {
        e->CheckBatch(batch, docCount);
    }
    if (stream == nullptr) {
        stream = evaluators[0]->GetStream();
    }
    uint8_t* base = static_cast<uint8_t*>(workspace);
    int32_t* places = reinterpret_cast<int32_t*>(base + parts.Places);
    int32_t* offsets = reinterpret_cast<int32_t*>(base + parts.Offsets);
    double* sortedResults = reinterpret_cast<double*>(base + parts.Results);
    const int32_t count = static_cast<int32_t>(evaluators.size());

    try {
        SortByExpert(slots, count, experts, places, offsets, base + parts.Sort, parts.SortBytes, stream);
        DispatchRows(CBHIP_FLOAT32, docCount, parts.Width, perDoc, batch.Floats, batch.Stride, places, base + parts.Floats, slots, parts.Width, stream);
        DispatchRows(CBHIP_FLOAT32, docCount, parts.CatWidth, perDoc, batch.Cats, batch.CatStride, places, base + parts.Cats, slots, parts.CatWidth, stream);
        std::vector<int32_t> begin(evaluators.size() + 1);
        evaluators[0]->CopyToHost(begin.data(), offsets, begin.size() * 4, stream);
        TFeatureBatch sorted;
        sorted.Layout = batch.Layout;
        sorted.Stride = parts.Width;
        sorted.CatStride = parts.CatWidth;
        for (size_t e = 0; e < evaluators.size(); ++e) {
            const size_t first = static_cast<size_t>(begin[e]), n = static_cast<size_t>(begin[e + 1] - begin[e]);
            if (n == 0) {
                continue;
            }
            sorted.Floats = reinterpret_cast<const float*>(base + parts.Floats) + first * parts.Width;
            sorted.Cats = parts.CatWidth > 0 ? reinterpret_cast<const int32_t*>(base + parts.Cats) + first * parts.CatWidth : nullptr;
            evaluators[e]->CalcDevice(sorted, n, 0, evaluators[e]->GetTreeCount(), sortedResults + first * parts.Dimension, stream);
        }
        CombineRows(CBHIP_FLOAT64, docCount, parts.Dimension, perDoc, sortedResults, slots, parts.Dimension, places, weights, results, parts.Dimension, stream);
        evaluators[0]->Synchronize(stream);
    } catch (...) {
        // nothing that was launched goes on in the workspace after the call
        try {
            evaluators[0]->Synchronize(stream);
        } catch (...) {
        }
        throw;
    }
}

}  // namespace cbamd
