// Documents evaluated by models of their own (CbHipEvalRouted of include/cb_hip_evaluator.h).
#pragma once

#include "hip_evaluator.h"

#include <vector>

namespace cbamd {

// `layout`: TFeatureBatch::ELayout
size_t EvalRoutedBytes(const std::vector<THipEvaluator*>& evaluators, int layout, size_t docCount, int32_t perDoc);
// waits for the stream (nullptr: the first evaluator's own)
void EvalRouted(const std::vector<THipEvaluator*>& evaluators, const TFeatureBatch& batch, size_t docCount, int32_t perDoc,
                const int32_t* experts, const double* weights, double* results, void* workspace, size_t workspaceBytes, void* stream);

}  // namespace cbamd
