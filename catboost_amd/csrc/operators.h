// Operators on scores and on routed rows in device memory (include/cb_hip_evaluator.h says what each does).
// No HIP types appear in this header. All throw TModelError and are asynchronous on `stream` (a hipStream_t,
// nullptr: the default stream of the output's device).
#pragma once

#include "../../include/cb_hip_evaluator.h"
#include "model.h"

#include <cstddef>
#include <cstdint>

namespace cbamd {

void AdjustScores(int valueType, size_t rows, size_t classes, const void* scores, size_t scoreStride,
                  const CbHipScoreAdjustment& adjustment, void* result, size_t resultStride, void* stream);

void SelectTop(int valueType, size_t rows, size_t classes, const void* scores, size_t scoreStride, int32_t count,
               bool amongSelected, int32_t* indexes, void* weights, void* stream);
void SelectTopBackward(int valueType, size_t rows, size_t classes, const void* scores, size_t scoreStride, int32_t count,
                       bool amongSelected, const int32_t* indexes, const void* weights, const void* weightGradients,
                       void* scoreGradients, size_t gradientStride, void* stream);

size_t SortByExpertBytes(size_t slots, int32_t experts);
void SortByExpert(size_t slots, int32_t experts, const int32_t* ids, int32_t* places, int32_t* offsets, void* workspace,
                  size_t workspaceBytes, void* stream);
void DispatchRows(int valueType, size_t rows, size_t width, int32_t perRow, const void* source, size_t sourceStride,
                  const int32_t* places, void* sorted, size_t sortedRows, size_t sortedStride, void* stream);
void CombineRows(int valueType, size_t rows, size_t width, int32_t perRow, const void* sorted, size_t sortedRows,
                 size_t sortedStride, const int32_t* places, const void* weights, void* result, size_t resultStride,
                 void* stream);
void CombineRowsBackward(int valueType, size_t rows, size_t width, int32_t perRow, const void* resultGradients,
                         size_t gradientStride, const void* sorted, size_t sortedRows, size_t sortedStride,
                         const int32_t* places, const void* weights, void* sortedGradients,
                         size_t sortedGradientStride, void* weightGradients, void* stream);

}  // namespace cbamd
