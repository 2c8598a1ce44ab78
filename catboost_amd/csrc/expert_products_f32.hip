// The experts' products of 32-bit values.
#include "expert_products.hip.h"

namespace cbamd {
namespace op {

template void MultiplyBy<kRows, 1, float>(const TCallDevice&, const TProduct<float>&);
template void MultiplyBy<kRows, 2, float>(const TCallDevice&, const TProduct<float>&);
template void MultiplyBy<kInputs, 1, float>(const TCallDevice&, const TProduct<float>&);
template void MultiplyBy<kInputs, 2, float>(const TCallDevice&, const TProduct<float>&);
template void MultiplyBy<kWeights, 1, float>(const TCallDevice&, const TProduct<float>&);
template void MultiplyBy<kWeights, 2, float>(const TCallDevice&, const TProduct<float>&);

}  // namespace op
}  // namespace cbamd
