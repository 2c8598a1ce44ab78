// The experts' products of 64-bit values.
#include "expert_products.hip.h"

namespace cbamd {
namespace op {

template void MultiplyBy<kRows, 1, double>(const TCallDevice&, const TProduct<double>&);
template void MultiplyBy<kRows, 2, double>(const TCallDevice&, const TProduct<double>&);
template void MultiplyBy<kInputs, 1, double>(const TCallDevice&, const TProduct<double>&);
template void MultiplyBy<kInputs, 2, double>(const TCallDevice&, const TProduct<double>&);
template void MultiplyBy<kWeights, 1, double>(const TCallDevice&, const TProduct<double>&);
template void MultiplyBy<kWeights, 2, double>(const TCallDevice&, const TProduct<double>&);

}  // namespace op
}  // namespace cbamd
