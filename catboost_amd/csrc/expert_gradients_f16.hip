// The experts' products' gradients of 16-bit values.
#include "expert_products.hip.h"

namespace cbamd {
namespace op {

template void MultiplyBy<kInputs, 1, _Float16>(const TCallDevice&, const TProduct<_Float16>&);
template void MultiplyBy<kInputs, 2, _Float16>(const TCallDevice&, const TProduct<_Float16>&);
template void MultiplyBy<kWeights, 1, _Float16>(const TCallDevice&, const TProduct<_Float16>&);
template void MultiplyBy<kWeights, 2, _Float16>(const TCallDevice&, const TProduct<_Float16>&);

}  // namespace op
}  // namespace cbamd
