// The experts' products' gradients of bfloat16 values.
#include "expert_products.hip.h"

namespace cbamd {
namespace op {

template void MultiplyBy<kInputs, 1, __bf16>(const TCallDevice&, const TProduct<__bf16>&);
template void MultiplyBy<kInputs, 2, __bf16>(const TCallDevice&, const TProduct<__bf16>&);
template void MultiplyBy<kWeights, 1, __bf16>(const TCallDevice&, const TProduct<__bf16>&);
template void MultiplyBy<kWeights, 2, __bf16>(const TCallDevice&, const TProduct<__bf16>&);

}  // namespace op
}  // namespace cbamd
