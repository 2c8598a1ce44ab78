// The experts' products of bfloat16 values.
#include "expert_products.hip.h"

namespace cbamd {
namespace op {

template void MultiplyBy<kRows, 1, __bf16>(const TCallDevice&, const TProduct<__bf16>&);
template void MultiplyBy<kRows, 2, __bf16>(const TCallDevice&, const TProduct<__bf16>&);

}  // namespace op
}  // namespace cbamd
