// Linear attention over sequences of bfloat16 operands (linear_attention.hpp).
#include "linear_attention.hpp"

namespace mca
{

MCA_LINEAR_ATTENTION(__bf16);

}  // namespace mca
