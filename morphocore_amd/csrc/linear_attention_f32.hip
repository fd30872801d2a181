// Linear attention over sequences of float32 operands (linear_attention.hpp).
#include "linear_attention.hpp"

namespace mca
{

MCA_LINEAR_ATTENTION(float);

}  // namespace mca
