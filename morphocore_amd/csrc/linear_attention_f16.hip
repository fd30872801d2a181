// Linear attention over sequences of float16 operands (linear_attention.hpp).
#include "linear_attention.hpp"

namespace mca
{

MCA_LINEAR_ATTENTION(_Float16);

}  // namespace mca
