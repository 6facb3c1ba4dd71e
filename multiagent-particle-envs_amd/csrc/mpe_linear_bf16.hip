// A layer's passes in bfloat16.
#include "mpe_linear_run.hpp"

namespace mpe {

template struct LinearRun<bf16>;

}  // namespace mpe
