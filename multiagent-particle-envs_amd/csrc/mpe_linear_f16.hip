// A layer's passes in float16.
#include "mpe_linear_run.hpp"

namespace mpe {

template struct LinearRun<f16>;

}  // namespace mpe
