// A layer's passes in float32.
#include "mpe_linear_run.hpp"

namespace mpe {

template struct LinearRun<float>;

}  // namespace mpe
