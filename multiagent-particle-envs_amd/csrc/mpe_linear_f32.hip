// A layer's passes in float32.
#include "mpe_linear_run.hpp"

namespace mpe {

const LinearOps& linear_f32() {
    static const LinearOps ops = {LinearRun<float>::backward_workspace, LinearRun<float>::forward, LinearRun<float>::backward};
    return ops;
}

}  // namespace mpe
