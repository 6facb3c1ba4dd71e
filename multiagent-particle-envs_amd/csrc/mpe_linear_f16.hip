// A layer's passes in float16.
#include "mpe_linear_run.hpp"

namespace mpe {

const LinearOps& linear_f16() {
    static const LinearOps ops = {LinearRun<f16>::backward_workspace, LinearRun<f16>::forward, LinearRun<f16>::backward};
    return ops;
}

}  // namespace mpe
