// A layer's passes in bfloat16.
#include "mpe_linear_run.hpp"

namespace mpe {

const LinearOps& linear_bf16() {
    static const LinearOps ops = {LinearRun<bf16>::backward_workspace, LinearRun<bf16>::forward, LinearRun<bf16>::backward};
    return ops;
}

}  // namespace mpe
