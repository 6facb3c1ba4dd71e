// y = f(x w^T + b) + r and its backward pass: dispatch over the element types (mpe_linear_<type>.hip).
#include "mpe_linear_run.hpp"

namespace mpe {

extern template struct LinearRun<float>;
extern template struct LinearRun<bf16>;
extern template struct LinearRun<f16>;

long long linear_forward_workspace(int, long long, long long, long long) { return 0; }

long long linear_backward_workspace(int dtype, int act, long long m, long long n, long long k) {
    switch (dtype) {
        case MPE_F32: return LinearRun<float>::backward_workspace(act, m, n, k);
        case MPE_BF16: return LinearRun<bf16>::backward_workspace(act, m, n, k);
        default: return LinearRun<f16>::backward_workspace(act, m, n, k);
    }
}

hipError_t launch_linear_forward(const LinearArgs& a, hipStream_t st) {
    return with_dtype(a.dtype, [&](auto z) { return LinearRun<decltype(z)>::forward(a, st); });
}

hipError_t launch_linear_backward(const LinearArgs& a, hipStream_t st) {
    return with_dtype(a.dtype, [&](auto z) { return LinearRun<decltype(z)>::backward(a, st); });
}

}  // namespace mpe
