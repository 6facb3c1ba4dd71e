// y = f(x w^T + b) + r and its backward pass: dispatch over the element types, whose kernels each stand in one object file
// of their own (mpe_linear_<type>.hip).
#include "mpe_learn.hpp"

namespace mpe {

static const LinearOps& ops_of(int dtype) { return dtype == MPE_F32 ? linear_f32() : dtype == MPE_BF16 ? linear_bf16() : linear_f16(); }

long long linear_forward_workspace(int, long long, long long, long long) { return 0; }

long long linear_backward_workspace(int dtype, int act, long long m, long long n, long long k) { return ops_of(dtype).backward_workspace(act, m, n, k); }

hipError_t launch_linear_forward(const LinearArgs& a, hipStream_t st) { return ops_of(a.dtype).forward(a, st); }

hipError_t launch_linear_backward(const LinearArgs& a, hipStream_t st) { return ops_of(a.dtype).backward(a, st); }

}  // namespace mpe
