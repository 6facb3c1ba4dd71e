// Shared by the trainer-side kernels (mpe_linear*.hip, mpe_ppo.hip, mpe_clip.hip): element types, their conversions, the
// reductions, and the launcher entry points.  Every sum, softmax statistic and norm is held in 32 bits or more; a value
// is rounded to 16 bits only where it leaves a kernel in that type or enters a matrix instruction of that type.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/mpe_hip.h"

namespace mpe {

typedef __bf16 bf16;
typedef _Float16 f16;

inline int dtype_bytes(int dtype) { return dtype == MPE_F64 ? 8 : dtype == MPE_F32 ? 4 : 2; }
inline bool learn_dtype(int dtype) { return dtype == MPE_F32 || dtype == MPE_BF16 || dtype == MPE_F16; }

// Calls f with a value of the element type that `dtype` names (one of the three that learn_dtype accepts).
template <typename F>
inline hipError_t with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case MPE_F32: return f(float(0));
        case MPE_BF16: return f(bf16(0));
        default: return f(f16(0));
    }
}

// exp by the hardware's 2^x: off by the rounding of x log2(e), |x| 2^-24, and one step
__device__ inline float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// f over the lanes of a wave, the result in all of them.  Within 16 lanes by DPP, which costs a few cycles where a shuffle
// through LDS costs some 70: neighbours, pairs, then the mirror image of 8 and of 16 lanes.
template <int CTRL>
__device__ inline float dpp(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true)); }
template <int CTRL>
__device__ inline double dpp(double v) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    const i32x2 a = __builtin_bit_cast(i32x2, v);
    const i32x2 r = {__builtin_amdgcn_update_dpp(0, a[0], CTRL, 0xf, 0xf, true), __builtin_amdgcn_update_dpp(0, a[1], CTRL, 0xf, 0xf, true)};
    return __builtin_bit_cast(double, r);
}
template <typename V, typename F>
__device__ inline V wave_reduce(V v, F&& f) {
    v = f(v, dpp<0xb1>(v));
    v = f(v, dpp<0x4e>(v));
    v = f(v, dpp<0x141>(v));
    v = f(v, dpp<0x140>(v));
    v = f(v, __shfl_xor(v, 16));
    return f(v, __shfl_xor(v, 32));
}

template <typename V>
__device__ inline V wave_sum(V v) { return wave_reduce(v, [](V a, V b) { return a + b; }); }

// Sum over a workgroup of WAVES waves, in a fixed order; the result is valid in every thread.  `scratch` holds WAVES
// doubles and may be reused after the call's next barrier.
template <int WAVES>
__device__ inline double block_sum(double v, double* scratch) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < WAVES; ++i) s += scratch[i];
    return s;
}

// ---- y = f(x w^T + b) + r (mpe_linear.hip) ----
struct LinearArgs {
    int dtype, act;
    long long m, n, k;
    const void* x;
    long long ldx;
    const void* w;
    long long ldw;
    const void* bias;       // may be null
    const void* residual;   // may be null
    long long ldr;
    void* y;
    long long ldy;
    void* pre;              // pre-activations [m][n], may be null (forward); saved by the forward (backward)
    const void* dy;
    long long lddy;
    void* dx;               // may be null
    long long lddx;
    void* dw;               // may be null
    void* db;               // may be null
    void* ws;
};
// one element type's passes
struct LinearOps {
    long long (*backward_workspace)(int act, long long m, long long n, long long k);
    hipError_t (*forward)(const LinearArgs& a, hipStream_t st);
    hipError_t (*backward)(const LinearArgs& a, hipStream_t st);
};
const LinearOps& linear_f32();
const LinearOps& linear_bf16();
const LinearOps& linear_f16();
long long linear_forward_workspace(int dtype, long long m, long long n, long long k);
long long linear_backward_workspace(int dtype, int act, long long m, long long n, long long k);
hipError_t launch_linear_forward(const LinearArgs& a, hipStream_t st);
hipError_t launch_linear_backward(const LinearArgs& a, hipStream_t st);

// ---- global norm and clipping (mpe_clip.hip) ----
hipError_t launch_clip(int n, const void* const* src, void* const* dst, const int64_t* count, const int32_t* dtype, double max_norm,
                       float* norm, double* ws, hipStream_t st);

// ---- policy loss (mpe_ppo.hip) ----
struct PpoArgs {
    int dtype;
    long long rows, v;
    const void* logits;
    long long ld;
    const void* actions;
    int action_bytes;
    const float *old_logp, *adv;
    const uint8_t* mask;    // may be null
    long long ldm;
    const float* weights;   // may be null
    const float *values, *old_values, *returns;     // all or none
    float clip, value_clip, value_coef, entropy_coef;   // value_clip < 0: values are not clipped
    float *loss, *stats;
    const float* grad;      // backward: d(objective)/d(loss), one device float
    void* dlogits;
    long long ldd;
    float* dvalues;
    double* ws;
};
hipError_t launch_ppo_forward(const PpoArgs& a, hipStream_t st);
hipError_t launch_ppo_backward(const PpoArgs& a, hipStream_t st);

}  // namespace mpe
