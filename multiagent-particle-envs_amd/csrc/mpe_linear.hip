// y = f(x w^T + b) + r and its backward pass.
#include "mpe_learn.hpp"

namespace mpe {

namespace {

__device__ inline float act_value(int act, float z) {
    switch (act) {
        case MPE_ACT_TANH: return tanhf(z);
        case MPE_ACT_RELU: return z > 0.0f || z != z ? z : 0.0f;
        case MPE_ACT_GELU: return 0.5f * z * erfcf(-0.70710678118654752f * z);
        case MPE_ACT_SILU: return z / (1.0f + expf(-z));
        default: return z;
    }
}

__device__ inline float act_slope(int act, float z) {
    switch (act) {
        case MPE_ACT_TANH: { const float t = tanhf(z); return 1.0f - t * t; }
        case MPE_ACT_RELU: return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
        case MPE_ACT_GELU: return 0.5f * erfcf(-0.70710678118654752f * z) + z * 0.39894228040143268f * expf(-0.5f * z * z);
        case MPE_ACT_SILU: { const float s = 1.0f / (1.0f + expf(-z)); return s * (1.0f + z * (1.0f - s)); }
        default: return 1.0f;
    }
}

// out[j][i] = sum_k P(i, k) Q(j, k), operands and output with element strides
template <typename T, bool FORWARD>
__global__ __launch_bounds__(256) void product(long long ni, long long nj, long long nk, const T* __restrict__ p, long long pi, long long pk,
                                               const T* __restrict__ q, long long qj, long long qk, T* out, long long ldo, int act,
                                               const T* __restrict__ bias, const T* residual, long long ldr, T* __restrict__ pre) {
    __shared__ float ps[16][17], qs[16][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long i0 = (long long)blockIdx.x * 16, j0 = (long long)blockIdx.y * 16;
    float acc = 0.0f;
    for (long long k0 = 0; k0 < nk; k0 += 16) {
        ps[ty][tx] = i0 + ty < ni && k0 + tx < nk ? (float)p[(i0 + ty) * pi + (k0 + tx) * pk] : 0.0f;
        qs[ty][tx] = j0 + ty < nj && k0 + tx < nk ? (float)q[(j0 + ty) * qj + (k0 + tx) * qk] : 0.0f;
        __syncthreads();
        for (int k = 0; k < 16; ++k) acc = fmaf(ps[tx][k], qs[ty][k], acc);
        __syncthreads();
    }
    const long long i = i0 + tx, j = j0 + ty;
    if (i >= ni || j >= nj) return;
    if (FORWARD) {
        if (bias) acc += (float)bias[i];
        if (pre) pre[j * ni + i] = (T)acc;
        acc = act_value(act, acc);
        if (residual) acc += (float)residual[j * ldr + i];
    }
    out[j * ldo + i] = (T)acc;
}

template <typename T>
__global__ __launch_bounds__(256) void slope_pass(long long m, long long n, const T* __restrict__ dy, long long lddy, const T* __restrict__ pre,
                                                  int act, T* __restrict__ dz) {
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= m * n) return;
    const long long j = at / n, i = at - j * n;
    dz[at] = (T)((float)dy[j * lddy + i] * (pre ? act_slope(act, (float)pre[at]) : 1.0f));
}

template <typename T>
__global__ __launch_bounds__(256) void column_sum(long long m, long long n, const T* __restrict__ dz, T* __restrict__ db) {
    __shared__ double scratch[4];
    double s = 0.0;
    for (long long j = threadIdx.x; j < m; j += 256) s += (double)(float)dz[j * n + blockIdx.x];
    s = block_sum<4>(s, scratch);
    if (threadIdx.x == 0) db[blockIdx.x] = (T)(float)s;
}

}  // namespace

long long linear_forward_workspace(int, long long, long long, long long) { return 0; }
long long linear_backward_workspace(int dtype, int, long long m, long long n, long long) { return m * n * dtype_bytes(dtype); }

hipError_t launch_linear_forward(const LinearArgs& a, hipStream_t st) {
    return with_dtype(a.dtype, [&](auto z) {
        typedef decltype(z) T;
        const dim3 grid((unsigned)((a.n + 15) / 16), (unsigned)((a.m + 15) / 16));
        hipLaunchKernelGGL((product<T, true>), grid, dim3(256), 0, st, a.n, a.m, a.k, (const T*)a.w, a.ldw, 1LL, (const T*)a.x, a.ldx, 1LL,
                           (T*)a.y, a.ldy, a.act, (const T*)a.bias, (const T*)a.residual, a.ldr, (T*)a.pre);
        return hipGetLastError();
    });
}

hipError_t launch_linear_backward(const LinearArgs& a, hipStream_t st) {
    return with_dtype(a.dtype, [&](auto z) {
        typedef decltype(z) T;
        T* dz = (T*)a.ws;
        if (a.m > 0) hipLaunchKernelGGL((slope_pass<T>), dim3((unsigned)((a.m * a.n + 255) / 256)), dim3(256), 0, st, a.m, a.n, (const T*)a.dy, a.lddy, (const T*)a.pre, a.act, dz);
        if (a.dx && a.m > 0) {
            const dim3 grid((unsigned)((a.k + 15) / 16), (unsigned)((a.m + 15) / 16));
            hipLaunchKernelGGL((product<T, false>), grid, dim3(256), 0, st, a.k, a.m, a.n, (const T*)a.w, 1LL, a.ldw, (const T*)dz, a.n, 1LL,
                               (T*)a.dx, a.lddx, 0, (const T*)nullptr, (const T*)nullptr, 0LL, (T*)nullptr);
        }
        if (a.dw) {
            const dim3 grid((unsigned)((a.k + 15) / 16), (unsigned)((a.n + 15) / 16));
            hipLaunchKernelGGL((product<T, false>), grid, dim3(256), 0, st, a.k, a.n, a.m, (const T*)a.x, 1LL, a.ldx, (const T*)dz, 1LL, a.n,
                               (T*)a.dw, a.k, 0, (const T*)nullptr, (const T*)nullptr, 0LL, (T*)nullptr);
        }
        if (a.db) hipLaunchKernelGGL((column_sum<T>), dim3((unsigned)a.n), dim3(256), 0, st, a.m, a.n, (const T*)dz, (T*)a.db);
        return hipGetLastError();
    });
}

}  // namespace mpe
