// Global norm over many tensors, and clipping to it:  n = sqrt(sum of g^2 over all tensors),  g' = g * s with
// s = max_norm / n where n > max_norm and 1 otherwise.
//
// Two passes that cannot be one: the factor is known only after the last element.  The squares are summed in float64
// (a float32 gradient above 1.8e19 would overflow its square, one below 1e-23 would lose it), every workgroup leaves one
// partial sum, and every workgroup of the second pass adds all partial sums in the same order: no atomics, so a result
// does not change from run to run.
#include "mpe_learn.hpp"

namespace mpe {

namespace {

constexpr int TENSORS = 120;        // per launch: the table travels as kernel arguments (under 4 KB)
constexpr int BLOCKS = MPE_CLIP_WORKSPACE_BYTES / 8;    // partial sums, one a workgroup
constexpr int CHUNK = 8192;         // elements a workgroup takes at a time

struct Table {
    const void* src[TENSORS];
    void* dst[TENSORS];
    long long count[TENSORS];
    unsigned first[TENSORS + 1];    // index of the tensor's first chunk
    uint8_t dtype[TENSORS];
};

template <typename T>
__device__ double chunk_squares(const T* p, int n) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) {
        const double g = (double)(float)p[i];
        s += g * g;
    }
    return s;
}

template <typename T>
__device__ void chunk_scale(const T* p, T* q, int n, float f, float f2) {
    for (int i = threadIdx.x; i < n; i += 256) q[i] = (T)((float)p[i] * f * f2);
}

// the tensor that chunk c belongs to
__device__ inline int find(const Table& t, int n, unsigned c) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(256) void norm_kernel(const Table t, int n, int more, double* __restrict__ partial) {
    __shared__ double scratch[4];
    double s = 0.0;
    for (unsigned c = blockIdx.x; c < t.first[n]; c += gridDim.x) {
        const int i = find(t, n, c);
        const long long at = (long long)(c - t.first[i]) * CHUNK;
        const int len = (int)min((long long)CHUNK, t.count[i] - at);
        if (t.dtype[i] == MPE_F32) s += chunk_squares((const float*)t.src[i] + at, len);
        else if (t.dtype[i] == MPE_BF16) s += chunk_squares((const bf16*)t.src[i] + at, len);
        else s += chunk_squares((const f16*)t.src[i] + at, len);
    }
    s = block_sum<4>(s, scratch);
    if (threadIdx.x == 0) partial[blockIdx.x] = more ? partial[blockIdx.x] + s : s;
}

__global__ __launch_bounds__(256) void scale_kernel(const Table t, int n, const double* __restrict__ partial, int n_partial, double max_norm,
                                                    float* __restrict__ norm_out) {
    __shared__ double scratch[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < n_partial; i += 256) s += partial[i];
    const double norm = sqrt(block_sum<4>(s, scratch));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const bool keep = norm <= max_norm;         // false for NaN: the factor below is then NaN
    // a factor too small for a normal float32 is applied in two steps, the second a power of two
    const double f_all = keep ? 1.0 : max_norm / norm;
    const bool small = f_all < 0x1p-100;
    const float f = (float)(small ? f_all * 0x1p100 : f_all), f2 = small ? 0x1p-100f : 1.0f;
    for (unsigned c = blockIdx.x; c < t.first[n]; c += gridDim.x) {
        const int i = find(t, n, c);
        if (!t.dst[i] || (keep && t.dst[i] == t.src[i])) continue;
        const long long at = (long long)(c - t.first[i]) * CHUNK;
        const int len = (int)min((long long)CHUNK, t.count[i] - at);
        if (t.dtype[i] == MPE_F32) chunk_scale((const float*)t.src[i] + at, (float*)t.dst[i] + at, len, f, f2);
        else if (t.dtype[i] == MPE_BF16) chunk_scale((const bf16*)t.src[i] + at, (bf16*)t.dst[i] + at, len, f, f2);
        else chunk_scale((const f16*)t.src[i] + at, (f16*)t.dst[i] + at, len, f, f2);
    }
}

}  // namespace

hipError_t launch_clip(int n, const void* const* src, void* const* dst, const int64_t* count, const int32_t* dtype, double max_norm,
                       float* norm, double* ws, hipStream_t st) {
    // one grid for every group of tensors, so that workgroup b of a later launch adds to partial sum b of the first
    unsigned grid = 1;
    for (int g = 0; g < n; g += TENSORS) {
        long long chunks = 0;
        for (int i = g; i < n && i < g + TENSORS; ++i) chunks += (count[i] + CHUNK - 1) / CHUNK;
        if (chunks > 0x7fffffffLL) return hipErrorInvalidValue;
        if (chunks > grid) grid = chunks < BLOCKS ? (unsigned)chunks : BLOCKS;
    }
    for (int pass = 0; pass < 2; ++pass) {
        int g = 0;
        do {
            Table t;
            const int here = n - g < TENSORS ? n - g : TENSORS;
            t.first[0] = 0;
            for (int i = 0; i < here; ++i) {
                t.src[i] = src[g + i];
                t.dst[i] = dst ? dst[g + i] : nullptr;
                t.count[i] = count[g + i];
                t.dtype[i] = (uint8_t)dtype[g + i];
                t.first[i + 1] = t.first[i] + (unsigned)((count[g + i] + CHUNK - 1) / CHUNK);
            }
            if (pass == 0) hipLaunchKernelGGL(norm_kernel, dim3(grid), dim3(256), 0, st, t, here, g > 0, ws);
            else hipLaunchKernelGGL(scale_kernel, dim3(dst ? grid : 1), dim3(256), 0, st, t, dst ? here : 0, ws, (int)grid, max_norm, g ? nullptr : norm);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            g += TENSORS;
        } while (g < n && (pass == 0 || dst));
    }
    return hipSuccess;
}

}  // namespace mpe
