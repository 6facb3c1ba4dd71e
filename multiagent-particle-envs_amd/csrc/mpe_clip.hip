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

// Four workgroups a CU: the norm of 302 M bfloat16 elements takes 133 us at 1024 workgroups (4.5 TB/s), 140 at 2048.  Scaling
// them takes 217 us (1.2 GB moved, 5.6 TB/s: part of it is still in the Infinity Cache).
constexpr int BLOCKS = 1024;
static_assert(BLOCKS * 8 <= MPE_CLIP_WORKSPACE_BYTES, "a partial sum for every workgroup");
// One workgroup takes everything below this: 10 630 elements in 7.9 us, where the two launches take 7.0 us on the GPU but
// some 4 us more of the host, which bounds calls of this size.
constexpr int TINY = 16384;
constexpr int CHUNK = 8192;         // elements a workgroup takes at a time
constexpr int WAVE_CHUNK = 512;     // and a wave where one workgroup takes everything

// Tensors of one launch: the table travels as kernel arguments, within 4 KB.  The norm needs no destinations.
template <int N, bool DST>
struct Table {
    const void* src[N];
    void* dst[DST ? N : 1];
    unsigned first[N + 1];          // index of the tensor's first chunk
    unsigned tail[N];               // elements of its last chunk << 2 | type
    static constexpr int TENSORS = N;
};
typedef Table<240, false> NormTable;
typedef Table<160, true> ScaleTable;
static_assert(sizeof(NormTable) <= 3968 && sizeof(ScaleTable) <= 3968, "kernel arguments");

// A chunk in 16-byte vectors: f(vector of E elements, how many of them are there).  Four loads are in flight at a time.
// Vectors need not lie on 16-byte borders: the memory takes them as they come.
template <typename T, int THREADS, typename F>
__device__ inline void each_vector(const T* p, int n, int tid, F&& f) {
    constexpr int E = 16 / (int)sizeof(T);
    int i = tid * E;
    for (; i + 3 * THREADS * E + E <= n; i += 4 * THREADS * E) {
        T v[4][E];
#pragma unroll
        for (int u = 0; u < 4; ++u) __builtin_memcpy(v[u], p + i + u * THREADS * E, 16);
#pragma unroll
        for (int u = 0; u < 4; ++u) f(i + u * THREADS * E, v[u], E);
    }
    for (; i < n; i += THREADS * E) {
        T v[E];
        const int have = min(E, n - i);
        if (have == E) __builtin_memcpy(v, p + i, 16);
        else
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = e < have ? p[i + e] : (T)0.0f;
        f(i, v, have);
    }
}

template <typename T, int THREADS>
__device__ double chunk_squares(const T* p, int n, int tid) {
    double s0 = 0.0, s1 = 0.0;
    each_vector<T, THREADS>(p, n, tid, [&](int, const T* v, int) {
#pragma unroll
        for (int e = 0; e < 16 / (int)sizeof(T); e += 2) {
            const double a = (double)(float)v[e], b = (double)(float)v[e + 1];
            s0 = fma(a, a, s0);
            s1 = fma(b, b, s1);
        }
    });
    return s0 + s1;
}

template <typename T, int THREADS>
__device__ void chunk_scale(const T* p, T* q, int n, int tid, float f, float f2) {
    each_vector<T, THREADS>(p, n, tid, [&](int i, const T* v, int have) {
        constexpr int E = 16 / (int)sizeof(T);
        T o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = (T)((float)v[e] * f * f2);
        if (have == E) __builtin_memcpy(q + i, o, 16);
        else
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < have) q[i + e] = o[e];
    });
}

// the tensor that chunk c belongs to
template <typename TABLE>
__device__ inline int find(const TABLE& t, int n, unsigned c) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

// runs f(element type, tensor, first element, length) on chunk c
template <int SIZE, typename TABLE, typename F>
__device__ inline void on_chunk(const TABLE& t, int n, unsigned c, F&& f) {
    const int i = find(t, n, c);
    const long long at = (long long)(c - t.first[i]) * SIZE;
    const int len = c + 1 == t.first[i + 1] ? (int)(t.tail[i] >> 2) : SIZE;
    switch (t.tail[i] & 3) {
        case MPE_F32: f(float(0), i, at, len); break;
        case MPE_BF16: f(bf16(0), i, at, len); break;
        default: f(f16(0), i, at, len);
    }
}

struct Factor {
    bool keep;
    float f, f2;
};

__device__ inline Factor factor_of(double norm, double max_norm) {
    Factor x;
    x.keep = norm <= max_norm;                  // false for NaN: the factor is then NaN
    // a factor too small for a normal float32 is applied in two steps, the second a power of two
    const double f = x.keep ? 1.0 : max_norm / norm;
    const bool small = f < 0x1p-100;
    x.f = (float)(small ? f * 0x1p100 : f);
    x.f2 = small ? 0x1p-100f : 1.0f;
    return x;
}

__global__ __launch_bounds__(256) void norm_kernel(const NormTable t, int n, int more, double* __restrict__ partial) {
    __shared__ double scratch[4];
    double s = 0.0;
    for (unsigned c = blockIdx.x; c < t.first[n]; c += gridDim.x)
        on_chunk<CHUNK>(t, n, c, [&](auto z, int i, long long at, int len) {
            s += chunk_squares<decltype(z), 256>((const decltype(z)*)t.src[i] + at, len, threadIdx.x);
        });
    s = block_sum<4>(s, scratch);
    if (threadIdx.x == 0) partial[blockIdx.x] = more ? partial[blockIdx.x] + s : s;
}

__global__ __launch_bounds__(256) void scale_kernel(const ScaleTable t, int n, const double* __restrict__ partial, int n_partial, double max_norm,
                                                    float* __restrict__ norm_out) {
    __shared__ double scratch[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < n_partial; i += 256) s += partial[i];
    const double norm = sqrt(block_sum<4>(s, scratch));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const Factor x = factor_of(norm, max_norm);
    // last chunk first: what the norm read last is still in the Infinity Cache
    for (unsigned b = blockIdx.x; b < t.first[n]; b += gridDim.x)
        on_chunk<CHUNK>(t, n, t.first[n] - 1 - b, [&](auto z, int i, long long at, int len) {
            typedef decltype(z) T;
            if (x.keep && t.dst[i] == t.src[i]) return;
            chunk_scale<T, 256>((const T*)t.src[i] + at, (T*)t.dst[i] + at, len, threadIdx.x, x.f, x.f2);
        });
}

// Few elements: one workgroup does both passes, the second from its L1 and L2, and there is one launch instead of two.
__global__ __launch_bounds__(1024) void clip_tiny(const ScaleTable t, int n, double max_norm, int scale, float* __restrict__ norm_out) {
    __shared__ double scratch[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    double s = 0.0;
    for (unsigned c = wave; c < t.first[n]; c += 16)
        on_chunk<WAVE_CHUNK>(t, n, c, [&](auto z, int i, long long at, int len) {
            s += chunk_squares<decltype(z), 64>((const decltype(z)*)t.src[i] + at, len, lane);
        });
    const double norm = sqrt(block_sum<16>(s, scratch));
    if (norm_out && threadIdx.x == 0) *norm_out = (float)norm;
    const Factor x = factor_of(norm, max_norm);
    if (!scale) return;
    for (unsigned c = wave; c < t.first[n]; c += 16)
        on_chunk<WAVE_CHUNK>(t, n, c, [&](auto z, int i, long long at, int len) {
            typedef decltype(z) T;
            if (x.keep && t.dst[i] == t.src[i]) return;
            chunk_scale<T, 64>((const T*)t.src[i] + at, (T*)t.dst[i] + at, len, lane, x.f, x.f2);
        });
}

// Fills t from tensor `from` on, empty ones left out; returns the first tensor that found no place.
template <typename TABLE>
int fill(TABLE& t, int& here, int from, int n, const void* const* src, void* const* dst, const int64_t* count, const int32_t* dtype, int size) {
    here = 0;
    t.first[0] = 0;
    for (; from < n && here < TABLE::TENSORS; ++from) {
        const int64_t k = count[from];
        if (k == 0) continue;
        const int64_t chunks = (k + size - 1) / size;
        if (chunks > 0x7fffffff - (int64_t)t.first[here]) break;     // chunk numbers are 31 bits a launch
        t.src[here] = src[from];
        if (sizeof(t.dst) > 8) t.dst[here] = dst ? dst[from] : nullptr;
        t.tail[here] = (unsigned)((k - (chunks - 1) * size) << 2 | (unsigned)dtype[from]);
        t.first[here + 1] = t.first[here] + (unsigned)chunks;
        ++here;
    }
    return from;
}

}  // namespace

hipError_t launch_clip(int n, const void* const* src, void* const* dst, const int64_t* count, const int32_t* dtype, double max_norm,
                       float* norm, double* ws, hipStream_t st) {
    int64_t total = 0;
    for (int i = 0; i < n; ++i) total += count[i];
    int here, next;
    if (total <= TINY) {
        ScaleTable t;
        if (fill(t, here, 0, n, src, dst, count, dtype, WAVE_CHUNK) == n) {
            hipLaunchKernelGGL(clip_tiny, dim3(1), dim3(1024), 0, st, t, here, max_norm, dst != nullptr, norm);
            return hipGetLastError();
        }
    }
    // one grid for every group of tensors, so that workgroup b of a later launch adds to partial sum b of the first
    int64_t most = 0;
    for (int g = 0; g < n; g = next) {
        NormTable t;
        next = fill(t, here, g, n, src, dst, count, dtype, CHUNK);
        if (t.first[here] > most) most = t.first[here];
    }
    const unsigned grid = most < 1 ? 1 : most < BLOCKS ? (unsigned)most : BLOCKS;
    for (int g = 0;; g = next) {
        NormTable t;
        next = fill(t, here, g, n, src, dst, count, dtype, CHUNK);
        hipLaunchKernelGGL(norm_kernel, dim3(grid), dim3(256), 0, st, t, here, g > 0, ws);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (next >= n) break;
    }
    if (!dst) {
        ScaleTable t;
        t.first[0] = 0;
        hipLaunchKernelGGL(scale_kernel, dim3(1), dim3(256), 0, st, t, 0, ws, (int)grid, max_norm, norm);
        return hipGetLastError();
    }
    // groups last to first, like the chunks within them
    for (int end = n; end > 0 || end == n; end = next) {
        ScaleTable t;
        next = end > ScaleTable::TENSORS ? end - ScaleTable::TENSORS : 0;
        while (fill(t, here, next, end, src, dst, count, dtype, CHUNK) < end) ++next;     // too many chunks for one launch
        hipLaunchKernelGGL(scale_kernel, dim3(grid), dim3(256), 0, st, t, here, ws, (int)grid, max_norm, end == n ? norm : nullptr);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (next == 0) break;
    }
    return hipSuccess;
}

}  // namespace mpe
