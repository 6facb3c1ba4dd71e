// The forward product for a few rows (one world's agents, one decision): the weights are the traffic, and the time is that of
// a single memory access if enough of them are in flight (4 x 1024 -> 4096 bf16: 8.4 MB in 3.9 us, 3 x 14 -> 64 f32 2.4 us, of
// which an empty launch takes 1.8).
#pragma once
#include <type_traits>

#include "mpe_linear_impl.hpp"

namespace mpe {

// eight consecutive elements as pieces
template <typename T> struct Frag {
    typedef typename Piece<T>::type PT;
    typedef PT pt8 __attribute__((ext_vector_type(8)));
    static constexpr int N = Piece<T>::N;
    pt8 c[N];
    template <typename V>
    __device__ inline void set(const V& f) {
        if constexpr (N == 3) {
            split3(f, c[0], c[1], c[2]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) c[0][e] = (PT)f[e];
        }
    }
};

// acc += P Q, the partial products of float32 smallest first
template <typename T>
__device__ inline f32x4 multiply(f32x4 acc, const Frag<T>& p, const Frag<T>& q) {
    constexpr int N = Frag<T>::N;
    if (N == 3) {
        acc = mfma(p.c[N - 1], q.c[0], acc);
        acc = mfma(p.c[0], q.c[N - 1], acc);
        acc = mfma(p.c[N / 2], q.c[N / 2], acc);
        acc = mfma(p.c[N / 2], q.c[0], acc);
        acc = mfma(p.c[0], q.c[N / 2], acc);
    }
    return mfma(p.c[0], q.c[0], acc);
}

// A workgroup of eight waves takes 16 outputs of up to 16 FJ rows; the waves share the sum and add up through LDS, wave
// after wave.  Operands go straight from memory into the instruction's layout (a lane reads eight consecutive elements of
// one row), AHEAD steps at a time.
template <typename T, int FJ>
__global__ __launch_bounds__(512) void forward_skinny(const ProductArgs<T> a) {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    constexpr int WAVES = 8, AHEAD = FJ == 1 ? 4 : 2;
    __shared__ float part[WAVES][FJ * 16][20];
    const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const long long i0 = (long long)blockIdx.x * 16, j0 = (long long)blockIdx.y * (16 * FJ);
    const int steps = (int)((a.nr + 31) / 32), each = (steps + WAVES - 1) / WAVES;
    const int t1 = min(steps, (wave + 1) * each);
    const unsigned row_p = (unsigned)min((long long)l, a.ni - 1 - i0);      // rows that are not there: the last one again, never stored
    unsigned row_q[FJ];
#pragma unroll
    for (int y = 0; y < FJ; ++y) row_q[y] = (unsigned)min((long long)(y * 16 + l), a.nj - 1 - j0);

    f32x4 acc[FJ];
    // a wave's share of the sums: on the matrix cores, or in plain float32, for which the lanes pass the elements around
    const auto share = [&](auto plain) __attribute__((always_inline)) {
#pragma unroll
        for (int y = 0; y < FJ; ++y) acc[y] = 0.0f;
        for (int t = wave * each; t < t1; t += AHEAD) {
            vec8 vp[AHEAD], vq[AHEAD][FJ];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (t + u < t1) {
                    const long long r = (long long)(t + u) * 32;
                    const Window wp(a.p.extent, i0 * a.p.ld + r, 8), wq(a.q.extent, j0 * a.q.ld + r, 8);
                    __builtin_memcpy(&vp[u], (const char*)(a.p.data + wp.base) + wp.at(row_p * (unsigned)a.p.ld + g * 8) * (unsigned)sizeof(T), sizeof(vec8));
#pragma unroll
                    for (int y = 0; y < FJ; ++y)
                        __builtin_memcpy(&vq[u][y], (const char*)(a.q.data + wq.base) + wq.at(row_q[y] * (unsigned)a.q.ld + g * 8) * (unsigned)sizeof(T), sizeof(vec8));
                }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (t + u < t1) {
                    const long long r = (long long)(t + u) * 32;
                    if (r + 32 > a.nr) {        // the sum ends here: elements into their places, zeros behind them
                        const Window wp(a.p.extent, i0 * a.p.ld + r, 8), wq(a.q.extent, j0 * a.q.ld + r, 8);
                        const int left = (int)(a.nr - r) - g * 8;
                        const int by = wp.moved(row_p * (unsigned)a.p.ld + g * 8);
                        if (by > 0 && by < 8) shift_down<8>(vp[u], by);
#pragma unroll
                        for (int e = 0; e < 8; ++e) vp[u][e] = e < left ? vp[u][e] : (T)0.0f;
#pragma unroll
                        for (int y = 0; y < FJ; ++y) {
                            const int byq = wq.moved(row_q[y] * (unsigned)a.q.ld + g * 8);
                            if (byq > 0 && byq < 8) shift_down<8>(vq[u][y], byq);
#pragma unroll
                            for (int e = 0; e < 8; ++e) vq[u][y][e] = e < left ? vq[u][y][e] : (T)0.0f;
                        }
                    }
                    if constexpr (decltype(plain)::value) {
#pragma unroll 1
                        for (int from = 0; from < 64; from += 16)
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                float p[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) p[e] = __shfl((float)vp[u][k], from + g * 4 + e);
#pragma unroll
                                for (int y = 0; y < FJ; ++y) {
                                    const float q = __shfl((float)vq[u][y][k], from + l);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) acc[y][e] = fmaf(p[e], q, acc[y][e]);
                                }
                            }
                    } else {
                        Frag<T> p;
                        p.set(vp[u]);
#pragma unroll
                        for (int y = 0; y < FJ; ++y) {
                            Frag<T> q;
                            q.set(vq[u][y]);
                            acc[y] = multiply<T>(acc[y], p, q);
                        }
                    }
                }
        }
#pragma unroll
        for (int y = 0; y < FJ; ++y) *(f32x4*)&part[wave][y * 16 + l][g * 4] = acc[y];
        __syncthreads();
    };
    const auto total = [&](int jt) {
        float f = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) f += part[w][jt][threadIdx.x & 15];
        return f;
    };
    share(std::false_type());
    constexpr int MINE = (FJ + 1) / 2;      // a thread's results, 32 rows apart
    float f[MINE];
    bool bad = false;
#pragma unroll
    for (int c = 0; c < MINE; ++c) {
        f[c] = (int)(threadIdx.x >> 4) + c * 32 < 16 * FJ ? total((threadIdx.x >> 4) + c * 32) : 0.0f;
        bad |= !(fabsf(f[c]) < INFINITY);
    }
    if (Frag<T>::N == 3 && __syncthreads_or(bad)) {      // an infinity times a piece of zero
        share(std::true_type());
#pragma unroll
        for (int c = 0; c < MINE; ++c)
            if (!(fabsf(f[c]) < INFINITY)) f[c] = total((threadIdx.x >> 4) + c * 32);
    }
    const long long i = i0 + (threadIdx.x & 15);
    if (i >= a.ni) return;
    const float bias[1] = {a.bias ? (float)a.bias[i] : 0.0f};
#pragma unroll
    for (int c = 0; c < MINE; ++c) {
        const int jt = (threadIdx.x >> 4) + c * 32;
        const long long j = j0 + jt;
        if (jt >= 16 * FJ || j >= a.nj) break;
        T res = (T)0.0f;
        if (a.residual) load_residual<T, 1>(a, i, j, 1u, res);
        const float one[1] = {f[c]};
        finish<T, EPI_FORWARD, 1>(a, 0, i, j, 1u, bias, res, one);
    }
}

template <typename T>
inline hipError_t launch_forward_skinny(const ProductArgs<T>& a, hipStream_t st) {
    const unsigned n = (unsigned)((a.ni + 15) / 16);
    if (a.nj <= 16) hipLaunchKernelGGL((forward_skinny<T, 1>), dim3(n), dim3(512), 0, st, a);
    else hipLaunchKernelGGL((forward_skinny<T, 4>), dim3(n, (unsigned)((a.nj + 63) / 64)), dim3(512), 0, st, a);
    return hipGetLastError();
}

}  // namespace mpe
