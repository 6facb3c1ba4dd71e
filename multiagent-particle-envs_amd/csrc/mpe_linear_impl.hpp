// The matrix products of a layer on the matrix cores: out[j][i] = sum_r P(i, r) Q(j, r), for
//   forward  y [m][n]:  i = n, j = m, r = k,   P = w,            Q = x
//   data     dx[m][k]:  i = k, j = m, r = n,   P = w transposed, Q = dz
//   weights  dw[n][k]:  i = k, j = n, r = m,   P = x transposed, Q = dz transposed
// i is the contiguous dimension of every output, so that P is the instruction's first operand: a lane then holds four
// consecutive elements of one output row.
//
// 16-bit types go into v_mfma_f32_16x16x32 as they are.  float32 has an instruction of its own, at 1/16 of that rate.
// Instead every float32 is written as the sum of three bfloat16 numbers h + m + l, each the rounded rest of what is
// before it (3 x 8 bits: the sum is exact), and a product is summed from the six of the nine partial products that
// float32 can tell: hh + (hm + mh) + (hl + mm + lh).  What is left out is below 2^-25 of |x||w|, half of a float32
// rounding, and the partial sums are float32 as ever: this is float32 arithmetic at 6/16 of the cost.  Where a result
// is not finite (infinities split into inf - inf) the element is summed again in plain float32.
//
// A workgroup of four waves computes a BI x BJ tile.  Global loads of the next step fly while the matrix instructions of
// this one run; the operands lie in LDS as rows of BK 16-bit pieces, in 16-byte chunks whose place is xored with the row,
// so that eight rows of one chunk column fall on different banks.  One LDS buffer and two barriers a step: two to four
// workgroups share a CU and fill each other's gaps.
#pragma once
#include "mpe_learn.hpp"

namespace mpe {

typedef float f32x4 __attribute__((ext_vector_type(4)));

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
        case MPE_ACT_TANH_OUT: return 1.0f - z * z;
        case MPE_ACT_TANH: { const float t = tanhf(z); return 1.0f - t * t; }
        case MPE_ACT_RELU: return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
        case MPE_ACT_GELU: return 0.5f * erfcf(-0.70710678118654752f * z) + z * 0.39894228040143268f * expf(-0.5f * z * z);
        case MPE_ACT_SILU: { const float s = 1.0f / (1.0f + expf(-z)); return s * (1.0f + z * (1.0f - s)); }
        default: return 1.0f;
    }
}

// ---- pieces ----
template <typename T> struct Piece {                // 16-bit types: the element itself
    typedef T type;
    static constexpr int N = 1, BK = 64;
};
template <> struct Piece<float> {
    typedef bf16 type;
    static constexpr int N = 3, BK = 32;
};

__device__ inline f32x4 mfma(bf16 __attribute__((ext_vector_type(8))) a, bf16 __attribute__((ext_vector_type(8))) b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x4 mfma(f16 __attribute__((ext_vector_type(8))) a, f16 __attribute__((ext_vector_type(8))) b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// ---- operands ----
enum { R_INNER, O_INNER };      // which index is contiguous in memory: the summed one, or the output's

// an operand's matrix; with DZ, what is read is data * slope(pre)
template <typename T>
struct Operand {
    const T* data;
    long long ld;               // may be 0 with DZ: one row for all
    const void* pre;            // [rows][ld_pre], float (relu: T), or null: slope 1
    long long ld_pre;
    int act;
};

template <typename T>
__device__ inline float pre_at(const Operand<T>& o, long long at) {
    return o.act == MPE_ACT_RELU ? (float)((const T*)o.pre)[at] : ((const float*)o.pre)[at];
}

// Loads a BO x BK tile of an operand into registers and writes it to LDS in pieces.  A thread's unit is one 16-byte chunk:
// eight consecutive r of one o.  R_INNER reads a unit as one run; O_INNER reads U neighbouring o at eight r and turns them
// by naming registers differently.  Addresses are a uniform base plus 32-bit offsets that stay the same from step to step
// (the host sees to it that a tile's rows lie within 4 GB).  A step that lies inside the matrix takes wide loads; the
// last step of the sum and, with O_INNER, the last tile of o read element by element from clamped places and put 0
// where nothing is.
template <typename T, int BO, int LAYOUT, bool DZ>
struct Loader {
    typedef Piece<T> P;
    typedef typename P::type PT;
    typedef PT pt8 __attribute__((ext_vector_type(8)));
    static constexpr int BK = P::BK, CH = BK / 8, UNITS = BO * CH;
    static constexpr int U = UNITS >= 256 ? UNITS / 256 : 1;
    static constexpr bool SOME = UNITS < 256;       // only the first UNITS threads have one
    static constexpr int PLANE = BO * BK * 2;       // bytes of one piece's tile

    T v[U][8];
    float z[DZ ? U : 1][8];

    static __device__ inline int row_of(int u) { return LAYOUT == R_INNER ? (threadIdx.x + u * 256) / CH : ((int)threadIdx.x % (BO / U)) * U + u; }
    static __device__ inline int chunk_of(int u) { return LAYOUT == R_INNER ? (threadIdx.x + u * 256) % CH : (int)threadIdx.x / (BO / U); }

    // N consecutive values of the saved array from element `at` of the uniform base
    template <int N>
    static __device__ inline void load_pre(const Operand<T>& op, long long base, unsigned at, float* out) {
        if (op.act == MPE_ACT_RELU) {
            T t[N];
            __builtin_memcpy(t, (const char*)((const T*)op.pre + base) + at * (unsigned)sizeof(T), sizeof(t));
#pragma unroll
            for (int e = 0; e < N; ++e) out[e] = (float)t[e];
        } else {
            __builtin_memcpy(out, (const char*)((const float*)op.pre + base) + at * 4u, N * 4);
        }
    }

    // rows [o0, no) and the sum's [r0, r1) exist; what lies outside reads as 0
    __device__ inline void load(const Operand<T>& op, long long o0, long long no, long long r0, long long r1) {
        if (SOME && (int)threadIdx.x >= UNITS) return;
        const unsigned ld = (unsigned)op.ld, ldp = (unsigned)op.ld_pre;
        const int left_o = (int)min(no - o0, (long long)BO), left_r = (int)min(r1 - r0, (long long)BK);     // uniform
        const bool with_pre = DZ && op.pre;
        if (LAYOUT == R_INNER) {
            const T* base = op.data + o0 * op.ld + r0;
            const long long base_pre = o0 * op.ld_pre + r0;
            if (left_r == BK) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const unsigned o = min(row_of(u), left_o - 1), r = chunk_of(u) * 8;     // a row that is not there: the last one again, never stored
                    __builtin_memcpy(v[u], (const char*)base + (o * ld + r) * (unsigned)sizeof(T), 8 * sizeof(T));
                    if (with_pre) load_pre<8>(op, base_pre, o * ldp + r, z[u]);
                }
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const unsigned o = min(row_of(u), left_o - 1);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int r = chunk_of(u) * 8 + e, rc = min(r, left_r - 1);
                        const T x = *(const T*)((const char*)base + (o * ld + rc) * (unsigned)sizeof(T));
                        v[u][e] = r < left_r ? x : (T)0.0f;
                        if (with_pre) load_pre<1>(op, base_pre, o * ldp + rc, &z[u][e]);
                    }
                }
            }
        } else {
            const T* base = op.data + r0 * op.ld + o0;
            const long long base_pre = r0 * op.ld_pre + o0;
            const unsigned o = row_of(0), r = chunk_of(0) * 8;
            if (left_r == BK && left_o == BO) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    T t[U];
                    __builtin_memcpy(t, (const char*)(base + e * op.ld) + (r * ld + o) * (unsigned)sizeof(T), sizeof(t));
#pragma unroll
                    for (int u = 0; u < U; ++u) v[u][e] = t[u];
                    if (with_pre) {
                        float f[U];
                        load_pre<U>(op, base_pre + e * op.ld_pre, r * ldp + o, f);
#pragma unroll
                        for (int u = 0; u < U; ++u) z[u][e] = f[u];
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const unsigned rc = min((int)r + e, left_r - 1);
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const unsigned oc = min((int)o + u, left_o - 1);
                        const T x = *(const T*)((const char*)base + (rc * ld + oc) * (unsigned)sizeof(T));
                        v[u][e] = (int)r + e < left_r && (int)o + u < left_o ? x : (T)0.0f;
                        if (with_pre) load_pre<1>(op, base_pre, rc * ldp + oc, &z[u][e]);
                    }
                }
            }
        }
    }

    static __device__ inline int place(int row, int chunk) {
        const int sw = CH == 8 ? row & 7 : (row >> 1) & 3;
        return row * (BK * 2) + ((chunk ^ sw) << 4);
    }

    // sums: with O_INNER, gains the tile's sums over r of the thread's o
    __device__ inline void store(const Operand<T>& op, char* lds, float* sums) {
        if (SOME && (int)threadIdx.x >= UNITS) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)v[u][e];
            if (DZ && op.pre) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= act_slope(op.act, z[u][e]);
            }
            if (sums) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sums[u] += f[e];
            }
            char* to = lds + place(row_of(u), chunk_of(u));
            pt8 h;
            if (P::N == 3) {
                pt8 m, l;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    h[e] = (PT)f[e];
                    const float rest = f[e] - (float)h[e];
                    m[e] = (PT)rest;
                    l[e] = (PT)(rest - (float)m[e]);
                }
                *(pt8*)to = h;
                *(pt8*)(to + PLANE) = m;
                *(pt8*)(to + 2 * PLANE) = l;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = DZ ? (PT)f[e] : (PT)v[u][e];
                *(pt8*)to = h;
            }
        }
    }
};

// one element's sum in plain float32, for results that are not finite
template <typename T, int PL, int QL, bool DZ>
__device__ inline float plain_sum(const Operand<T>& p, const Operand<T>& q, long long i, long long j, long long r0, long long r1) {
    float s = 0.0f;
    for (long long r = r0; r < r1; ++r) {
        const float a = (float)p.data[PL == R_INNER ? i * p.ld + r : r * p.ld + i];
        float b = (float)q.data[QL == R_INNER ? j * q.ld + r : r * q.ld + j];
        if (DZ && q.pre) b *= act_slope(q.act, pre_at(q, QL == R_INNER ? j * q.ld_pre + r : r * q.ld_pre + j));
        s = fmaf(a, b, s);
    }
    return s;
}

enum { EPI_FORWARD, EPI_STORE, EPI_PARTIAL };

template <typename T>
struct ProductArgs {
    Operand<T> p, q;
    long long ni, nj, nr;       // sizes
    long long r_split;          // how much of the sum a split takes (a multiple of BK)
    int ti;                     // tiles along i
    unsigned tiles;             // tiles of the output; splits follow one another
    T* out;
    long long ldo;
    const T *bias, *residual;   // EPI_FORWARD
    long long ldr;
    void* pre;
    int act;
    float *partial, *partial_sum;   // EPI_PARTIAL: [split][nj][ni], and [split][nj] or null
};

// Finishes N consecutive elements of row j: those whose bit is set in mask.
template <typename U, int N>
__device__ inline void put(U* to, const U* v, unsigned mask) {
    if (mask == (1u << N) - 1) __builtin_memcpy(to, v, N * sizeof(U));
    else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (mask >> e & 1) to[e] = v[e];
    }
}

template <typename T, int EPI, int N, typename F>
__device__ inline void finish(const ProductArgs<T>& a, unsigned split, long long i, long long j, unsigned mask, const float* bias, const F& sum) {
    float f[N];
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = sum[e];
    if (EPI == EPI_PARTIAL) {
        put<float, N>(a.partial + ((long long)split * a.nj + j) * a.ni + i, f, mask);
        return;
    }
    T o[N];
    if (EPI == EPI_FORWARD) {
        T res[N];
        if (a.residual) {
            const T* from = a.residual + j * a.ldr + i;
            if (mask == (1u << N) - 1) __builtin_memcpy(res, from, sizeof(res));
            else {
#pragma unroll
                for (int e = 0; e < N; ++e) res[e] = mask >> e & 1 ? from[e] : (T)0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] += bias[e];
        if (a.pre) {
            if (a.act == MPE_ACT_RELU) {
#pragma unroll
                for (int e = 0; e < N; ++e) o[e] = (T)f[e];
                put<T, N>((T*)a.pre + j * a.ni + i, o, mask);
            } else {
                put<float, N>((float*)a.pre + j * a.ni + i, f, mask);
            }
        }
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = act_value(a.act, f[e]);
        if (a.residual) {
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] += (float)res[e];
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = (T)f[e];
    put<T, N>(a.out + j * a.ldo + i, o, mask);
}

// Workgroups are dealt to the eight XCDs in turn; this gives every XCD a run of neighbouring tiles, which share operands in
// its L2.
__device__ inline unsigned xcd_run(unsigned b, unsigned n) {
    const unsigned q = n / 8, r = n % 8, x = b % 8;
    return x * q + (x < r ? x : r) + b / 8;
}

template <typename T, int EPI, int PL, int QL, bool DZ, int BI, int BJ, int WI, int WJ>
__global__ __launch_bounds__(256) void product(const ProductArgs<T> a) {
    typedef Piece<T> P;
    typedef typename P::type PT;
    typedef PT pt8 __attribute__((ext_vector_type(8)));
    typedef Loader<T, BI, PL, false> LP;
    typedef Loader<T, BJ, QL, DZ> LQ;
    constexpr int NP = P::N, BK = P::BK, FI = BI / WI / 16, FJ = BJ / WJ / 16;
    __shared__ __attribute__((aligned(16))) char lds[NP * (LP::PLANE + LQ::PLANE)];
    char* const lp = lds;
    char* const lq = lds + NP * LP::PLANE;

    const unsigned t = xcd_run(blockIdx.x, gridDim.x), split = t / a.tiles, tile = t % a.tiles;
    const long long i0 = (long long)(tile % a.ti) * BI, j0 = (long long)(tile / a.ti) * BJ;
    const long long r0 = (long long)split * a.r_split, r1 = EPI == EPI_PARTIAL ? min(r0 + a.r_split, a.nr) : a.nr;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wi = (wave % WI) * (BI / WI), wj = (wave / WI) * (BJ / WJ);

    f32x4 acc[FI][FJ];
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) acc[x][y] = 0.0f;
    float sums[LQ::U];
#pragma unroll
    for (int u = 0; u < LQ::U; ++u) sums[u] = 0.0f;
    const bool want_sums = EPI == EPI_PARTIAL && a.partial_sum && i0 == 0;

    LP gp;
    LQ gq;
    gp.load(a.p, i0, a.ni, r0, r1);
    gq.load(a.q, j0, a.nj, r0, r1);
    for (long long r = r0; r < r1; r += BK) {
        gp.store(a.p, lp, nullptr);
        gq.store(a.q, lq, want_sums ? sums : nullptr);
        __syncthreads();
        if (r + BK < r1) {
            gp.load(a.p, i0, a.ni, r + BK, r1);
            gq.load(a.q, j0, a.nj, r + BK, r1);
        }
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            pt8 fp[FI][NP];
#pragma unroll
            for (int x = 0; x < FI; ++x)
#pragma unroll
                for (int c = 0; c < NP; ++c) fp[x][c] = *(const pt8*)(lp + c * LP::PLANE + LP::place(wi + x * 16 + (lane & 15), kk * 4 + (lane >> 4)));
#pragma unroll
            for (int y = 0; y < FJ; ++y) {
                pt8 fq[NP];
#pragma unroll
                for (int c = 0; c < NP; ++c) fq[c] = *(const pt8*)(lq + c * LQ::PLANE + LQ::place(wj + y * 16 + (lane & 15), kk * 4 + (lane >> 4)));
                if (NP == 3) {
                    // smallest first
#pragma unroll
                    for (int x = 0; x < FI; ++x) acc[x][y] = mfma(fp[x][NP - 1], fq[0], acc[x][y]);
#pragma unroll
                    for (int x = 0; x < FI; ++x) acc[x][y] = mfma(fp[x][0], fq[NP - 1], acc[x][y]);
#pragma unroll
                    for (int x = 0; x < FI; ++x) acc[x][y] = mfma(fp[x][NP / 2], fq[NP / 2], acc[x][y]);
#pragma unroll
                    for (int x = 0; x < FI; ++x) acc[x][y] = mfma(fp[x][NP / 2], fq[0], acc[x][y]);
#pragma unroll
                    for (int x = 0; x < FI; ++x) acc[x][y] = mfma(fp[x][0], fq[NP / 2], acc[x][y]);
                }
#pragma unroll
                for (int x = 0; x < FI; ++x) acc[x][y] = mfma(fp[x][0], fq[0], acc[x][y]);
            }
        }
        __syncthreads();
    }

    // column sums: the threads that hold the same columns add up through LDS, in the order of their rows
    if (EPI == EPI_PARTIAL) {
        if (want_sums) {        // the same for the whole workgroup
            float* s = (float*)lds;
            if (!LQ::SOME || (int)threadIdx.x < LQ::UNITS) {
#pragma unroll
                for (int u = 0; u < LQ::U; ++u) s[LQ::chunk_of(0) * BJ + LQ::row_of(u)] = sums[u];
            }
            __syncthreads();
            if ((int)threadIdx.x < BJ && j0 + threadIdx.x < a.nj) {
                float tot = 0.0f;
                for (int c = 0; c < LQ::CH; ++c) tot += s[c * BJ + threadIdx.x];
                a.partial_sum[split * a.nj + j0 + threadIdx.x] = tot;
            }
        }
    }

    // Results that are not finite are left out here, noted in LDS and summed again below.
    constexpr bool AGAIN = NP == 3;
    unsigned* const again = (unsigned*)lds;
    static_assert(!AGAIN || BI * BJ / 8 <= (int)sizeof(lds), "a bit for every element");
    bool bad = false;
    if (AGAIN) {
#pragma unroll
        for (int y = 0; y < FJ; ++y)
#pragma unroll
            for (int x = 0; x < FI; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) bad = bad || !(fabsf(acc[x][y][e]) < INFINITY);
        bad = __syncthreads_or(bad);
        if (bad) {
            for (int w = threadIdx.x; w < BI * BJ / 32; w += 256) again[w] = 0;
            __syncthreads();
        }
    }
#pragma unroll
    for (int x = 0; x < FI; ++x) {
        const int it = wi + x * 16 + (lane >> 4) * 4;
        const long long i = i0 + it;
        const int have = a.ni - i < 4 ? (int)(a.ni - i) : 4;
        if (have <= 0) continue;
        float bias[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = EPI == EPI_FORWARD && a.bias && e < have ? (float)a.bias[i + e] : 0.0f;
#pragma unroll
        for (int y = 0; y < FJ; ++y) {
            const int jt = wj + y * 16 + (lane & 15);
            const long long j = j0 + jt;
            if (j >= a.nj) continue;
            unsigned mask = (1u << have) - 1;       // of the four elements
            if (AGAIN && bad) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < have && !(fabsf(acc[x][y][e]) < INFINITY)) {
                        mask &= ~(1u << e);
                        atomicOr(&again[(jt * BI + it + e) >> 5], 1u << ((it + e) & 31));
                    }
            }
            finish<T, EPI, 4>(a, split, i, j, mask, bias, acc[x][y]);
        }
    }
    if (AGAIN && bad) {
        __syncthreads();
        for (int n = threadIdx.x; n < BI * BJ; n += 256) {
            if (!(again[n >> 5] >> (n & 31) & 1)) continue;
            const long long i = i0 + n % BI, j = j0 + n / BI;
            const float bias[1] = {EPI == EPI_FORWARD && a.bias ? (float)a.bias[i] : 0.0f};
            const float f[1] = {plain_sum<T, PL, QL, DZ>(a.p, a.q, i, j, r0, r1)};
            finish<T, EPI, 1>(a, split, i, j, 1u, bias, f);
        }
    }
}

}  // namespace mpe
