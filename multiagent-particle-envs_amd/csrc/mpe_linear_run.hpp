// The launches of a layer's two passes for one element type (mpe_linear_<type>.hip instantiate it).
#pragma once
#include <algorithm>

#include "mpe_linear_skinny.hpp"
#include "mpe_linear_wide.hpp"

namespace mpe {

inline long long tiles_of(long long n, int b) { return (n + b - 1) / b; }

// workgroups of 256 threads that a grid dimension holds: their threads are counted in 32 bits
constexpr int MAX_GROUPS = 0xffffff;

// ---- dz = dy f'(pre) as an array of its own: in float32 [m][n], in 16-bit types two pieces (split2), [m][2][piece_row(n)], or
// one where that is exact ----
// whole vectors, so that no row starts between two
inline long long piece_row(long long n) { return (n + 7) / 8 * 8; }
template <typename T>
inline long long dz_elements(long long m, long long n) { return sizeof(T) == 2 ? m * piece_row(n) * 2 : m * n; }

// float32 (the one T), dense dy: eight elements a thread, whatever the rows' length
template <typename T>
__global__ __launch_bounds__(256) void slope_flat(long long total, const T* __restrict__ dy, const T* __restrict__ pre, int act, T* __restrict__ dz) {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    for (long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; at < total; at += (long long)gridDim.x * 2048) {
        if (at + 8 <= total) {
            vec8 d, z;
            __builtin_memcpy(&d, dy + at, sizeof(d));
            __builtin_memcpy(&z, pre + at, sizeof(z));
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] *= act_slope(act, z[e]);
            __builtin_memcpy(dz + at, &d, sizeof(d));
        } else {
            for (long long k = at; k < total; ++k) dz[k] = dy[k] * act_slope(act, pre[k]);
        }
    }
}

// any dy
template <typename T>
__global__ __launch_bounds__(256) void slope_pass(long long m, long long n, const T* __restrict__ dy, long long lddy, const T* __restrict__ pre, int act,
                                                  T* __restrict__ dz) {
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < m * n; at += (long long)gridDim.x * 256) {
        const long long j = at / n, i = at - j * n;
        dz[at] = dy[j * lddy + i] * act_slope(act, pre[at]);
    }
}

// The same for 16-bit types, with the column sums of dz before it is rounded (the bias's gradient would see every rounding where
// its terms cancel): a workgroup takes 8 WIDE columns (WIDE up to 32, by n) of `rows` rows and leaves sums[blockIdx.y][n], where
// sums are wanted.  Without pre (no activation) dz is dy and only the sums are made, and so without a place for dz.  65 536 x 1024
// bf16 gelu: 537 MB in 97 us, 5.5 TB/s (part of it stays in the Infinity Cache).
template <typename T, bool SPLIT, int WIDE>
__global__ __launch_bounds__(256) void slope_sums(long long m, long long n, const T* __restrict__ dy, long long lddy, const void* __restrict__ pre,
                                                  int act, T* __restrict__ dz, int rows, float* __restrict__ sums) {
    constexpr int E = 8, STEP = 256 / WIDE;
    __shared__ float part[STEP][WIDE][E + 1];
    const int c = threadIdx.x % WIDE, g = threadIdx.x / WIDE;
    const long long i = ((long long)blockIdx.x * WIDE + c) * E, row = (n + E - 1) / E * E, j1 = min((long long)(blockIdx.y + 1) * rows, m);
    float s[E] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (i + E <= n) {
#pragma unroll 4
        for (long long j = (long long)blockIdx.y * rows + g; j < j1; j += STEP) {
            T d[E];
            float f[E];
            __builtin_memcpy(d, dy + j * lddy + i, sizeof(d));
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = (float)d[e];
            if (pre) {
                float z[E];
                T rest[E];
                if (small_pre(act)) {
                    T t[E];
                    __builtin_memcpy(t, (const T*)pre + j * n + i, sizeof(t));
#pragma unroll
                    for (int e = 0; e < E; ++e) z[e] = kept_small<T>(act, t[e]);
                } else {
                    __builtin_memcpy(z, (const float*)pre + j * n + i, sizeof(z));
                }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    f[e] *= act_slope(act, z[e]);
                    if (SPLIT) split2(f[e], d[e], rest[e]);
                    else d[e] = (T)f[e];
                }
                if (dz && !SPLIT) {
                    __builtin_memcpy(dz + j * n + i, d, sizeof(d));
                } else if (dz) {
                    __builtin_memcpy(dz + j * row * 2 + i, d, sizeof(d));
                    __builtin_memcpy(dz + j * row * 2 + row + i, rest, sizeof(rest));
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] += f[e];
        }
    } else if (i < n) {         // the last columns
#pragma unroll 4
        for (long long j = (long long)blockIdx.y * rows + g; j < j1; j += STEP)
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (i + e < n) {
                    float f = (float)dy[j * lddy + i + e];
                    if (pre) {
                        const long long at = j * n + i + e;
                        f *= act_slope(act, small_pre(act) ? kept_small<T>(act, ((const T*)pre)[at]) : ((const float*)pre)[at]);
                        if (dz && !SPLIT) dz[at] = (T)f;
                        else if (dz) split2(f, dz[j * row * 2 + i + e], dz[j * row * 2 + row + i + e]);
                    }
                    s[e] += f;
                }
    }
    if (!sums) return;
#pragma unroll
    for (int e = 0; e < E; ++e) part[g][c][e] = s[e];
    __syncthreads();
    const int col = threadIdx.x;
    if (col < WIDE * E && (long long)blockIdx.x * (WIDE * E) + col < n) {
        float t = 0.0f;
        for (int k = 0; k < STEP; ++k) t += part[k][col / E][col % E];
        sums[blockIdx.y * n + (long long)blockIdx.x * (WIDE * E) + col] = t;
    }
}

// As many columns side by side as there are: 131 072 x 128 bf16 19.4 us (dw and db together 56; 67 with 32 wherever n is).
template <typename T, bool SPLIT, int WIDE = 32>
inline hipError_t launch_slope_sums(long long m, long long n, const T* dy, long long lddy, const void* pre, int act, T* dz, int rows, float* sums, hipStream_t st) {
    if constexpr (WIDE > 2) {
        if (n <= WIDE * 4) return launch_slope_sums<T, SPLIT, WIDE / 2>(m, n, dy, lddy, pre, act, dz, rows, sums, st);
    }
    hipLaunchKernelGGL((slope_sums<T, SPLIT, WIDE>), dim3((unsigned)tiles_of(n, WIDE * 8), (unsigned)tiles_of(m, rows)), dim3(256), 0, st, m, n, dy, lddy, pre, act, dz, rows, sums);
    return hipGetLastError();
}

// ---- the bias's gradient without the weights' ----
// Column sums of dz over a split's rows, in the order in which a tile of the weights' product takes them (a thread the r of one
// chunk of every step, then chunk after chunk): a gradient does not depend on which others are asked for.  65 536 x 1024 f32: 268 MB
// in 71 us from call to call, 3.8 TB/s; with one step in flight instead of four 282.
template <typename T>
__global__ __launch_bounds__(256) void column_sums(const Operand<T> q, long long n, long long m, long long r_split, float* __restrict__ partial) {
    constexpr int BK = Piece<T>::BK, CH = BK / 8, COLS = 256 / CH, AHEAD = 4;
    __shared__ float part[CH][COLS];
    const int c = threadIdx.x % COLS, g = threadIdx.x / COLS;
    const long long j = (long long)blockIdx.x * COLS + c, r0 = blockIdx.y * r_split, r1 = min(r0 + r_split, m);
    float s = 0.0f;
    if (j < n)
        for (long long r = r0 + g * 8; r < r1; r += AHEAD * BK) {
            float f[AHEAD][8], z[AHEAD][8];
            const auto row = [&](int u, int e) { return min(r + u * BK + e, r1 - 1); };
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)         // all are asked for before any is looked at
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f[u][e] = (float)q.data[row(u, e) * q.ld + j];
                    if (q.pre) z[u][e] = pre_at(q, row(u, e) * q.ld_pre + j);
                }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (q.pre) f[u][e] *= act_slope(q.act, z[u][e]);
                    s += r + u * BK + e < r1 ? f[u][e] : 0.0f;
                }
        }
    part[g][c] = s;
    __syncthreads();
    if (g == 0 && j < n) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < CH; ++k) t += part[k][c];
        partial[blockIdx.y * n + j] = t;
    }
}

// ---- sums of the splits: column c of [splits][ld], in the order of the splits within a group and then of the groups ----
// The first n columns go to out, the next ones to sums; either may be null.
template <typename T, int COLS, int GROUPS>
__global__ __launch_bounds__(COLS * GROUPS) void add_splits(const float* __restrict__ partial, int splits, long long ld, long long n, T* __restrict__ out,
                                                            T* __restrict__ sums) {
    __shared__ float part[COLS < 64 ? GROUPS * COLS / 64 : GROUPS][COLS];
    const int c = threadIdx.x % COLS, g = threadIdx.x / COLS;
    for (long long first = (long long)blockIdx.x * COLS; first < ld; first += (long long)gridDim.x * COLS) {
        const long long at = first + c;
        const bool here = at < ld && (at < n ? out : sums) != nullptr;
        float s = 0.0f;
        if (here) {
            int k = g;
            for (; k + 3 * GROUPS < splits; k += 4 * GROUPS) {
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = partial[(k + u * GROUPS) * ld + at];
#pragma unroll
                for (int u = 0; u < 4; ++u) s += v[u];
            }
            for (; k < splits; k += GROUPS) s += partial[k * ld + at];
        }
        // groups that share a wave first
        constexpr int SHARE = COLS < 64 ? 64 / COLS : 1;
#pragma unroll
        for (int o = COLS; o < 64; o *= 2) s += __shfl_xor(s, o);
        __syncthreads();
        if (g % SHARE == 0) part[g / SHARE][c] = s;
        __syncthreads();
        if (g == 0 && here) {
            s = 0.0f;
#pragma unroll
            for (int k = 0; k < GROUPS / SHARE; ++k) s += part[k][c];
            if (at < n) out[at] = (T)s;
            else sums[at - n] = (T)s;
        }
    }
}

// Few columns and many splits take 64 threads a column, many columns have threads enough with 4.  `together`: the columns by
// which that is settled, for sums that have to come out as if they stood beside others.
template <typename T>
inline hipError_t launch_add_splits(const float* partial, int splits, long long ld, long long n, T* out, T* sums, long long together, hipStream_t st) {
    if (together >= 65536) hipLaunchKernelGGL((add_splits<T, 64, 4>), dim3((unsigned)std::min(tiles_of(ld, 64), (long long)MAX_GROUPS)), dim3(256), 0, st, partial, splits, ld, n, out, sums);
    else hipLaunchKernelGGL((add_splits<T, 16, 64>), dim3((unsigned)tiles_of(ld, 16)), dim3(1024), 0, st, partial, splits, ld, n, out, sums);
    return hipGetLastError();
}

template <typename T, int EPI, int PL, int QL, int SRC, int BI, int BJ, int WI, int WJ>
inline hipError_t launch_product(ProductArgs<T> a, int splits, hipStream_t st) {
    const long long ti = tiles_of(a.ni, BI), tiles = ti * tiles_of(a.nj, BJ);
    if (tiles * splits > MAX_GROUPS) return hipErrorInvalidValue;       // the callers' limits on sizes keep it from happening
    if constexpr (SRC != SRC_SPLIT) {       // own_dz: the other operand has more than 64 elements
        if (a.p.extent < 8 || a.q.extent < 8 || (a.q.pre && a.q.extent_pre < 8)) {
            const long long want = (a.ni * a.nj * splits + 255) / 256;
            hipLaunchKernelGGL((product_few<T, EPI, PL, QL, SRC>), dim3((unsigned)(want < 8192 ? want : 8192)), dim3(256), 0, st, a, splits);
            return hipGetLastError();
        }
    }
    a.ti = (int)ti;
    a.tiles = (unsigned)tiles;
    hipLaunchKernelGGL((product<T, EPI, PL, QL, SRC, BI, BJ, WI, WJ>), dim3((unsigned)(tiles * splits)), dim3(256), 0, st, a);
    return hipGetLastError();
}

// Tiles of the products that write rows of m.  16-bit types that fill every CU with a wide tile: product_wide (65 536 x 1024 ->
// 1024 bf16 155 us against 199 forward; dz in two pieces and dx 350 against 467, 16 384 x 512 -> 256, 256 tiles, 44 against 46; with
// 128 wide tiles a forward pass takes 21 us both ways, with 64 it is 20 against 13).  Others by the output's width.  Up to 64
// columns: 64 x 64 (196 608 x 64 -> 64 f32 28 us forward and 35.5 for dx, against 30.4 and 36.5 with 64 x 128).
template <typename T, int EPI, int PL, int QL, int SRC>
inline hipError_t launch_rows(const ProductArgs<T>& a, hipStream_t st) {
    if constexpr (sizeof(T) == 2 && SRC != SRC_DZ) {
        constexpr bool SPLIT = SRC == SRC_SPLIT;
        if (a.nr >= 64 && tiles_of(a.ni, Wide::BI) * tiles_of(a.nj, SPLIT ? Wide::BJ / 2 : Wide::BJ) >= 256 && a.ni > 64 && wide_operand(a.p, PL, a.ni) &&
            wide_operand(a.q, QL, a.nj))
            return launch_product_wide<T, EPI, PL, QL, SPLIT>(a, 1, st);
    }
    if constexpr (SRC != SRC_SPLIT) {       // own_dz: with SRC_SPLIT there are more than 64 columns, with SRC_DZ at most
        if (a.ni <= 16) return launch_product<T, EPI, PL, QL, SRC, 16, 128, 1, 4>(a, 1, st);
    }
    if (a.ni <= 64 || tiles_of(a.ni, 128) * tiles_of(a.nj, 128) < 256) return launch_product<T, EPI, PL, QL, SRC, 64, 64, 2, 2>(a, 1, st);
    if constexpr (SRC != SRC_DZ) return launch_product<T, EPI, PL, QL, SRC, 128, SRC == SRC_SPLIT ? 64 : 128, 2, 2>(a, 1, st);
    return hipErrorInvalidValue;
}

// Weight gradients: the sum over m is long and the output small, so it is split over workgroups that leave float32 partial
// sums.  One rule for the launch and the workspace.
struct WeightPlan {
    bool wide;              // product_wide, the column sums by slope_sums
    int bi, bj, splits;
    long long r_split;
};
// two: 16-bit dz in two pieces, split: from an array
inline WeightPlan weight_plan(int bk, bool wide, bool two, bool split, long long m, long long n, long long k) {
    WeightPlan p;
    p.wide = wide;
    if (wide) {
        const long long tiles = tiles_of(k, Wide::BI) * tiles_of(n, split ? Wide::BJ / 2 : Wide::BJ);
        long long s = 512 / tiles;        // two workgroups a CU
        if (s > tiles_of(m, 512)) s = tiles_of(m, 512);
        if (s < 1) s = 1;
        p.r_split = tiles_of(tiles_of(m, s), Wide::BK) * Wide::BK;
        p.splits = (int)tiles_of(m, p.r_split);
        return p;
    }
    p.bi = k <= 16 ? 16 : n <= 16 || k <= 64 || n <= 64 ? 64 : 128;
    p.bj = p.bi == 128 ? (split ? 64 : 128) : p.bi == 64 && n <= 16 ? 16 : 64;
    const long long tiles = tiles_of(k, p.bi) * tiles_of(n, p.bj);
    // four workgroups a CU (64/64 f32 over 196 608 rows, product and sum of the splits: 38.6 us at 1024 workgroups, 41.2 at
    // 768, 46.0 at 512); of two pieces as many as there is room for (64/64 bf16 over 524 288 rows 77 at 768, 100 at 1024)
    long long s = (two ? 256 * groups_a_cu(1, EPI_PARTIAL, split ? SRC_SPLIT : SRC_DZ, p.bi * p.bj) : 1024) / tiles;
    const long long most = tiles_of(m, 4 * bk);      // at least four steps each
    if (s > most) s = most;
    if (s < 1) s = 1;
    p.r_split = tiles_of(tiles_of(m, s), bk) * bk;
    p.splits = (int)tiles_of(m, p.r_split);
    return p;
}

// Large weight gradients of 16-bit types, if the operands' addresses allow it too (wide_operand): 65 536 x 1024 -> 1024 bf16
// with the bias's 145 us against 233, dz in two pieces and dw 335 against 488; 4096 x 256 -> 256 takes 39 both ways, below the tiles
// that split more finely are as fast or faster.
inline bool wide_weights(int size, long long m, long long n, long long k) {
    return size == 2 && k >= 256 && n >= 128 && k % 8 == 0 && n % 8 == 0 && m >= 4096;
}
// Rows a workgroup of slope_sums takes: 128, or 32 where that would be less than four workgroups a CU (65 536 x 256 -> 256 bf16 relu,
// all gradients: 66 us, 79 with 128; 65 536 x 512 -> 512 silu 213 and 206); more where there would be more than 32768 strips (a
// grid's second dimension ends at 65535).
inline int strip_rows(long long m, long long n) {
    const long long rows = tiles_of(m, 128) * tiles_of(n, 256) < 1024 ? 32 : 128;
    return (int)std::max(rows, tiles_of(tiles_of(m, 32768), 8) * 8);
}

// Wide inputs: dz becomes an array of its own, where it would otherwise be worked out in every tile of k of both products
// (131 072 x 128 -> 128 gelu, both gradients: bf16 75 us against 116, f32 140 against 177; at the border, x 64 -> 64, about even: bf16 57
// with an array and 54 without, f32 61 and 63; over 524 288 rows 139 and 154, 196 and 209).
inline bool own_dz(int act, long long k) { return act != MPE_ACT_NONE && k > 64; }

inline long long round_up(long long n) { return (n + 255) / 256 * 256; }

template <typename T>
struct LinearRun {
    // dz as an array of its own in 16-bit types: its column sums are taken while it is made
    static bool own_sums(int act, long long k) { return sizeof(T) == 2 && own_dz(act, k); }
    // relu's is dy or zero, which one number of the type holds
    static bool split_dz(int act, long long k) { return own_sums(act, k) && act != MPE_ACT_RELU; }
    static bool two_pieces(int act, long long k) { return split_dz(act, k) || (sizeof(T) == 2 && act != MPE_ACT_NONE && !own_dz(act, k)); }

    static long long backward_workspace(int act, long long m, long long n, long long k) {
        if (m == 0) return 0;
        const WeightPlan p = weight_plan(Piece<T>::BK, false, two_pieces(act, k), split_dz(act, k), m, n, k);
        const long long strips = tiles_of(m, strip_rows(m, n)) * n;
        long long sums = p.splits * n * k + (own_sums(act, k) ? strips : p.splits * n);
        if (wide_weights(sizeof(T), m, n, k)) sums = std::max(sums, weight_plan(Piece<T>::BK, true, two_pieces(act, k), split_dz(act, k), m, n, k).splits * n * k + strips);
        return (own_dz(act, k) ? round_up(dz_elements<T>(m, n) * (long long)sizeof(T)) : 0) + sums * 4;
    }

    static hipError_t forward(const LinearArgs& a, hipStream_t st) {
        ProductArgs<T> g = {};
        g.p = {(const T*)a.w, a.ldw, (a.n - 1) * a.ldw + a.k, nullptr, 0, 0, 0, 0};
        g.q = {(const T*)a.x, a.ldx, (a.m - 1) * a.ldx + a.k, nullptr, 0, 0, 0, 0};
        g.ni = a.n; g.nj = a.m; g.nr = a.k;
        g.out = (T*)a.y; g.ldo = a.ldy;
        g.bias = (const T*)a.bias; g.residual = (const T*)a.residual; g.ldr = a.ldr; g.pre = a.act != MPE_ACT_NONE ? a.pre : nullptr; g.act = a.act;
        // Up to two small workgroups a CU: their waves share the sum, where a tile's steps would follow one another (4 x 1024
        // -> 4096 bf16: 3.9 us against 14.1 in tiles; 2048 x 64 -> 64 f32 3.7 against 7.0; with 512 workgroups 1024 x 258 ->
        // 512 f32 10.4 against 13.6, 512 x 1024 -> 1024 bf16 12.6 against 11.4; with 1024 of them 10.9 against 7.6).
        if ((a.m <= 16 || tiles_of(a.m, 64) * tiles_of(a.n, 16) <= 512) && g.p.extent >= 8 && g.q.extent >= 8) return launch_forward_skinny<T>(g, st);
        return launch_rows<T, EPI_FORWARD, R_INNER, R_INNER, SRC_PLAIN>(g, st);
    }

    template <int SRC>
    static hipError_t weights(const ProductArgs<T>& g, const WeightPlan& p, hipStream_t st) {
        if constexpr (SRC != SRC_DZ) {      // own_dz: with SRC_DZ k is at most 64
            if (p.bi == 128) return launch_product<T, EPI_PARTIAL, O_INNER, O_INNER, SRC, 128, SRC == SRC_SPLIT ? 64 : 128, 2, 2>(g, p.splits, st);
        }
        if constexpr (SRC != SRC_SPLIT) {   // and with SRC_SPLIT above
            if (p.bi == 16) return launch_product<T, EPI_PARTIAL, O_INNER, O_INNER, SRC, 16, 64, 1, 4>(g, p.splits, st);
        }
        if (p.bj == 16) return launch_product<T, EPI_PARTIAL, O_INNER, O_INNER, SRC, 64, 16, 4, 1>(g, p.splits, st);
        return launch_product<T, EPI_PARTIAL, O_INNER, O_INNER, SRC, 64, 64, 2, 2>(g, p.splits, st);
    }

    static hipError_t backward(const LinearArgs& a, hipStream_t st) {
        hipError_t e = hipSuccess;
        if (a.m == 0) {         // no rows: the gradients are empty sums
            return launch_add_splits<T>(nullptr, 0, a.n * a.k + a.n, a.n * a.k, (T*)a.dw, (T*)a.db, a.n * a.k + a.n, st);
        }
        const int act = kept_act<T>(a.act);
        Operand<T> dz = {(const T*)a.dy, a.lddy, (a.m - 1) * a.lddy + a.n, a.act != MPE_ACT_NONE ? a.pre : nullptr, a.n, a.m * a.n, act, 0};
        const Operand<T> x = {(const T*)a.x, a.ldx, (a.m - 1) * a.ldx + a.k, nullptr, 0, 0, 0, 0};
        const bool own = own_dz(a.act, a.k), split = split_dz(a.act, a.k);
        const bool wide = wide_weights(sizeof(T), a.m, a.n, a.k) && wide_operand(x, O_INNER, a.k) && (own || wide_operand(dz, O_INNER, a.n));
        char* const ws = (char*)a.ws;
        float* const partial = (float*)(ws + (own ? round_up(dz_elements<T>(a.m, a.n) * (long long)sizeof(T)) : 0));
        const WeightPlan p = weight_plan(Piece<T>::BK, wide, two_pieces(a.act, a.k), split, a.m, a.n, a.k);
        const int strip = strip_rows(a.m, a.n), strips = (int)tiles_of(a.m, strip);
        const bool products = a.dx || a.dw;
        const bool own_16 = own_sums(a.act, a.k);
        float* const sums = a.db && (wide || own_16) ? partial + p.splits * a.n * a.k : nullptr;
        if (sums || (own_16 && products)) {
            if constexpr (sizeof(T) == 2) {
                T* const to = products ? (T*)ws : nullptr;
                if (split) e = launch_slope_sums<T, true>(a.m, a.n, (const T*)a.dy, a.lddy, a.pre, act, to, strip, sums, st);
                else e = launch_slope_sums<T, false>(a.m, a.n, (const T*)a.dy, a.lddy, own ? (const void*)a.pre : nullptr, act, to, strip, sums, st);
            }
        } else if (own && products) {
            if constexpr (sizeof(T) == 4) {
                const bool dense = a.lddy == a.n;
                const long long want = dense ? (a.m * a.n + 2047) / 2048 : (a.m * a.n + 255) / 256;
                const dim3 grid((unsigned)(want < 8192 ? want : 8192));
                if (dense) hipLaunchKernelGGL((slope_flat<float>), grid, dim3(256), 0, st, a.m * a.n, (const float*)a.dy, (const float*)a.pre, act, (float*)ws);
                else hipLaunchKernelGGL((slope_pass<float>), grid, dim3(256), 0, st, a.m, a.n, (const float*)a.dy, a.lddy, (const float*)a.pre, act, (float*)ws);
                e = hipGetLastError();
            }
        }
        if (e != hipSuccess) return e;
        const long long row = piece_row(a.n);
        if (split && products) dz = {(const T*)ws, row * 2, a.m * row * 2 - row, nullptr, 0, 0, MPE_ACT_NONE, row};
        else if (own && products) dz = {(const T*)ws, a.n, a.m * a.n, nullptr, 0, 0, MPE_ACT_NONE, 0};
        if (a.dx) {
            ProductArgs<T> g = {};
            g.p = {(const T*)a.w, a.ldw, (a.n - 1) * a.ldw + a.k, nullptr, 0, 0, 0, 0};
            g.q = dz;
            g.ni = a.k; g.nj = a.m; g.nr = a.n;
            g.out = (T*)a.dx; g.ldo = a.lddx;
            if constexpr (sizeof(T) == 2) {
                if (split) e = launch_rows<T, EPI_STORE, O_INNER, R_INNER, SRC_SPLIT>(g, st);
            }
            if (!split) e = dz.pre ? launch_rows<T, EPI_STORE, O_INNER, R_INNER, SRC_DZ>(g, st) : launch_rows<T, EPI_STORE, O_INNER, R_INNER, SRC_PLAIN>(g, st);
            if (e != hipSuccess) return e;
        }
        const bool few = x.extent < 8 || dz.extent < 8 || (dz.pre && dz.extent_pre < 8);       // product_few sums in an order of its own
        if (a.db && !sums && !a.dw && !few) {
            constexpr int COLS = 256 / (Piece<T>::BK / 8);
            hipLaunchKernelGGL((column_sums<T>), dim3((unsigned)tiles_of(a.n, COLS), (unsigned)p.splits), dim3(256), 0, st, dz, a.n, a.m, p.r_split, partial);
            e = hipGetLastError();
            if (e == hipSuccess) e = launch_add_splits<T>(partial, p.splits, a.n, 0, nullptr, (T*)a.db, a.n * a.k + a.n, st);
        } else if (a.dw || (a.db && !sums)) {
            ProductArgs<T> g = {};
            g.p = x;
            g.q = dz;
            g.ni = a.k; g.nj = a.n; g.nr = a.m; g.r_split = p.r_split;
            g.partial = partial;
            g.partial_ld = a.n * a.k + (sums ? 0 : a.n);
            g.with_sums = a.db && !sums;
            if constexpr (sizeof(T) == 2) {
                if (wide) e = split ? launch_product_wide<T, EPI_PARTIAL, O_INNER, O_INNER, true>(g, p.splits, st)
                                    : launch_product_wide<T, EPI_PARTIAL, O_INNER, O_INNER, false>(g, p.splits, st);
                else if (split) e = weights<SRC_SPLIT>(g, p, st);
            }
            if (!wide && !split) e = dz.pre ? weights<SRC_DZ>(g, p, st) : weights<SRC_PLAIN>(g, p, st);
            if (e == hipSuccess) e = launch_add_splits<T>(partial, p.splits, g.partial_ld, a.n * a.k, (T*)a.dw, sums ? nullptr : (T*)a.db, g.partial_ld, st);
        }
        if (e == hipSuccess && sums) e = launch_add_splits<T>(sums, strips, a.n, 0, nullptr, (T*)a.db, a.n, st);
        return e;
    }
};

}  // namespace mpe
