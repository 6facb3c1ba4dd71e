// The matrix products of a layer on the matrix cores: out[j][i] = sum_r P(i, r) Q(j, r), for
//   forward  y [m][n]:  i = n, j = m, r = k,   P = w,            Q = x
//   data     dx[m][k]:  i = k, j = m, r = n,   P = w transposed, Q = dz
//   weights  dw[n][k]:  i = k, j = n, r = m,   P = x transposed, Q = dz transposed
// i is the contiguous dimension of every output, so that P is the instruction's first operand: a lane then holds four
// consecutive elements of one output row.
//
// 16-bit types go into v_mfma_f32_16x16x32 as they are.  float32 has an instruction of its own, at 1/16 of that rate.
// Instead every float32 is written as the sum of three bfloat16 numbers h + m + l, each the rounded rest of what is
// before it (3 x 8 bits: the sum is exact, for numbers above 2^-109; of smaller ones what lies below bfloat16's smallest, up to
// 2^-134, is lost), and a product is summed from the six of the nine partial products that
// float32 can tell: hh + (hm + mh) + (hl + mm + lh).  What is left out is below 2^-25 of |x||w|, half of a float32
// rounding, and the partial sums are float32 as ever: this is float32 arithmetic at 6/16 of the cost.  Infinities split into
// inf - inf: where a tile's result is not finite its sums are made again in plain float32 (plain_tile).
//
// A workgroup of four waves computes a BI x BJ tile.  Global loads of the next step fly while the matrix instructions of
// this one run; the operands lie in LDS as rows of BK 16-bit pieces, in 16-byte chunks whose place is xored with the row,
// so that eight rows of one chunk column fall on different banks.  One LDS buffer and two barriers a step: two to four
// workgroups share a CU and fill each other's gaps (a second buffer, loads two or three steps ahead and steps of 64 for float32
// were all no faster).
//
// What bounds it.  float32, 65 536 x 1024 -> 1024: 699 us, 197 TFLOP/s of float32 where the library's own instruction reaches
// 154: six matrix instructions a product, and 5.5 vector instructions an element of a tile to split it.  Narrow layers,
// 196 608 x 64 -> 64 f32 tanh: memory, 100 MB in 28.0 us (3.6 TB/s), dx 150 MB in 35.5 (4.2), dw and db 150 MB in 30.5 and 7.4 for
// the sum of the splits; bf16 21, 30.5 and 31.5.  In between, 10 007 x 258 -> 255 f32: 25, 20 and 20 us, a chain of nine dependent steps
// on 2.5 workgroups a CU.  Of the 16-bit tiles those of two pieces and the weights' 128 x 128 keep some registers in memory.
#pragma once
#include "mpe_learn.hpp"

namespace mpe {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// 1 / (1 + e^-z); e^-z overflows to infinity and gives 0
__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-z)); }

// tanh: its series below 0.3 (the next term is 1.9e-9 of it), elsewhere 1 - 2 / (1 + e^2|z|), which loses bits only where
// they are far behind the point.
__device__ inline float tanh_of(float z) {
    const float q = z * z;
    float s = fmaf(q, -0.00886323552990219657f, 0.0218694885361552028f);
    s = fmaf(q, s, -0.0539682539682539683f);
    s = fmaf(q, s, 0.133333333333333333f);
    s = fmaf(q, s, -0.333333333333333333f);
    const float big = copysignf(fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + fast_exp(2.0f * fabsf(z))), 1.0f), z);
    return fabsf(z) < 0.3f ? fmaf(z * q, s, z) : big;
}

// Phi(z) and e^(-z^2/2).  erfc(x) e^(x^2) / 2 = t Q(t) with t = 1 / (1 + 0.33 x) and Q a polynomial fitted to it (relative error
// 1.4e-7 as far as float32 does not underflow, |z| = 13.5), so that the far tail keeps its relative precision: in float32, where the
// exponential is off by its argument's rounding, Phi is off by 1.9e-6 of it for |z| < 6 and by 7.3e-6 for |z| < 12.
struct Normal {
    float phi, e;
};
__device__ inline Normal normal_of(float z) {
    Normal n;
    n.e = fast_exp(-0.5f * z * z);
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.33f * 0.70710678118654752f, 1.0f));
    float q = fmaf(t, -0.0676722f, 0.230115935f);
    q = fmaf(t, q, -0.1755705f);
    q = fmaf(t, q, 0.204246135f);
    q = fmaf(t, q, 0.023612296f);
    q = fmaf(t, q, 0.100611365f);
    q = fmaf(t, q, 0.091478065f);
    q = fmaf(t, q, 0.0931789f);
    const float h = t * q * n.e;
    n.phi = z < 0.0f ? h : 1.0f - h;
    return n;
}

// tanh as exact as a 16-bit type can tell (2e-6 of it): the series' first two terms below 1/16, elsewhere 1 - 2 r with
// e = e^2z and r = 1 / (1 + e).  Its slope is 4 e r^2, which keeps its relative precision where 1 - tanh^2 has none left.
__device__ inline float tanh_16(float z, float& slope) {
    const float e = __builtin_amdgcn_exp2f(z * (2.0f * 1.44269504088896341f)), r = __builtin_amdgcn_rcpf(1.0f + e);
    slope = fminf(e, 0x1p127f) * r * (4.0f * r);        // not infinity times zero; of a NaN r is one
    return fabsf(z) < 0.0625f ? fmaf(z * z * z, -1.0f / 3.0f, z) : fmaf(-2.0f, r, 1.0f);
}
template <typename T>
__device__ inline float tanh_for(float z, float& slope) {
    if (sizeof(T) == 2) return tanh_16(z, slope);
    const float t = tanh_of(z);
    slope = fmaf(-t, t, 1.0f);
    return t;
}

__device__ inline float relu(float z) { return z > 0.0f || z != z ? z : 0.0f; }

constexpr int ACT_SLOPE = 16;       // what was kept are the slopes

__device__ inline float act_slope(int act, float z) {
    switch (act) {
        case MPE_ACT_TANH_OUT: return 1.0f - z * z;
        case MPE_ACT_TANH: { const float t = tanh_of(z); return 1.0f - t * t; }
        case MPE_ACT_RELU: return z > 0.0f ? 1.0f : z != z ? z : 0.0f;
        case MPE_ACT_GELU: { const Normal n = normal_of(z); return fmaf(z * 0.39894228040143268f, n.e, n.phi); }
        case MPE_ACT_SILU: { const float s = sigmoid(z); return s * (1.0f + z * (1.0f - s)); }
        case ACT_SLOPE: return z;
        default: return 1.0f;
    }
}

// The value, and the slope too: they share what is dear.  Four elements share the question which activation it is.
template <typename T, int N>
__device__ inline void act_both(int act, float* z, float* slope) {
    switch (act) {
        case MPE_ACT_TANH:
#pragma unroll
            for (int e = 0; e < N; ++e) {
                z[e] = tanh_for<T>(z[e], slope[e]);
            }
            break;
        case MPE_ACT_GELU:
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const Normal n = normal_of(z[e]);
                slope[e] = fmaf(z[e] * 0.39894228040143268f, n.e, n.phi);
                z[e] *= n.phi;
            }
            break;
        case MPE_ACT_SILU:
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float s = sigmoid(z[e]), v = z[e] * s;
                slope[e] = fmaf(v, 1.0f - s, s);
                z[e] = v;
            }
            break;
        default:
#pragma unroll
            for (int e = 0; e < N; ++e) {
                slope[e] = 1.0f;        // no activation; relu keeps a sign
            }
    }
}
template <typename T, int N>
__device__ inline void act_values(int act, float* z) {
    switch (act) {
        case MPE_ACT_NONE: break;
        case MPE_ACT_TANH:
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float slope;
                z[e] = tanh_for<T>(z[e], slope);
            }
            break;
        case MPE_ACT_RELU:
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] = relu(z[e]);
            break;
        case MPE_ACT_GELU:
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] *= normal_of(z[e]).phi;
            break;
        default:
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] *= sigmoid(z[e]);
    }
}

// What the forward pass keeps for the backward pass.  relu: anything with the pre-activation's sign, in the element type.
// bfloat16: the slope itself, times 2^14, in float16: its rounding is an eighth of the gradient's own, which makes the error 1/128
// larger, and with the factor float16 is as exact down to slopes of 4e-9.  float16's gradients are rounded no more coarsely than
// such slopes: a second rounding of that size would make their error 1.4 times as large, so it keeps the float32 pre-activation,
// as float32 does, or tanh's output where nothing was added to it.  Pre-activations in 16 bits would cost more than either.
constexpr float SLOPE_SCALE = 16384.0f;
template <typename T> struct Kept { static constexpr bool SLOPE = false; };
template <> struct Kept<bf16> { static constexpr bool SLOPE = true; };
template <typename T>
__device__ __host__ inline int kept_act(int act) { return Kept<T>::SLOPE && act != MPE_ACT_NONE && act != MPE_ACT_RELU ? ACT_SLOPE : act; }

// one kept value in the element type's size
template <typename T>
__device__ inline float kept_small(int act, T v) {
    return act == ACT_SLOPE ? (float)__builtin_bit_cast(f16, v) * (1.0f / SLOPE_SCALE) : (float)v;
}
template <> __device__ inline float kept_small<float>(int, float v) { return v; }

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

// Eight float32 numbers as three times eight bfloat16 ones, f = h + m + l.  In pairs, so that one instruction rounds two
// numbers and the pair's halves become float32 again by a shift and a mask.
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
template <typename F>
__device__ inline void split3(const F& f, bf16x8& h, bf16x8& m, bf16x8& l) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 p[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f32x2 rest = {f[2 * e], f[2 * e + 1]};
#pragma unroll
        for (int c = 0; c < 3; ++c) {
            p[c][e] = __builtin_bit_cast(unsigned, __builtin_convertvector(rest, bf16x2));
            if (c < 2) {
                rest[0] -= __builtin_bit_cast(float, p[c][e] << 16);
                rest[1] -= __builtin_bit_cast(float, p[c][e] & 0xffff0000u);
            }
        }
    }
    h = __builtin_bit_cast(bf16x8, p[0]);
    m = __builtin_bit_cast(bf16x8, p[1]);
    l = __builtin_bit_cast(bf16x8, p[2]);
}

// 16-bit dz enters a product as two pieces, value and rest: rounded to one it would add as much to the gradients' error again
// as their own rounding does.  The rests are summed apart, so that an infinity of the other operand, which times a rest of zero
// is NaN, spoils only what is then left out: the values alone tell what such a sum is.
// float16 reaches neither far enough up (a slope of 1.13 takes dy beyond 65504) nor down (a rest below 2^-24 would be lost, and with
// it the bits of every dz below 2^-13): the value is half of dz and the rest is kept 2^11 times as large.  Half of dz is no zero
// unless dz is one, so that it times an infinity is one.
template <typename T> struct Two { static constexpr float SCALE = 1.0f, REST = 1.0f; };
template <> struct Two<f16> { static constexpr float SCALE = 0.5f, REST = 2048.0f; };
template <typename T>
__device__ inline void split2(float f, T& h, T& rest) {
    // f as it is: the compiler folds the product that made it into its rounding to float16 (one rounding instead of two), but not
    // where it becomes a float again, and next to a tie the rest would belong to another h
    f *= Two<T>::SCALE;
    asm("" : "+v"(f));
    h = (T)f;
    if (Two<T>::SCALE != 1.0f && h == (T)0.0f && f != 0.0f) h = (T)copysignf(0x1p-24f, f);
    const float d = f - (float)h;
    rest = (T)(fabsf(d) < INFINITY ? d * Two<T>::REST : 0.0f);      // of an infinity or a NaN nothing is left
}
template <typename T>
__device__ inline float join2(float sum, float rests) {
    return (fabsf(rests) < INFINITY ? fmaf(rests, 1.0f / Two<T>::REST, sum) : sum) * (1.0f / Two<T>::SCALE);
}

// ---- operands ----
enum { R_INNER, O_INNER };      // which index is contiguous in memory: the summed one, or the output's
// what an operand is read from: its matrix; dy and what the forward pass kept (data * slope(pre)); or dz in two pieces, rows of
// the values and `rest` elements behind them of the rests
enum { SRC_PLAIN, SRC_DZ, SRC_SPLIT };

template <typename T>
struct Operand {
    const T* data;
    long long ld;               // may be 0 with SRC_DZ: one row for all
    long long extent;           // elements from the first to behind the last, at least 8 (SRC_SPLIT: to behind the values' last row)
    const void* pre;            // [rows][ld_pre], what the forward pass kept, or null: slope 1
    long long ld_pre, extent_pre;
    int act;
    long long rest;
};

__device__ inline bool small_pre(int act) { return act == MPE_ACT_RELU || act == ACT_SLOPE; }

template <typename T>
__device__ inline float pre_at(const Operand<T>& o, long long at) {
    return small_pre(o.act) ? kept_small<T>(o.act, ((const T*)o.pre)[at]) : ((const float*)o.pre)[at];
}

// Where a tile's vectors of W elements lie: a uniform base, and offsets from it that fit 32 bits (the host sees to it that
// a tile's rows lie within 4 GB).  A vector that would reach beyond the matrix is moved back to end with it.
struct Window {
    long long base;
    unsigned skip, last;
    __device__ inline Window(long long extent, long long first, int w) {
        base = min(first, extent - w);
        skip = (unsigned)(first - base);
        last = (unsigned)min(extent - w - base, (long long)0x7fffffff);
    }
    __device__ inline unsigned at(unsigned off) const { return min(skip + off, last); }
    __device__ inline int moved(unsigned off) const { return (int)(skip + off - at(off)); }     // by how many elements
};

// v[e] = v[e + by] for 0 <= by < N; what comes in at the end is of no interest
template <int N, typename V>
__device__ inline void shift_down(V& v, int by) {
#pragma unroll
    for (int s = N / 2; s > 0; s /= 2)
        if (by & s)
#pragma unroll
            for (int e = 0; e + s < N; ++e) v[e] = v[e + s];
}

// Loads a BO x BK tile of an operand into registers and writes it to LDS in pieces.  A thread's unit is one 16-byte chunk:
// eight consecutive r of one o.  R_INNER reads a unit as one run; O_INNER reads U neighbouring o at eight r and turns them
// by naming registers differently.  Loads ask nothing: they take whatever lies in the vector's place.  Only in the steps
// that reach the end of the sum or of the matrix does a Window keep them inside it, and fix() puts the elements into their
// places and zeros where the sum has ended; rows and columns of the output that do not exist may hold anything.
template <typename T, int BO, int LAYOUT, int SRC>
struct Loader {
    typedef Piece<T> P;
    static constexpr bool DZ = SRC == SRC_DZ, SPLIT = SRC == SRC_SPLIT;
    typedef typename P::type PT;
    typedef PT pt8 __attribute__((ext_vector_type(8)));
    static constexpr int BK = P::BK, CH = BK / 8, UNITS = BO * CH;
    static constexpr int U = UNITS >= 256 ? UNITS / 256 : 1;
    static constexpr bool SOME = UNITS < 256;       // only the first UNITS threads have one
    static constexpr int PLANE = BO * BK * 2;       // bytes of one piece's tile
    static constexpr int PIECES = P::N == 1 && SRC != SRC_PLAIN ? 2 : P::N;
    static_assert(!SPLIT || P::N == 1, "float32 dz is one number");
    static constexpr int NV = LAYOUT == R_INNER ? U : 8, W = LAYOUT == R_INNER ? 8 : U;      // vectors and their width

    typedef T vec __attribute__((ext_vector_type(W)));      // two 16-bit elements a register
    typedef float zvec __attribute__((ext_vector_type(W)));
    vec v[NV], rest[SPLIT ? NV : 1];
    zvec z[DZ ? NV : 1];

    // What stays the same from step to step: the vectors' offsets within the tile and, uniform, the place of the next step
    // and how many steps lie wholly inside the matrix (their loads are plain and need no fix()).
    unsigned off[LAYOUT == R_INNER ? U : 1], off_pre[DZ ? (LAYOUT == R_INNER ? U : 1) : 1];
    const char *next, *next_pre;
    long long row_bytes, row_bytes_pre;
    int inside;

    static __device__ inline int row_of(int u) { return LAYOUT == R_INNER ? (threadIdx.x + u * 256) / CH : ((int)threadIdx.x % (BO / U)) * U + u; }
    static __device__ inline int chunk_of(int u) { return LAYOUT == R_INNER ? (threadIdx.x + u * 256) % CH : (int)threadIdx.x / (BO / U); }
    // offset of vector i within the tile
    static __device__ inline unsigned offset(int i, unsigned ld, int left_o) {
        return LAYOUT == R_INNER ? (unsigned)min(row_of(i), left_o - 1) * ld + chunk_of(i) * 8 : (unsigned)(chunk_of(0) * 8 + i) * ld + row_of(0);
    }
    static __device__ inline long long first(long long o0, long long r0, long long ld) { return LAYOUT == R_INNER ? o0 * ld + r0 : r0 * ld + o0; }
    static __device__ inline unsigned pre_size(const Operand<T>& op) { return small_pre(op.act) ? (unsigned)sizeof(T) : 4u; }

    // steps from r0 on, of `steps`, whose vectors all end inside the matrix
    static __device__ inline int steps_inside(long long extent, long long ld, long long o0, long long r0, int steps) {
        const long long room = extent - first(o0, r0, ld) - (LAYOUT == R_INNER ? (long long)(BO - 1) * ld + BK : (long long)(BK - 1) * ld + BO);
        const long long stride = LAYOUT == R_INNER ? (long long)BK : BK * ld;
        if (room < 0) return 0;
        return stride == 0 ? steps : (int)min((long long)steps, room / stride + 1);
    }

    __device__ inline void init(const Operand<T>& op, long long o0, long long no, long long r0, long long r1) {
        const int left_o = (int)min(no - o0, (long long)BO);
#pragma unroll
        for (int i = 0; i < (LAYOUT == R_INNER ? U : 1); ++i) {
            off[i] = offset(i, (unsigned)op.ld, left_o) * (unsigned)sizeof(T);
            if (DZ) off_pre[i] = op.pre ? offset(i, (unsigned)op.ld_pre, left_o) * pre_size(op) : 0u;
        }
        next = (const char*)(op.data + first(o0, r0, op.ld));
        row_bytes = op.ld * (long long)sizeof(T);
        row_bytes_pre = DZ && op.pre ? op.ld_pre * pre_size(op) : 0;
        inside = steps_inside(op.extent, op.ld, o0, r0, (int)((r1 - r0) / BK));      // the step in which the sum ends is not one of them
        if (DZ && op.pre) {
            next_pre = (const char*)op.pre + first(o0, r0, op.ld_pre) * pre_size(op);
            inside = min(inside, steps_inside(op.extent_pre, op.ld_pre, o0, r0, inside));
        }
    }

    __device__ inline void load(const Operand<T>& op, long long o0, long long no, long long r0, int step) {
        if (!SOME || (int)threadIdx.x < UNITS) {
            if (step < inside) {
                const char* p = next;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    __builtin_memcpy(&v[i], p + off[LAYOUT == R_INNER ? i : 0], W * sizeof(T));
                    if (SPLIT) __builtin_memcpy(&rest[i], p + op.rest * (long long)sizeof(T) + off[LAYOUT == R_INNER ? i : 0], W * sizeof(T));
                    if (LAYOUT == O_INNER) p += row_bytes;
                }
                if (DZ && op.pre) {
                    const char* q = next_pre;
                    if (small_pre(op.act)) {
#pragma unroll
                        for (int i = 0; i < NV; ++i) {
                            vec t;
                            __builtin_memcpy(&t, q + off_pre[LAYOUT == R_INNER ? i : 0], W * sizeof(T));
                            if (LAYOUT == O_INNER) q += row_bytes_pre;
#pragma unroll
                            for (int e = 0; e < W; ++e) z[i][e] = kept_small<T>(op.act, t[e]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < NV; ++i) {
                            __builtin_memcpy(&z[i], q + off_pre[LAYOUT == R_INNER ? i : 0], W * 4);
                            if (LAYOUT == O_INNER) q += row_bytes_pre;
                        }
                    }
                }
            } else {
                load_edge(op, o0, no, r0);
            }
        }
        next += LAYOUT == R_INNER ? (long long)(BK * sizeof(T)) : BK * row_bytes;
        if (DZ && op.pre) next_pre += LAYOUT == R_INNER ? (long long)(BK * pre_size(op)) : BK * row_bytes_pre;
    }

    __device__ inline void load_edge(const Operand<T>& op, long long o0, long long no, long long r0) {
        const int left_o = (int)min(no - o0, (long long)BO);
        const Window w(op.extent, first(o0, r0, op.ld), W);
        const char* base = (const char*)(op.data + w.base);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const unsigned at = w.at(offset(i, (unsigned)op.ld, left_o)) * (unsigned)sizeof(T);
            __builtin_memcpy(&v[i], base + at, W * sizeof(T));
            if (SPLIT) __builtin_memcpy(&rest[i], base + op.rest * (long long)sizeof(T) + at, W * sizeof(T));
        }
        if (DZ && op.pre) {
            const Window wp(op.extent_pre, first(o0, r0, op.ld_pre), W);
            if (small_pre(op.act)) {
                const char* bp = (const char*)((const T*)op.pre + wp.base);
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    vec t;
                    __builtin_memcpy(&t, bp + wp.at(offset(i, (unsigned)op.ld_pre, left_o)) * (unsigned)sizeof(T), W * sizeof(T));
#pragma unroll
                    for (int e = 0; e < W; ++e) z[i][e] = kept_small<T>(op.act, t[e]);
                }
            } else {
                const char* bp = (const char*)((const float*)op.pre + wp.base);
#pragma unroll
                for (int i = 0; i < NV; ++i) __builtin_memcpy(&z[i], bp + wp.at(offset(i, (unsigned)op.ld_pre, left_o)) * 4u, W * 4);
            }
        }
    }

    __device__ inline void fix(const Operand<T>& op, long long o0, long long no, long long r0, long long r1) {
        if (SOME && (int)threadIdx.x >= UNITS) return;
        const int left_o = (int)min(no - o0, (long long)BO), left_r = (int)min(r1 - r0, (long long)BK);
        const Window w(op.extent, first(o0, r0, op.ld), W);
        const Window wp(DZ && op.pre ? op.extent_pre : (long long)W, DZ && op.pre ? first(o0, r0, op.ld_pre) : 0, W);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int by = w.moved(offset(i, (unsigned)op.ld, left_o));
            if (by > 0 && by < W) {
                shift_down<W>(v[i], by);
                if (SPLIT) shift_down<W>(rest[i], by);
            }
            if (DZ && op.pre) {
                const int byp = wp.moved(offset(i, (unsigned)op.ld_pre, left_o));
                if (byp > 0 && byp < W) shift_down<W>(z[i], byp);
            }
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const bool in = (LAYOUT == R_INNER ? chunk_of(i) * 8 + e : chunk_of(0) * 8 + i) < left_r;
                v[i][e] = in ? v[i][e] : (T)0.0f;
                if (SPLIT) rest[i][e] = in ? rest[i][e] : (T)0.0f;
                if (DZ) z[i][e] = in ? z[i][e] : 0.0f;
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
            char* to = lds + place(row_of(u), chunk_of(u));
            pt8 h;
            if (P::N == 1 && !DZ && !sums) {
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = LAYOUT == R_INNER ? (PT)v[u][e] : (PT)v[e][u];
                *(pt8*)to = h;
                if (SPLIT) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[e] = LAYOUT == R_INNER ? (PT)rest[u][e] : (PT)rest[e][u];
                    *(pt8*)(to + PLANE) = h;
                }
                continue;
            }
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = LAYOUT == R_INNER ? (float)v[u][e] : (float)v[e][u];
            if (DZ && op.pre) {
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= act_slope(op.act, LAYOUT == R_INNER ? z[u][e] : z[e][u]);
            }
            if (sums) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sums[u] += f[e];
            }
            if constexpr (P::N == 3) {
                pt8 m, l;
                split3(f, h, m, l);
                *(pt8*)(to + PLANE) = m;
                *(pt8*)(to + 2 * PLANE) = l;
            } else if constexpr (PIECES == 2) {
                pt8 r;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    PT one, two;
                    split2<PT>(f[e], one, two);
                    h[e] = one;
                    r[e] = two;
                }
                *(pt8*)(to + PLANE) = r;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = (PT)f[e];
            }
            *(pt8*)to = h;
        }
    }
};

// one element's sum in plain float32
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
    float* partial;             // EPI_PARTIAL: [split], of [nj][ni] products and, with_sums, [nj] sums of Q over r
    long long partial_ld;       // floats a split
    int with_sums;
};

// N consecutive elements as one register value: arrays of 16-bit elements get copied in odd pieces
template <typename U, int N> struct Run { typedef U type __attribute__((ext_vector_type(N))); };
template <typename U> struct Run<U, 1> { typedef U type; };

template <typename T, int N>
__device__ inline void load_residual(const ProductArgs<T>& a, long long i, long long j, unsigned mask, typename Run<T, N>::type& res) {
    const T* from = a.residual + j * a.ldr + i;
    if (mask == (1u << N) - 1) __builtin_memcpy(&res, from, N * sizeof(T));
    else if constexpr (N > 1) {
#pragma unroll
        for (int e = 0; e < N; ++e) res[e] = mask >> e & 1 ? from[e] : (T)0.0f;
    }
}

template <typename U, int N, typename V>
__device__ inline void put(U* to, const V& v, unsigned mask) {
    if (mask == (1u << N) - 1) {
        typename Run<U, N>::type r;
        if constexpr (N > 1) {
#pragma unroll
            for (int e = 0; e < N; ++e) r[e] = v[e];
        } else r = v[0];
        __builtin_memcpy(to, &r, N * sizeof(U));
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (mask >> e & 1) to[e] = v[e];
    }
}

// Finishes N consecutive elements of row j: those whose bit is set in mask.
template <typename T, int EPI, int N, typename F>
__device__ inline void finish(const ProductArgs<T>& a, unsigned split, long long i, long long j, unsigned mask, const float* bias, const typename Run<T, N>::type& res, const F& sum) {
    float f[N];
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = sum[e];
    if (EPI == EPI_PARTIAL) {
        put<float, N>(a.partial + split * a.partial_ld + j * a.ni + i, f, mask);
        return;
    }
    T o[N];
    if (EPI == EPI_FORWARD) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] += bias[e];
        if (a.pre && Kept<T>::SLOPE && a.act != MPE_ACT_RELU) {
            float slope[N];
            f16 z[N];
            act_both<T, N>(a.act, f, slope);
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] = (f16)(slope[e] * SLOPE_SCALE);
            put<f16, N>((f16*)a.pre + j * a.ni + i, z, mask);
        } else {
            if (a.pre && a.act == MPE_ACT_RELU) {
#pragma unroll
                for (int e = 0; e < N; ++e) o[e] = (T)f[e];
                put<T, N>((T*)a.pre + j * a.ni + i, o, mask);
            } else if (a.pre) {
                put<float, N>((float*)a.pre + j * a.ni + i, f, mask);
            }
            act_values<T, N>(a.act, f);
        }
        if (a.residual) {
            if constexpr (N == 1) f[0] += (float)res;
            else
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] += (float)res[e];
        }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = (T)f[e];
    put<T, N>(a.out + j * a.ldo + i, o, mask);
}

// A thread's share of `rows` rows of results in LDS: N columns of every STEP-th row from jt on.  What the residual holds is
// asked for two rows ahead: the compiler may not do that, since y may be the residual itself.
template <typename T, int EPI, int N, int STEP, typename GET>
__device__ inline void finish_rows(const ProductArgs<T>& a, unsigned split, long long i, long long j0, int jt, int rows, unsigned mask, const float* bias, GET&& get) {
    constexpr int AHEAD = 2;
    typename Run<T, N>::type res[AHEAD];
    const bool with_residual = EPI == EPI_FORWARD && a.residual;
    const auto ask = [&](int from) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (from + u * STEP < rows) load_residual<T, N>(a, i, j0 + from + u * STEP, mask, res[u]);
    };
    if (with_residual) ask(jt);
#pragma unroll 1
    for (; jt < rows; jt += AHEAD * STEP) {
        typename Run<T, N>::type now[AHEAD];
        if (with_residual) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) now[u] = res[u];
            ask(jt + AHEAD * STEP);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (jt + u * STEP < rows) {
                __attribute__((aligned(16))) float f[N];
                get(jt + u * STEP, f);
                finish<T, EPI, N>(a, split, i, j0 + jt + u * STEP, mask, bias, now[u], f);
            }
    }
}

// Operands of fewer than eight elements, for which there is no vector to load: a thread an element of the output, whose sum
// then has fewer than eight terms (of an expanded dy: as many as there are rows).
template <typename T, int EPI, int PL, int QL, int SRC>
__global__ __launch_bounds__(256) void product_few(const ProductArgs<T> a, int splits) {
    constexpr bool DZ = SRC == SRC_DZ;
    const long long n = a.ni * a.nj * splits;
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
        const long long i = at % a.ni, j = at / a.ni % a.nj;
        const unsigned split = (unsigned)(at / (a.ni * a.nj));
        const long long r0 = split * a.r_split, r1 = EPI == EPI_PARTIAL ? min(r0 + a.r_split, a.nr) : a.nr;
        const float bias[1] = {EPI == EPI_FORWARD && a.bias ? (float)a.bias[i] : 0.0f};
        const float f[1] = {plain_sum<T, PL, QL, DZ>(a.p, a.q, i, j, r0, r1)};
        T res = (T)0.0f;
        if (EPI == EPI_FORWARD && a.residual) load_residual<T, 1>(a, i, j, 1u, res);
        finish<T, EPI, 1>(a, split, i, j, 1u, bias, res, f);
        if (EPI == EPI_PARTIAL && a.with_sums && i == 0) {
            float s = 0.0f;
            for (long long r = r0; r < r1; ++r) {
                float b = (float)a.q.data[r * a.q.ld + j];
                if (DZ && a.q.pre) b *= act_slope(a.q.act, pre_at(a.q, r * a.q.ld_pre + j));
                s += b;
            }
            a.partial[split * a.partial_ld + a.nj * a.ni + j] = s;
        }
    }
}

// Workgroups are dealt to the eight XCDs in turn; this gives every XCD a run of neighbouring tiles, which share operands in
// its L2.
__device__ inline unsigned xcd_run(unsigned b, unsigned n) {
    const unsigned q = n / 8, r = n % 8, x = b % 8;
    return x * q + (x < r ? x : r) + b / 8;
}

// A tile's sums in plain float32, in the place of those that are not finite.  A whole tile at a time, since a NaN or an infinity
// in a row of one operand reaches a row of results: 16 384 x 1024 -> 1024 takes 1.0 ms if all of x is NaN and 0.75 with one NaN row
// of weights, where finite numbers take 0.19 (one thread an element: 30 and 2.1).
template <typename T, int PL, int QL, bool DZ, int BI, int BJ, int FI, int FJ>
__device__ inline void plain_tile(const ProductArgs<T>& a, long long i0, long long j0, long long r0, long long r1, int wi, int wj, char* lds, f32x4 (&acc)[FI][FJ]) {
    constexpr int KS = 16, PP = BI + 4, PQ = BJ + 4;
    float* const tp = (float*)lds;
    float* const tq = tp + KS * PP;
    const int lane = threadIdx.x & 63;
    f32x4 sum[FI][FJ];
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) sum[x][y] = 0.0f;
#pragma unroll 1
    for (long long r = r0; r < r1; r += KS) {
        __syncthreads();
#pragma unroll 1
        for (int u = threadIdx.x; u < BI * KS; u += 256) {
            const int o = PL == R_INNER ? u / KS : u % BI, k = PL == R_INNER ? u % KS : u / BI;
            const long long i = min(i0 + o, a.ni - 1);
            tp[k * PP + o] = r + k < r1 ? (float)a.p.data[PL == R_INNER ? i * a.p.ld + r + k : (r + k) * a.p.ld + i] : 0.0f;
        }
#pragma unroll 1
        for (int u = threadIdx.x; u < BJ * KS; u += 256) {
            const int o = QL == R_INNER ? u / KS : u % BJ, k = QL == R_INNER ? u % KS : u / BJ;
            const long long j = min(j0 + o, a.nj - 1);
            float f = 0.0f;
            if (r + k < r1) {
                f = (float)a.q.data[QL == R_INNER ? j * a.q.ld + r + k : (r + k) * a.q.ld + j];
                if (DZ && a.q.pre) f *= act_slope(a.q.act, pre_at(a.q, QL == R_INNER ? j * a.q.ld_pre + r + k : (r + k) * a.q.ld_pre + j));
            }
            tq[k * PQ + o] = f;
        }
        __syncthreads();
#pragma unroll 1
        for (int k = 0; k < KS; ++k) {
            f32x4 p[FI];
#pragma unroll
            for (int x = 0; x < FI; ++x) p[x] = *(const f32x4*)&tp[k * PP + wi + x * 16 + (lane >> 4) * 4];
#pragma unroll
            for (int y = 0; y < FJ; ++y) {
                const float q = tq[k * PQ + wj + y * 16 + (lane & 15)];
#pragma unroll
                for (int x = 0; x < FI; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[x][y][e] = fmaf(p[x][e], q, sum[x][y][e]);
            }
        }
    }
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[x][y][e] = fabsf(acc[x][y][e]) < INFINITY ? acc[x][y][e] : sum[x][y][e];
    __syncthreads();
}

// Workgroups that a CU's registers are shared among.  Two 16-bit pieces have two sums: one workgroup fewer, where registers would
// be kept in memory otherwise.  Small forward tiles fit five by a few registers (196 608 x 14 -> 64 bf16 19.2 us against 20.5 with four).
constexpr int groups_a_cu(int pieces, int epi, int src, int tile) {
    const bool two = pieces == 1 && src != SRC_PLAIN;
    if (tile > 8192) return pieces == 1 && epi == EPI_PARTIAL ? 3 : 2;
    if (epi == EPI_FORWARD && tile == 4096) return 5;
    return tile > 4096 ? (two ? 2 : 3) : two ? 3 : 4;
}

template <typename T, int EPI, int PL, int QL, int SRC, int BI, int BJ, int WI, int WJ>
__global__ __launch_bounds__(256, groups_a_cu(Piece<T>::N, EPI, SRC, BI * BJ)) void product(const ProductArgs<T> a) {
    typedef Piece<T> P;
    typedef typename P::type PT;
    typedef PT pt8 __attribute__((ext_vector_type(8)));
    typedef Loader<T, BI, PL, SRC_PLAIN> LP;
    typedef Loader<T, BJ, QL, SRC> LQ;
    constexpr bool DZ = SRC == SRC_DZ;
    constexpr int NP = P::N, NQ = LQ::PIECES, BK = P::BK, FI = BI / WI / 16, FJ = BJ / WJ / 16;
    // the results pass through LDS too, ROWS rows at a time, so that they leave as whole rows from a loop of little code
    constexpr int HALVES = BI * BJ > 8192 ? 2 : 1, ROWS = BJ / HALVES, PITCH = BI + 4;
    constexpr int TILES = NP * LP::PLANE + NQ * LQ::PLANE, RESULTS = ROWS * PITCH * 4;
    __shared__ __attribute__((aligned(16))) char lds[TILES > RESULTS ? TILES : RESULTS];
    char* const lp = lds;
    char* const lq = lds + NP * LP::PLANE;

    const unsigned t = xcd_run(blockIdx.x, gridDim.x), split = t / a.tiles, tile = t % a.tiles;
    const long long i0 = (long long)(tile % a.ti) * BI, j0 = (long long)(tile / a.ti) * BJ;
    const long long r0 = (long long)split * a.r_split, r1 = EPI == EPI_PARTIAL ? min(r0 + a.r_split, a.nr) : a.nr;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wi = (wave % WI) * (BI / WI), wj = (wave / WI) * (BJ / WJ);

    f32x4 acc[FI][FJ], rests[NQ == 2 ? FI : 1][NQ == 2 ? FJ : 1];
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) {
            acc[x][y] = 0.0f;
            if constexpr (NQ == 2) rests[x][y] = 0.0f;
        }
    float sums[LQ::U];
#pragma unroll
    for (int u = 0; u < LQ::U; ++u) sums[u] = 0.0f;
    const bool want_sums = EPI == EPI_PARTIAL && a.with_sums && i0 == 0;

    LP gp;
    LQ gq;
    gp.init(a.p, i0, a.ni, r0, r1);
    gq.init(a.q, j0, a.nj, r0, r1);
    const int steps = (int)((r1 - r0 + BK - 1) / BK);
    gp.load(a.p, i0, a.ni, r0, 0);
    gq.load(a.q, j0, a.nj, r0, 0);
    for (int step = 0; step < steps; ++step) {
        if (step >= gp.inside) gp.fix(a.p, i0, a.ni, r0 + (long long)step * BK, r1);
        if (step >= gq.inside) gq.fix(a.q, j0, a.nj, r0 + (long long)step * BK, r1);
        gp.store(a.p, lp, nullptr);
        gq.store(a.q, lq, want_sums ? sums : nullptr);
        __syncthreads();
        if (step + 1 < steps) {
            gp.load(a.p, i0, a.ni, r0 + (long long)(step + 1) * BK, step + 1);
            gq.load(a.q, j0, a.nj, r0 + (long long)(step + 1) * BK, step + 1);
        }
        // float32's steps alternate between splitting and multiplying: who multiplies goes first (65536 x 1024 -> 1024: 749 -> 699 us)
        if (NP == 3) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            pt8 fp[FI][NP];
#pragma unroll
            for (int x = 0; x < FI; ++x)
#pragma unroll
                for (int c = 0; c < NP; ++c) fp[x][c] = *(const pt8*)(lp + c * LP::PLANE + LP::place(wi + x * 16 + (lane & 15), kk * 4 + (lane >> 4)));
            // a result comes back after several issue slots: four sums at least take turns
            constexpr int YB = FI >= 4 || FJ == 1 ? 1 : 2;
#pragma unroll
            for (int y = 0; y < FJ; y += YB) {
                pt8 fq[YB][NQ];
#pragma unroll
                for (int b = 0; b < YB; ++b)
#pragma unroll
                    for (int c = 0; c < NQ; ++c) fq[b][c] = *(const pt8*)(lq + c * LQ::PLANE + LQ::place(wj + (y + b) * 16 + (lane & 15), kk * 4 + (lane >> 4)));
                // float32's partial products, smallest first
                constexpr int PAIRS = NP == 3 ? 6 : 1;
                constexpr int PC[6] = {NP == 3 ? 2 : 0, 0, NP / 2, NP / 2, 0, 0}, QC[6] = {0, NP - 1, NP / 2, 0, NP / 2, 0};
#pragma unroll
                for (int c = 0; c < PAIRS; ++c)
#pragma unroll
                    for (int b = 0; b < YB; ++b)
#pragma unroll
                        for (int x = 0; x < FI; ++x) acc[x][y + b] = mfma(fp[x][PC[c]], fq[b][QC[c]], acc[x][y + b]);
                if constexpr (NQ == 2) {
#pragma unroll
                    for (int b = 0; b < YB; ++b)
#pragma unroll
                        for (int x = 0; x < FI; ++x) rests[x][y + b] = mfma(fp[x][0], fq[b][1], rests[x][y + b]);
                }
            }
        }
        if (NP == 3) __builtin_amdgcn_s_setprio(0);
        __syncthreads();
    }

    if constexpr (NP == 3) {        // an infinity times a piece of zero
        bool bad = false;
#pragma unroll
        for (int x = 0; x < FI; ++x)
#pragma unroll
            for (int y = 0; y < FJ; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e) bad |= !(fabsf(acc[x][y][e]) < INFINITY);
        static_assert(16 * (BI + BJ + 8) * 4 <= sizeof(lds), "plain_tile's operands");
        if (__syncthreads_or(bad)) plain_tile<T, PL, QL, DZ, BI, BJ>(a, i0, j0, r0, r1, wi, wj, lds, acc);
    }
    if constexpr (NQ == 2) {
#pragma unroll
        for (int x = 0; x < FI; ++x)
#pragma unroll
            for (int y = 0; y < FJ; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[x][y][e] = join2<T>(acc[x][y][e], rests[x][y][e]);
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
                a.partial[split * a.partial_ld + a.nj * a.ni + j0 + threadIdx.x] = tot;
            }
        }
    }

    const int it = threadIdx.x % (BI / 4) * 4;      // a thread's four columns, the same in every row it takes
    const long long i = i0 + it;
    const int have = (int)max(0LL, min(4LL, a.ni - i));
    const unsigned mask = (1u << have) - 1;
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = EPI == EPI_FORWARD && a.bias && e < have ? (float)a.bias[i + e] : 0.0f;
    float* const res = (float*)lds;
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
        __syncthreads();
        if (wj / ROWS == half) {
#pragma unroll
            for (int y = 0; y < FJ; ++y)
#pragma unroll
                for (int x = 0; x < FI; ++x) *(f32x4*)&res[(wj % ROWS + y * 16 + (lane & 15)) * PITCH + wi + x * 16 + (lane >> 4) * 4] = acc[x][y];
        }
        __syncthreads();
        const int rows = (int)min((long long)ROWS, a.nj - j0 - half * ROWS);
        if (have > 0)
            finish_rows<T, EPI, 4, 1024 / BI>(a, split, i, j0 + half * ROWS, threadIdx.x / (BI / 4), rows, mask, bias, [&](int jt, float* f) {
                *(f32x4*)f = *(const f32x4*)&res[jt * PITCH + it];
            });
    }
}

}  // namespace mpe
