// Large products of 16-bit types.  Operands go from memory to LDS without passing registers (one instruction moves 64 x 16
// bytes), three stages deep: while a stage is multiplied the next has landed and the one after it is on its way.  A
// workgroup of four waves computes 128 x 256, each wave 64 x 128, which reads 12 KB of LDS for 32 matrix instructions;
// with 73 KB of LDS and half the registers two workgroups share a CU and one's results leave while the other multiplies.
//
// What bounds it (65 536 x 1024 -> 1024 bf16, 137 GFLOP): without activation 141 us, 0.97 PFLOP/s, where a large library product
// reaches 1.31.  Nothing is saturated: by the counters the matrix cores are busy for 26 % of the cycles of a forward pass with gelu,
// its slope and a residual (232 us), for 48 % of dx's with dz in two pieces (272 us for 275 GFLOP) and for 56 % of the weight
// gradient's (230 us, where LDS conflicts take a fifth of the cycles).  The rest are waits, and the ends of a tile, which only the
// CU's other workgroup covers: two stages of copies before its first product, activations and stores behind its last.
//
// An operand whose contiguous index is the output's lies in LDS as it lies in memory, and ds_read_b64_tr_b16 turns it: 16
// lanes read four rows of 16 elements and each gets one column.
#pragma once
#include <type_traits>

#include "mpe_linear_impl.hpp"

namespace mpe {

struct Wide {
    static constexpr int BI = 128, BJ = 256, BK = 32, STAGES = 3;
};

typedef __attribute__((address_space(3))) void lds_void;

// a pointer that is the same in all lanes, in scalar registers
__device__ inline const char* uniform(const char* p) {
    const unsigned long long a = (unsigned long long)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
    return (const char*)((unsigned long long)hi << 32 | lo);
}

// 16 bytes a lane from base + off (bytes) to LDS address `to`, lane after lane
__device__ inline void copy_to_lds(const char* base, unsigned off, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
}

// One operand's tile of BO x 32.  R_INNER: rows of 64 bytes, their four 16-byte chunks xored with the row, as Loader::place.
// O_INNER: 32 rows of BO elements, chunks xored with twice the row's last two bits, so that the four rows a transposed read
// touches lie on different banks.
// SPLIT: every 64 outputs stand twice, 64 rows (columns) of their values and 64 of their rests, so that a wave's 128 are both
// pieces of its 64 outputs and nothing else in the kernel has to know.
template <typename T, int BO, int LAYOUT, bool SPLIT = false>
struct WideTile {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    typedef short v4i16 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4i16 lds_v4;
    static constexpr int COPIES = BO / 64;      // instructions a wave and stage: 1 KB each
    static constexpr int BYTES = BO * 64;
    static constexpr int RUN = LAYOUT == R_INNER ? 4 : BO / 8;     // chunks a row of the tile
    static constexpr int OUTPUTS = SPLIT ? BO / 2 : BO;
    // the output that a row (column) of the tile belongs to, and whether it is its rest
    static __device__ inline int output_of(int at) { return SPLIT ? (at >> 7) * 64 + (at & 63) : at; }
    static __device__ inline unsigned piece_of(const Operand<T>& op, int at) { return SPLIT && at & 64 ? (unsigned)op.rest : 0u; }

    unsigned off[COPIES];       // bytes from the tile's first element
    const char* next;
    long long step;

    static __device__ inline int swizzle(int row, int chunk) { return LAYOUT == R_INNER ? chunk ^ ((row >> 1) & 3) : chunk ^ ((row & 3) << 1); }

    __device__ inline void init(const Operand<T>& op, long long o0, long long no, long long r0) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, left = (int)min(no - o0, (long long)OUTPUTS);
        const unsigned ld = (unsigned)op.ld;
#pragma unroll
        for (int u = 0; u < COPIES; ++u) {
            const int slot = (wave * COPIES + u) * 64 + lane, row = slot / RUN, chunk = swizzle(row, slot % RUN);
            // outputs that are not there read the last ones again and are never stored
            off[u] = (LAYOUT == R_INNER ? (unsigned)min(output_of(row), left - 1) * ld + chunk * 8 + piece_of(op, row)
                                        : (unsigned)row * ld + min(output_of(chunk * 8), left - 8) + piece_of(op, chunk * 8)) * 2u;
        }
        next = (const char*)(op.data + (LAYOUT == R_INNER ? o0 * op.ld + r0 : r0 * op.ld + o0));
        step = LAYOUT == R_INNER ? 64 : 64 * op.ld;
    }

    __device__ inline void copy(unsigned lds, int wave) {
#pragma unroll
        for (int u = 0; u < COPIES; ++u) copy_to_lds(next, off[u], lds + (wave * COPIES + u) * 1024);
        next += step;
    }

    // The end of the sum, `left` < 32 of it.  What lies wholly behind it is replaced by what is there anyway; the chunk the
    // end lies in is copied whole, but in the matrix's last row (or a row repeated with stride 0), behind which there is nothing: there it starts back() elements
    // earlier, an even number, because addresses are multiples of four bytes.  mend_end() then puts the elements into their
    // places, with the one that an odd number leaves out, and zeros behind the end; a lane mends the chunks it has copied.
    static __device__ inline int back(int left) { return (8 - left % 8) % 8 + (left & 1); }
    // rows of pieces hold whole chunks
    static __device__ inline bool nothing_behind(const Operand<T>& op, long long row, long long no) { return !SPLIT && (row == no - 1 || op.ld == 0); }

    __device__ inline void copy_end(unsigned lds, int wave, const Operand<T>& op, long long o0, long long no, int left) {
        const int lane = threadIdx.x & 63, left_o = (int)min(no - o0, (long long)OUTPUTS), before = LAYOUT == R_INNER ? 8 : 0;
        const unsigned ld = (unsigned)op.ld;
        const char* const base = uniform(next - before * 2);
#pragma unroll
        for (int u = 0; u < COPIES; ++u) {
            const int slot = (wave * COPIES + u) * 64 + lane, row = slot / RUN, chunk = swizzle(row, slot % RUN);
            unsigned at;
            if (LAYOUT == R_INNER) {
                const int r = min(output_of(row), left_o - 1), c = chunk * 8 < left ? chunk * 8 : 0;
                at = (unsigned)r * ld + piece_of(op, row) + (unsigned)(c + before - (nothing_behind(op, o0 + r, no) && c + 8 > left ? back(left) : 0));
            } else {
                at = (unsigned)min(row, left - 1) * ld + (unsigned)min(output_of(chunk * 8), left_o - 8) + piece_of(op, chunk * 8);
            }
            copy_to_lds(base, at * 2u, lds + (wave * COPIES + u) * 1024);
        }
    }

    static __device__ inline void mend_end(char* lds, int wave, const Operand<T>& op, long long o0, long long no, long long nr, int left) {
        const int lane = threadIdx.x & 63, left_o = (int)min(no - o0, (long long)OUTPUTS);
#pragma unroll
        for (int u = 0; u < COPIES; ++u) {
            const int slot = (wave * COPIES + u) * 64 + lane, row = slot / RUN, chunk = swizzle(row, slot % RUN);
            if (LAYOUT == R_INNER ? chunk * 8 + 8 <= left : row < left) continue;
            vec8 v = (T)0.0f;
            if (LAYOUT == R_INNER && chunk * 8 < left) {
                v = *(const vec8*)(lds + slot * 16);
                if (nothing_behind(op, o0 + min(output_of(row), left_o - 1), no)) {
                    if (back(left) < 8) shift_down<8>(v, back(left));
                    if (left & 1) {
                        const T last = op.data[(no - 1) * op.ld + nr - 1];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = chunk * 8 + e == left - 1 ? last : v[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = chunk * 8 + e < left ? v[e] : (T)0.0f;
            }
            *(vec8*)(lds + slot * 16) = v;
        }
    }

    // the instruction's operand for the outputs o .. o + 15
    static __device__ inline vec8 read(const char* lds, int o) {
        const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
        if (LAYOUT == R_INNER) {
            const int row = o + l;
            return *(const vec8*)(lds + row * 64 + swizzle(row, g) * 16);
        }
        struct { v4i16 lo, hi; } v;
        const int at = (l / 4 + g * 8) * (BO * 2) + swizzle(l / 4, o / 8 + (l & 3) / 2) * 16 + (l & 1) * 8;
        v.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)(lds + at));
        v.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4*)(lds + at + 4 * (BO * 2)));
        return __builtin_bit_cast(vec8, v);
    }
};

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// A wave's 64 x 16 FJ sums, four consecutive columns from i0 + x 16 + 4 (lane / 16) on of row j0 + y 16 + lane % 16 in acc[x][y],
// become results in LDS, rows of `pitch` bytes from to on, and in kept[x][y] what is kept, if that has the results' size (if it
// is float32 it is stored at once).  The activation is a template parameter, since a switch would stand 32 times in the
// unrolled code.
template <typename T, int ACT, bool KEPT, int FJ>
__device__ __forceinline__ void seal(const ProductArgs<T>& a, const f32x4 (&acc)[4][8], u32x2 (&kept)[4][FJ], long long i0, long long j0, char* to, int pitch) {
    typedef typename Run<T, 4>::type vec4;
    typedef f16 half4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, jl = lane & 15, left_j = (int)min(a.nj - j0, 16LL * FJ);
    // what is read is kept inside its row and the matrix; results that are not there get whatever it holds
    const auto four = [&](const T* row, long long i) __attribute__((always_inline)) {
        vec4 v;
        const long long at = min(i, a.ni - 4);
        __builtin_memcpy(&v, row + at, 8);
        if (at < i) shift_down<4>(v, (int)min(i - at, 3LL));
        return v;
    };
    const long long i0l = i0 + (lane >> 4) * 4;
    // everything is asked for at once; the four blocks of a row after one another, since they share lines
    vec4 res[4][FJ];
    if (a.residual) {
#pragma unroll
        for (int y = 0; y < FJ; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) res[x][y] = four(a.residual + min(j0 + y * 16 + jl, a.nj - 1) * a.ldr, i0l + x * 16);
    }
    float bias[4][4] = {};
    if (a.bias) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const vec4 b = four(a.bias, i0l + x * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[x][e] = (float)b[e];
        }
    }
#pragma unroll
    for (int y = 0; y < FJ; ++y) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const long long i = i0l + x * 16;
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = acc[x][y][e] + bias[x][e];
            if (KEPT && Kept<T>::SLOPE && ACT != MPE_ACT_RELU) {
                float slope[4];
                act_both<T, 4>(ACT, f, slope);
                half4 z;
#pragma unroll
                for (int e = 0; e < 4; ++e) z[e] = (f16)(slope[e] * SLOPE_SCALE);
                kept[x][y] = __builtin_bit_cast(u32x2, z);
            } else {
                if (KEPT && ACT == MPE_ACT_RELU) {
                    vec4 z;
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = (T)f[e];
                    kept[x][y] = __builtin_bit_cast(u32x2, z);
                } else if (KEPT && y * 16 + jl < left_j) {
                    put<float, 4>((float*)a.pre + (j0 + y * 16 + jl) * a.ni + i, f, (1u << (int)max(0LL, min(4LL, a.ni - i))) - 1);
                }
                act_values<T, 4>(ACT, f);
            }
            if (a.residual) {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[e] += (float)res[x][y][e];
            }
            vec4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (T)f[e];
            __builtin_memcpy(to + (y * 16 + jl) * pitch + (x * 16 + (lane >> 4) * 4) * 2, &o, 8);
            if (KEPT && (Kept<T>::SLOPE || ACT == MPE_ACT_RELU)) asm volatile("" : "+v"(kept[x][y]));      // two words from here on, not four halves
            __builtin_amdgcn_sched_barrier(0);      // else the scheduler starts on all blocks at once and runs out of registers
        }
    }
}

// SPLIT: Q is dz in two pieces.  The tile is 128 x 128 then, and the second half of a wave's sums are those of the rests.
template <typename T, int EPI, int PL, int QL, bool SPLIT>
__global__ __launch_bounds__(256, 2) void product_wide(const ProductArgs<T> a) {
    typedef WideTile<T, Wide::BI, PL> TP;
    typedef WideTile<T, Wide::BJ, QL, SPLIT> TQ;
    typedef T vec8 __attribute__((ext_vector_type(8)));
    constexpr int BI = Wide::BI, BJ = TQ::OUTPUTS, BK = Wide::BK, FI = 4, FJ = 8, STAGE = TP::BYTES + TQ::BYTES;
    constexpr int ROWS = 128, HALVES = BJ / ROWS, PITCH = BI + 4;
    static_assert(ROWS * PITCH * 4 <= Wide::STAGES * STAGE, "the results pass through the stages' memory");
    __shared__ __attribute__((aligned(16))) char lds[Wide::STAGES * STAGE];

    const unsigned t = xcd_run(blockIdx.x, gridDim.x), split = t / a.tiles, tile = t % a.tiles;
    const long long i0 = (long long)(tile % a.ti) * BI, j0 = (long long)(tile / a.ti) * BJ;
    const long long r0 = (long long)split * a.r_split, r1 = EPI == EPI_PARTIAL ? min(r0 + a.r_split, a.nr) : a.nr;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned base = (unsigned)(uintptr_t)(lds_void*)lds;
    const int wi = (wave & 1) * 64, half = wave >> 1;

    f32x4 acc[FI][FJ];
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
        for (int y = 0; y < FJ; ++y) acc[x][y] = 0.0f;
    const auto multiply = [&](const char* stage) {
        vec8 fp[FI];
#pragma unroll
        for (int x = 0; x < FI; ++x) fp[x] = TP::read(stage, wi + x * 16);
#pragma unroll
        for (int y = 0; y < FJ; ++y) {
            const vec8 fq = TQ::read(stage + TP::BYTES, half * 128 + y * 16);
#pragma unroll
            for (int x = 0; x < FI; ++x) acc[x][y] = mfma(fp[x], fq, acc[x][y]);
        }
    };

    TP p;
    TQ q;
    p.init(a.p, i0, a.ni, r0);
    q.init(a.q, j0, a.nj, r0);
    const int whole = (int)((r1 - r0) / BK), left = (int)((r1 - r0) % BK), steps = whole + (left ? 1 : 0);
    const auto copy = [&](unsigned to) __attribute__((always_inline)) {
        p.copy(to, wave);
        q.copy(to + TP::BYTES, wave);
    };
    const auto copy_end = [&](unsigned to) __attribute__((always_inline)) {
        p.copy_end(to, wave, a.p, i0, a.ni, left);
        q.copy_end(to + TP::BYTES, wave, a.q, j0, a.nj, left);
    };
    for (int s = 0; s < 2 && s < steps; ++s) {
        if (s < whole) copy(base + s * STAGE);
        else copy_end(base + s * STAGE);
    }
    // Stage s has landed when at most the copies of stage s + 1 are under way, and a wave is done with stage s - 1 when its reads
    // have returned: the compiler leaves the last of them, and the products that want them, for after the barrier, so the wait
    // for them stands with it.  The barrier makes both true of every wave, and stage s + 2 goes where stage s - 1 was.  The loop
    // that runs long asks nothing and knows its stages.
    int s = 0, stage = 0;
    for (; s + 4 < whole; s += 3) {
#pragma unroll
        for (int u = 0; u < 3; ++u) {
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(TP::COPIES + TQ::COPIES) : "memory");
            copy(base + (u + 2) % 3 * STAGE);
            multiply(lds + u * STAGE);
        }
    }
    for (; s < steps; ++s) {
        if (s + 1 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(TP::COPIES + TQ::COPIES) : "memory");
        else if (!left) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            TP::mend_end(lds + stage * STAGE, wave, a.p, i0, a.ni, r1, left);
            TQ::mend_end(lds + stage * STAGE + TP::BYTES, wave, a.q, j0, a.nj, r1, left);
            __syncthreads();
        }
        const unsigned to = base + (stage == 0 ? 2 : stage - 1) * STAGE;
        if (s + 2 < whole) copy(to);
        else if (s + 2 < steps) copy_end(to);
        multiply(lds + stage * STAGE);
        stage = stage == 2 ? 0 : stage + 1;
    }

    constexpr int OJ = SPLIT ? FJ / 2 : FJ;
    const int wj = half * (16 * OJ);
    if constexpr (SPLIT) {
#pragma unroll
        for (int x = 0; x < FI; ++x)
#pragma unroll
            for (int y = 0; y < OJ; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[x][y][e] = join2<T>(acc[x][y][e], acc[x][y + OJ][e]);
    }

    if constexpr (EPI != EPI_PARTIAL) {
        // Results become what is stored while they are in registers, pass through LDS and leave as whole rows.
        constexpr int PITCH = BI * 2 + 16;
        static_assert(BJ * PITCH <= Wide::STAGES * STAGE, "the results pass through the stages' memory");
        const int it = threadIdx.x % (BI / 8) * 8;
        const int have = (int)max(0LL, min(8LL, a.ni - i0 - it)), rows = (int)min((long long)BJ, a.nj - j0);
        const auto leave = [&](T* to, long long ld) __attribute__((always_inline)) {
            T* const column = to + j0 * ld + i0 + it;
            __syncthreads();
            if (have > 0)
#pragma unroll 4
                for (int jt = threadIdx.x / (BI / 8); jt < rows; jt += 256 / (BI / 8))
                    put<T, 8>(column + jt * ld, *(const vec8*)(lds + jt * PITCH + it * 2), (1u << have) - 1);
        };
        // one path an activation, to the end: where paths meet again the compiler holds the tile twice
        const auto finish_as = [&](auto act, auto keep) __attribute__((always_inline)) {
            constexpr bool SMALL = decltype(keep)::value && (Kept<T>::SLOPE || decltype(act)::value == MPE_ACT_RELU);
            u32x2 kept[FI][OJ];
            char* const mine = lds + wj * PITCH + wi * 2;
            __syncthreads();
            seal<T, decltype(act)::value, decltype(keep)::value, OJ>(a, acc, kept, i0 + wi, j0 + wj, mine, PITCH);
            leave(a.out, a.ldo);
            if constexpr (SMALL) {
                __syncthreads();
#pragma unroll
                for (int y = 0; y < OJ; ++y)
#pragma unroll
                    for (int x = 0; x < FI; ++x) *(u32x2*)(mine + (y * 16 + (lane & 15)) * PITCH + (x * 16 + (lane >> 4) * 4) * 2) = kept[x][y];
                leave((T*)a.pre, a.ni);
            }
        };
        const auto with = [&](auto act) __attribute__((always_inline)) {
            if (a.pre) finish_as(act, std::true_type());
            else finish_as(act, std::false_type());
        };
        if constexpr (EPI == EPI_STORE) return finish_as(std::integral_constant<int, MPE_ACT_NONE>(), std::false_type());
        switch (a.act) {
            case MPE_ACT_NONE: return finish_as(std::integral_constant<int, MPE_ACT_NONE>(), std::false_type());
            case MPE_ACT_TANH: return with(std::integral_constant<int, MPE_ACT_TANH>());
            case MPE_ACT_RELU: return with(std::integral_constant<int, MPE_ACT_RELU>());
            case MPE_ACT_GELU: return with(std::integral_constant<int, MPE_ACT_GELU>());
            default: return with(std::integral_constant<int, MPE_ACT_SILU>());
        }
    }
    // partial sums are float32 and pass 128 rows at a time
    constexpr int N = 4;                                // a thread's columns
    const int it = threadIdx.x % (BI / N) * N;          // a thread's columns, the same in every row it takes
    const long long i = i0 + it;
    const int have = (int)max(0LL, min((long long)N, a.ni - i));
    const unsigned mask = (1u << have) - 1;
    const float bias[N] = {};
    float* const res = (float*)lds;
#pragma unroll
    for (int turn = 0; turn < HALVES; ++turn) {
        __syncthreads();
        if (wj / ROWS == turn) {
#pragma unroll
            for (int y = 0; y < OJ; ++y)
#pragma unroll
                for (int x = 0; x < FI; ++x) *(f32x4*)&res[(wj % ROWS + y * 16 + (lane & 15)) * PITCH + wi + x * 16 + (lane >> 4) * 4] = acc[x][y];
        }
        __syncthreads();
        const int rows = (int)max(0LL, min((long long)ROWS, a.nj - j0 - turn * ROWS));
        if (have > 0)
            finish_rows<T, EPI, N, 256 * N / BI>(a, split, i, j0 + turn * ROWS, threadIdx.x / (BI / N), rows, mask, bias, [&](int jt, float* f) {
#pragma unroll
                for (int e = 0; e < N; e += 4) *(f32x4*)&f[e] = *(const f32x4*)&res[jt * PITCH + it + e];
            });
    }
}

// What the copies need: four-byte addresses, whole chunks of columns where the columns are the outputs, and outputs enough
// for the device's CUs.
template <typename T>
inline bool wide_operand(const Operand<T>& o, int layout, long long outputs) {
    return !o.pre && o.ld % 2 == 0 && (uintptr_t)o.data % 4 == 0 && (layout == R_INNER || outputs % 8 == 0);
}

template <typename T, int EPI, int PL, int QL, bool SPLIT>
inline hipError_t launch_product_wide(ProductArgs<T> a, int splits, hipStream_t st) {
    const long long bj = SPLIT ? Wide::BJ / 2 : Wide::BJ, ti = (a.ni + Wide::BI - 1) / Wide::BI, tiles = ti * ((a.nj + bj - 1) / bj);
    a.ti = (int)ti;
    a.tiles = (unsigned)tiles;
    hipLaunchKernelGGL((product_wide<T, EPI, PL, QL, SPLIT>), dim3((unsigned)(tiles * splits)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace mpe
