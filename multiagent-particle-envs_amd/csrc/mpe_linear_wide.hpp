// Large products of 16-bit types.  Operands go from memory to LDS without passing registers (one instruction moves 64 x 16
// bytes), three stages deep: while a stage is multiplied the next has landed and the one after it is on its way.  A
// workgroup of four waves computes 128 x 256, each wave 64 x 128, which reads 12 KB of LDS for 32 matrix instructions;
// with 73 KB of LDS and half the registers two workgroups share a CU and one's results leave while the other multiplies.
//
// An operand whose contiguous index is the output's lies in LDS as it lies in memory, and ds_read_b64_tr_b16 turns it: 16
// lanes read four rows of 16 elements and each gets one column.
#pragma once
#include "mpe_linear_impl.hpp"

namespace mpe {

struct Wide {
    static constexpr int BI = 128, BJ = 256, BK = 32, STAGES = 3;
};

typedef __attribute__((address_space(3))) void lds_void;

// 16 bytes a lane from base + off (bytes) to LDS address `to`, lane after lane
__device__ inline void copy_to_lds(const char* base, unsigned off, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory", "m0");
}

// One operand's tile of BO x 32.  R_INNER: rows of 64 bytes, their four 16-byte chunks xored with the row, as Loader::place.
// O_INNER: 32 rows of BO elements, chunks xored with twice the row's last two bits, so that the four rows a transposed read
// touches lie on different banks.
template <typename T, int BO, int LAYOUT>
struct WideTile {
    typedef T vec8 __attribute__((ext_vector_type(8)));
    typedef short v4i16 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4i16 lds_v4;
    static constexpr int COPIES = BO / 64;      // instructions a wave and stage: 1 KB each
    static constexpr int BYTES = BO * 64;
    static constexpr int RUN = LAYOUT == R_INNER ? 4 : BO / 8;     // chunks a row of the tile

    unsigned off[COPIES];       // bytes from the tile's first element
    const char* next;
    long long step;

    static __device__ inline int swizzle(int row, int chunk) { return LAYOUT == R_INNER ? chunk ^ ((row >> 1) & 3) : chunk ^ ((row & 3) << 1); }

    __device__ inline void init(const Operand<T>& op, long long o0, long long no, long long r0) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, left = (int)min(no - o0, (long long)BO);
        const unsigned ld = (unsigned)op.ld;
#pragma unroll
        for (int u = 0; u < COPIES; ++u) {
            const int slot = (wave * COPIES + u) * 64 + lane, row = slot / RUN, chunk = swizzle(row, slot % RUN);
            // outputs that are not there read the last ones again and are never stored
            off[u] = (LAYOUT == R_INNER ? (unsigned)min(row, left - 1) * ld + chunk * 8 : (unsigned)row * ld + min(chunk * 8, left - 8)) * 2u;
        }
        next = (const char*)(op.data + (LAYOUT == R_INNER ? o0 * op.ld + r0 : r0 * op.ld + o0));
        step = LAYOUT == R_INNER ? 64 : 64 * op.ld;
    }

    __device__ inline void copy(unsigned lds, int wave) {
#pragma unroll
        for (int u = 0; u < COPIES; ++u) copy_to_lds(next, off[u], lds + (wave * COPIES + u) * 1024);
        next += step;
    }

    // The end of the sum, `left` < 32 of it, through registers: vectors kept inside the matrix by a Window, elements shifted
    // to their places, zeros behind the end.  All loads first.
    struct End {
        vec8 v[COPIES];
    };
    static __device__ inline int end_slot(int u) { return threadIdx.x + u * 256; }
    static __device__ inline unsigned end_off(int u, unsigned ld, int left_o) {
        const int row = end_slot(u) / RUN, chunk = swizzle(row, end_slot(u) % RUN);
        return LAYOUT == R_INNER ? (unsigned)min(row, left_o - 1) * ld + chunk * 8 : (unsigned)row * ld + min(chunk * 8, left_o - 8);
    }
    static __device__ inline void load_end(End& x, const Operand<T>& op, long long o0, long long no, long long r0) {
        const Window w(op.extent, LAYOUT == R_INNER ? o0 * op.ld + r0 : r0 * op.ld + o0, 8);
        const char* base = (const char*)(op.data + w.base);
#pragma unroll
        for (int u = 0; u < COPIES; ++u) __builtin_memcpy(&x.v[u], base + w.at(end_off(u, (unsigned)op.ld, (int)min(no - o0, (long long)BO))) * 2u, 16);
    }
    static __device__ inline void store_end(End& x, const Operand<T>& op, long long o0, long long no, long long r0, int left, char* lds) {
        const Window w(op.extent, LAYOUT == R_INNER ? o0 * op.ld + r0 : r0 * op.ld + o0, 8);
#pragma unroll
        for (int u = 0; u < COPIES; ++u) {
            const int row = end_slot(u) / RUN, chunk = swizzle(row, end_slot(u) % RUN);
            if (LAYOUT == R_INNER) {
                const int by = w.moved(end_off(u, (unsigned)op.ld, (int)min(no - o0, (long long)BO)));
                if (by > 0 && by < 8) shift_down<8>(x.v[u], by);
#pragma unroll
                for (int e = 0; e < 8; ++e) x.v[u][e] = chunk * 8 + e < left ? x.v[u][e] : (T)0.0f;
            } else if (row >= left) {
                x.v[u] = (T)0.0f;
            }
            *(vec8*)(lds + end_slot(u) * 16) = x.v[u];
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

template <typename T, int EPI, int PL, int QL>
__global__ __launch_bounds__(256, 2) void product_wide(const ProductArgs<T> a) {
    typedef WideTile<T, Wide::BI, PL> TP;
    typedef WideTile<T, Wide::BJ, QL> TQ;
    typedef T vec8 __attribute__((ext_vector_type(8)));
    constexpr int BI = Wide::BI, BJ = Wide::BJ, BK = Wide::BK, FI = 4, FJ = 8, STAGE = TP::BYTES + TQ::BYTES;
    constexpr int HALVES = 2, ROWS = BJ / HALVES, PITCH = BI + 4;
    static_assert(ROWS * PITCH * 4 <= Wide::STAGES * STAGE, "the results pass through the stages' memory");
    __shared__ __attribute__((aligned(16))) char lds[Wide::STAGES * STAGE];

    const unsigned t = xcd_run(blockIdx.x, gridDim.x), split = t / a.tiles, tile = t % a.tiles;
    const long long i0 = (long long)(tile % a.ti) * BI, j0 = (long long)(tile / a.ti) * BJ;
    const long long r0 = (long long)split * a.r_split, r1 = EPI == EPI_PARTIAL ? min(r0 + a.r_split, a.nr) : a.nr;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned base = (unsigned)(uintptr_t)(lds_void*)lds;
    const int wi = (wave & 1) * 64, wj = (wave >> 1) * 128;

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
            const vec8 fq = TQ::read(stage + TP::BYTES, wj + y * 16);
#pragma unroll
            for (int x = 0; x < FI; ++x) acc[x][y] = mfma(fp[x], fq, acc[x][y]);
        }
    };

    TP p;
    TQ q;
    p.init(a.p, i0, a.ni, r0);
    q.init(a.q, j0, a.nj, r0);
    const int steps = (int)((r1 - r0) / BK), left = (int)((r1 - r0) % BK);
    for (int s = 0; s < 2 && s < steps; ++s) {
        p.copy(base + s * STAGE, wave);
        q.copy(base + s * STAGE + TP::BYTES, wave);
    }
    if (left) {         // the end of the sum first, in the stage that is still free
        typename TP::End ep;
        typename TQ::End eq;
        TP::load_end(ep, a.p, i0, a.ni, r1 - left);
        TQ::load_end(eq, a.q, j0, a.nj, r1 - left);
        TP::store_end(ep, a.p, i0, a.ni, r1 - left, left, lds + 2 * STAGE);
        TQ::store_end(eq, a.q, j0, a.nj, r1 - left, left, lds + 2 * STAGE + TP::BYTES);
        __syncthreads();
        multiply(lds + 2 * STAGE);
    }
    int stage = 0;
    for (int s = 0; s < steps; ++s) {
        // stage s has landed when at most the copies of stage s + 1 are under way; the barrier makes that true of every
        // wave's share, and says that nobody reads stage s - 1 any more, into which stage s + 2 goes
        if (s + 1 < steps) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(TP::COPIES + TQ::COPIES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 2 < steps) {
            const unsigned to = base + (stage == 0 ? 2 : stage - 1) * STAGE;
            p.copy(to, wave);
            q.copy(to + TP::BYTES, wave);
        }
        multiply(lds + stage * STAGE);
        stage = stage == 2 ? 0 : stage + 1;
    }

    constexpr int N = EPI == EPI_FORWARD ? 8 : 4;       // a thread's columns
    const int it = threadIdx.x % (BI / N) * N;          // a thread's columns, the same in every row it takes
    const long long i = i0 + it;
    const int have = (int)max(0LL, min((long long)N, a.ni - i));
    const unsigned mask = (1u << have) - 1;
    float bias[N];
#pragma unroll
    for (int e = 0; e < N; ++e) bias[e] = EPI == EPI_FORWARD && a.bias && e < have ? (float)a.bias[i + e] : 0.0f;
    float* const res = (float*)lds;
#pragma unroll
    for (int half = 0; half < HALVES; ++half) {
        __syncthreads();
        if (wj / ROWS == half) {
#pragma unroll
            for (int y = 0; y < FJ; ++y)
#pragma unroll
                for (int x = 0; x < FI; ++x) *(f32x4*)&res[(y * 16 + (lane & 15)) * PITCH + wi + x * 16 + (lane >> 4) * 4] = acc[x][y];
        }
        __syncthreads();
        const int rows = (int)max(0LL, min((long long)ROWS, a.nj - j0 - half * ROWS));
        if (have > 0)
            finish_rows<T, EPI, N, 256 * N / BI>(a, split, i, j0 + half * ROWS, threadIdx.x / (BI / N), rows, mask, bias, [&](int jt, float* f) {
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

template <typename T, int EPI, int PL, int QL>
inline hipError_t launch_product_wide(ProductArgs<T> a, int splits, hipStream_t st) {
    const long long ti = (a.ni + Wide::BI - 1) / Wide::BI, tiles = ti * ((a.nj + Wide::BJ - 1) / Wide::BJ);
    if (tiles * splits > 0x7fffffffLL) return hipErrorInvalidValue;
    a.ti = (int)ti;
    a.tiles = (unsigned)tiles;
    hipLaunchKernelGGL((product_wide<T, EPI, PL, QL>), dim3((unsigned)(tiles * splits)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace mpe
