// The clipped policy loss over a rollout, and its gradient.  Per row (one decision of one agent), with the softmax over
// the allowed words only:
//   lp = l_a - lse(l),  q = exp(lp - old_lp),  s = min(q A, clamp(q, 1 - c, 1 + c) A),  H = lse(l) - sum p l
//   v  = max((V - R)^2, (V0 + clamp(V - V0, -c', c') - R)^2) / 2
//   loss = sum w (-s + cv v - ce H) / sum w
//   d loss / d l_k = w / sum w * (g (1[k = a] - p_k) + ce p_k (log p_k + H)),   g = -q A where q A <= the clamped term, else 0
// A row counts only if its weight is not zero and its action lies in [0, v), is allowed and has a logit above -inf (so
// that at least one word is left); any other row's gradients are zero.
//
// The backward pass takes no softmax statistics from the forward pass: it has to read the logits again anyway and
// recomputes them while the row is at hand.
#include <type_traits>

#include "mpe_learn.hpp"

namespace mpe {

namespace {

constexpr int NSTAT = 6;        // policy, value, entropy, kl, clipped, weight
// Grids.  Forward: five workgroups a CU, which all find room at once (the rollout of 4.9 M rows of five words: 67 us at 1024
// workgroups, 64 at 1280, 72 at 1792, when the last ones have to wait for a place), three and two where registers and LDS hold no
// more (ppo_few from 9 and from 33 words on; 50 M logits, 9 words 105 us at 768 and 112 at 1280, 24 words 87 and 95, 48 words 107 at
// 512 and 134 at 768).  Backward: enough that none is left over at the
// end (86 us at 4096 workgroups of 256 rows, 84 at 8192, 88 at 16384; whole rows: 50 us from 2048 to 16384, 55 at 1280).
//
// What bounds it.  4.9 M rows of five words: memory, 236 MB in 62 us (3.8 TB/s) and 354 MB in 82 (4.3); 60 float64 and some 150
// float32 operations a row hide behind it.  4096 rows of 8192 bf16 words with a mask: 101 MB in 23.8 us (4.2 TB/s), and 168 MB in
// 48.8 backwards (3.4 TB/s; asking for the next row while one is worked on was slower: 58, there are waves enough).
constexpr int FORWARD_GRID = 1280, FORWARD_GRID_32 = 768, FORWARD_GRID_FEW = 512, BACKWARD_GRID = 8192;
static_assert(FORWARD_GRID * 8 * NSTAT <= MPE_PPO_WORKSPACE_BYTES, "a partial sum for every workgroup");

struct Row {
    bool live;
    float w, old_lp, adv, v, v0, ret;
    long long a;
};

// the row but for its action's logit, which the caller looks at
__device__ inline Row read_row(const PpoArgs& p, long long r) {
    Row x;
    x.a = p.action_bytes == 8 ? ((const long long*)p.actions)[r] : (long long)((const int32_t*)p.actions)[r];
    x.w = p.weights ? p.weights[r] : 1.0f;
    x.live = x.w != 0.0f && x.a >= 0 && x.a < p.v;
    // read whether the row counts or not: no load waits for another
    x.old_lp = p.old_logp[r];
    x.adv = p.adv[r];
    x.v = p.values ? p.values[r] : 0.0f;
    x.v0 = p.values ? p.old_values[r] : 0.0f;
    x.ret = p.values ? p.returns[r] : 0.0f;
    return x;
}

// The value half of a row in float64: which square is the larger decides the gradient's branch, and differences of
// float32 numbers are exact there.
__device__ inline void value_terms(const PpoArgs& p, const Row& x, double& loss, double& slope) {
    const double v = x.v, v0 = x.v0, ret = x.ret;
    const double d = v - ret;
    loss = 0.5 * d * d;
    slope = d;
    if (p.value_clip >= 0.0f) {
        const double c = p.value_clip, step = v - v0;
        const double held = (step < -c ? v0 - c : step > c ? v0 + c : step == step ? v : step) - ret;     // NaN stays NaN
        if (d == d && !(held * held <= d * d)) {
            loss = 0.5 * held * held;
            slope = held == held ? 0.0 : held;      // beyond the border the held value does not move with v; inside it the two are equal
        }
    }
}

__device__ inline float fast_log(float x) { return __builtin_amdgcn_logf(x) * 0.69314718055994531f; }

// e^d d without 0 * inf where d is -inf or the type's lowest value (a NaN is left to the sum of e^d)
__device__ inline float weighted(float e, float d) { return e * fmaxf(d, -200.0f); }

// A row's softmax over the allowed words as maximum, sum of e^(l - m) and sum of e^(l - m) (l - m).  Maxima pass over NaN;
// the sums do not, so that a NaN logit reaches the loss whatever stands beside it.
struct Soft {
    float m, s, t;
};

__device__ inline Soft merge(Soft a, Soft b) {
    const float m = fmaxf(a.m, b.m);
    // a side that holds nothing (-inf) has the factor 0, which a NaN sum survives
    const float da = a.m == -INFINITY ? -INFINITY : a.m - m, db = b.m == -INFINITY ? -INFINITY : b.m - m;
    const float ea = fast_exp(da), eb = fast_exp(db);
    Soft c;
    c.m = m;
    c.s = a.s * ea + b.s * eb;
    c.t = ea * a.t + a.s * weighted(ea, da) + eb * b.t + b.s * weighted(eb, db);
    return c;
}

// What a row contributes, and the factors of its gradient, once its softmax is known.
struct Terms {
    float logs, ent, g, ce;
    double vslope, share;
};

template <bool BACK>
__device__ inline Terms row_terms(const PpoArgs& p, const Row& x, const Soft& q, float at, float share_all, double* sum) {
    Terms y;
    y.logs = fast_log(q.s);
    y.ent = y.logs - q.t / q.s;
    const float diff = at - q.m - y.logs - x.old_lp, ratio = fast_exp(diff);
    const float held = fminf(fmaxf(ratio, 1.0f - p.clip), 1.0f + p.clip);      // of a NaN a number: free_term shows it
    // a ratio beyond float32 is a number all the same, and nothing times zero
    const float free_term = x.adv == 0.0f && fabsf(diff) < INFINITY ? 0.0f : ratio * x.adv, held_term = held * x.adv;
    double vloss = 0.0, vslope = 0.0;
    if (p.values) value_terms(p, x, vloss, vslope);
    if (BACK) {
        const float share = share_all * x.w;
        y.g = free_term <= held_term ? -free_term * share : 0.0f;
        if (free_term != free_term) y.g = free_term;      // and here
        y.ce = p.entropy_coef * share;
        y.vslope = vslope;
        y.share = (double)(p.value_coef * share);
    } else {
        const double w = x.w;
        sum[0] -= w * (double)(free_term > held_term ? held_term : free_term);      // NaN has to show
        sum[1] += w * vloss;
        sum[2] += w * y.ent;
        sum[3] += w * 0.5 * (double)diff * (double)diff;
        sum[4] += fabsf(ratio - 1.0f) > p.clip ? w : 0.0;
        sum[5] += w;
    }
    return y;
}

// gradient of one allowed logit
__device__ inline float logit_grad(const Terms& y, const Soft& q, float l, bool is_action) {
    const float lk = l - q.m - y.logs, pk = fast_exp(lk);
    return (is_action ? y.g : 0.0f) + pk * (y.ce * y.ent - y.g) + y.ce * weighted(pk, lk);
}

__device__ inline float share_of(const PpoArgs& p) {
    const float total = p.stats[5];
    return total != 0.0f ? p.grad[0] / total : 0.0f;
}

// loss and stats from the total sums
__device__ inline void write_totals(const double* tot, float value_coef, float entropy_coef, float* loss, float* stats) {
    const double inv = tot[5] != 0.0 ? 1.0 / tot[5] : 0.0;
    for (int i = 0; i < 5; ++i) stats[i] = (float)(tot[i] * inv);
    stats[5] = (float)tot[5];
    *loss = (float)((tot[0] + (double)value_coef * tot[1] - (double)entropy_coef * tot[2]) * inv);
}

// Sums over a workgroup, sum i in thread i; all threads have to come here.
template <int WAVES>
__device__ inline double group_sums(const double* sum, double (*scratch)[NSTAT]) {
    for (int i = 0; i < NSTAT; ++i) {
        const double v = wave_sum(sum[i]);
        if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6][i] = v;
    }
    __syncthreads();
    double t = 0.0;
    if (threadIdx.x < NSTAT)
#pragma unroll
        for (int w = 0; w < WAVES; ++w) t += scratch[w][threadIdx.x];
    return t;
}

// A launch of one workgroup is done with its sums, another leaves partial sums for ppo_finish.
template <int WAVES>
__device__ inline void leave_sums(const PpoArgs& p, const double* sum, double (*scratch)[NSTAT]) {
    const double t = group_sums<WAVES>(sum, scratch);
    if (gridDim.x > 1) {
        if (threadIdx.x < NSTAT) p.ws[blockIdx.x * NSTAT + threadIdx.x] = t;
        return;
    }
    __syncthreads();
    if (threadIdx.x < NSTAT) scratch[0][threadIdx.x] = t;
    __syncthreads();
    if (threadIdx.x == 0) write_totals(scratch[0], p.value_coef, p.entropy_coef, p.loss, p.stats);
}

// Few words: a lane takes a row.  A workgroup's 256 rows are fetched into LDS (consecutive lanes read consecutive elements
// whatever v is; rows there are an odd number of words apart, so that 64 lanes walking their rows meet 64 banks) and the
// gradients leave the same way.
constexpr int FEW = 62;         // 256 rows of 63 floats end with 64 KB of LDS

template <typename T, bool BACK, int VR>        // VR: at least v
__global__ __launch_bounds__(256) void ppo_few(const PpoArgs p) {
    extern __shared__ float tile[];
    __shared__ double scratch[4][NSTAT];
    const int v = (int)p.v, stride = v | 1, tid = threadIdx.x;
    const int dr = 256 / v, dc = 256 % v, row0 = tid / v, col0 = tid % v;
    double sum[NSTAT] = {0, 0, 0, 0, 0, 0};
    const float share_all = BACK ? share_of(p) : 0.0f;

    // the next tile's loads are in flight while this one is worked on
    typedef std::conditional_t<(VR > 32), unsigned long long, unsigned> bits;
    T raw[VR];
    bits ok = 0;
    Row next;
    auto load = [&](long long r0) {
        const int rows = (int)min(256LL, p.rows - r0), n = rows * v;
        next = read_row(p, r0 + min(tid, rows - 1));
        const T* base = (const T*)p.logits + r0 * p.ld;
        const uint8_t* mask = p.mask ? p.mask + r0 * p.ldm : nullptr;
        int row = row0, col = col0;
        ok = 0;
#pragma unroll
        for (int u = 0; u < VR; ++u)
            if (u < v) {
                if (tid + u * 256 < n) {
                    raw[u] = base[(long long)row * p.ld + col];
                    ok |= (!mask || mask[(long long)row * p.ldm + col] ? (bits)1 : (bits)0) << u;
                }
                row += dr;
                col += dc;
                if (col >= v) { col -= v; ++row; }
            }
    };

    const long long step = (long long)gridDim.x * 256;
    long long r0 = (long long)blockIdx.x * 256;
    if (r0 < p.rows) load(r0);
    for (; r0 < p.rows; r0 += step) {
        const int rows = (int)min(256LL, p.rows - r0), n = rows * v;
        Row x = next;
        __syncthreads();
        {
            int row = row0, col = col0;
#pragma unroll
            for (int u = 0; u < VR; ++u)
                if (u < v) {
                    if (tid + u * 256 < n) tile[row * stride + col] = ok >> u & 1 ? (float)raw[u] : -INFINITY;     // a forbidden word is one of weight zero
                    row += dr;
                    col += dc;
                    if (col >= v) { col -= v; ++row; }
                }
        }
        __syncthreads();
        if (r0 + step < p.rows) load(r0 + step);
        float* l = tile + tid * stride;
        if (tid < rows) {
            const long long r = r0 + tid;
            float at = 0.0f;
            if (x.live) {
                at = l[x.a];
                x.live = at != -INFINITY;
            }
            if (x.live) {
                Soft q = {-INFINITY, 0.0f, 0.0f};
                for (int k = 0; k < v; ++k) q.m = fmaxf(q.m, l[k]);
                for (int k = 0; k < v; ++k) {
                    const float d = l[k] - q.m, e = fast_exp(d);
                    q.s += e;
                    q.t += weighted(e, d);
                }
                const Terms y = row_terms<BACK>(p, x, q, at, share_all, sum);
                if (BACK) {
                    for (int k = 0; k < v; ++k) l[k] = logit_grad(y, q, l[k], k == x.a);
                    if (p.dvalues) p.dvalues[r] = (float)(y.vslope * y.share);
                }
            } else if (BACK) {
                for (int k = 0; k < v; ++k) l[k] = 0.0f;
                if (p.dvalues) p.dvalues[r] = 0.0f;
            }
        }
        if (BACK) {
            __syncthreads();
            int row = row0, col = col0;
            T* base = (T*)p.dlogits + r0 * p.ldd;
            for (int i = tid; i < n; i += 256) {
                base[(long long)row * p.ldd + col] = (T)tile[row * stride + col];
                row += dr;
                col += dc;
                if (col >= v) { col -= v; ++row; }
            }
        }
    }
    if (!BACK) leave_sums<4>(p, sum, scratch);
}

// Many words: W waves take a row and hold it in registers, NV 16-byte vectors a thread (NV 0: the row is too long; it is
// read twice, the second time mostly from L2).
template <typename T, bool BACK, int W, int NV>
__global__ __launch_bounds__(256) void ppo_many(const PpoArgs p) {
    constexpr int E = 16 / (int)sizeof(T), GROUPS = 4 / W, LANES = W * 64;
    __shared__ double scratch[4][NSTAT];
    __shared__ Soft part[4];
    const int lane = threadIdx.x % LANES;
    double sum[NSTAT] = {0, 0, 0, 0, 0, 0};
    const float share_all = BACK ? share_of(p) : 0.0f;

    // words [k, k + E) of the row, a forbidden one and one behind the end as -inf
    auto fetch = [&](long long r, long long k, T* f) {
        const T* l = (const T*)p.logits + r * p.ld + k;
        if (k + E <= p.v) {
            __builtin_memcpy(f, l, E * sizeof(T));
            if (p.mask) {
                uint8_t ok[E];
                __builtin_memcpy(ok, p.mask + r * p.ldm + k, E);
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = ok[e] ? f[e] : (T)-INFINITY;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = k + e < p.v && (!p.mask || p.mask[r * p.ldm + k + e]) ? l[e] : (T)-INFINITY;
        }
    };
    auto take = [&](Soft& q, const T* f, float m) {      // adds E words relative to m; where m is -inf there are only -inf and NaN
        const float m0 = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = (float)f[e] - m0, x = fast_exp(d);
            q.s += x;
            q.t += weighted(x, d);
        }
    };
    auto give = [&](long long r, long long k, const T* f, const Row& x, const Terms& y, const Soft& q) {
        T* d = (T*)p.dlogits + r * p.ldd + k;
        T out[E];
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = (T)(x.live ? logit_grad(y, q, (float)f[e], k + e == x.a) : 0.0f);
        if (k + E <= p.v) __builtin_memcpy(d, out, sizeof(out));
        else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (k + e < p.v) d[e] = out[e];
        }
    };

    // all waves of a workgroup take as many turns, so that they meet at the barriers
    const long long turns = (p.rows + GROUPS - 1) / GROUPS;
    for (long long turn = blockIdx.x; turn < turns; turn += gridDim.x) {
        const long long r = turn * GROUPS + (GROUPS > 1 ? (int)threadIdx.x / LANES : 0);
        const bool here = r < p.rows;
        Row x = {};
        if (here) x = read_row(p, r);
        float at = 0.0f;
        if (x.live) {
            at = !p.mask || p.mask[r * p.ldm + x.a] ? (float)((const T*)p.logits)[r * p.ld + x.a] : -INFINITY;
            x.live = at != -INFINITY;
        }
        T f[NV ? NV : 1][E];
        Soft q = {-INFINITY, 0.0f, 0.0f};
        if (x.live) {
            if (NV) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const long long k = ((long long)i * LANES + lane) * E;
                    if (k < p.v) fetch(r, k, f[i]);
                    else
#pragma unroll
                        for (int e = 0; e < E; ++e) f[i][e] = (T)-INFINITY;
                }
                // one maximum for all that a thread holds
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) q.m = fmaxf(q.m, (float)f[i][e]);
#pragma unroll
                for (int i = 0; i < NV; ++i) take(q, f[i], q.m);
            } else {
                for (long long k = (long long)lane * E; k < p.v; k += LANES * E) {
                    fetch(r, k, f[0]);
                    Soft w = {-INFINITY, 0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < E; ++e) w.m = fmaxf(w.m, (float)f[0][e]);
                    take(w, f[0], w.m);
                    q = merge(q, w);
                }
            }
        }
        // the wave's maximum first: then its sums are plain sums
        {
            const float m = wave_reduce(q.m, [](float a, float b) { return fmaxf(a, b); });
            const float d = q.m == -INFINITY ? -INFINITY : q.m - m, e = fast_exp(d);       // a thread that holds nothing has the factor 0
            const float t = e * q.t + q.s * weighted(e, d);
            q.m = m;
            q.t = wave_sum(t);
            q.s = wave_sum(q.s * e);
        }
        if (W > 1) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = q;
            __syncthreads();
            q = part[0];
#pragma unroll
            for (int w = 1; w < W; ++w) q = merge(q, part[w]);
        }
        Terms y = {};
        if (x.live) {
            double mine[NSTAT] = {0, 0, 0, 0, 0, 0};
            y = row_terms<BACK>(p, x, q, at, share_all, mine);
            if (!BACK && lane == 0)
                for (int i = 0; i < NSTAT; ++i) sum[i] += mine[i];
        }
        if (BACK && here) {
            if (NV) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const long long k = ((long long)i * LANES + lane) * E;
                    if (k < p.v) give(r, k, f[i], x, y, q);
                }
            } else {
                for (long long k = (long long)lane * E; k < p.v; k += LANES * E) {
                    if (x.live) fetch(r, k, f[0]);
                    give(r, k, f[0], x, y, q);
                }
            }
            if (p.dvalues && lane == 0) p.dvalues[r] = x.live ? (float)(y.vslope * y.share) : 0.0f;
        }
    }
    if (!BACK) leave_sums<4>(p, sum, scratch);
}

// The values' gradient alone: which rows count, and nothing of the softmax.
template <typename T>
__global__ __launch_bounds__(256) void ppo_values(const PpoArgs p) {
    const float share_all = share_of(p);
    for (long long r = (long long)blockIdx.x * 256 + threadIdx.x; r < p.rows; r += (long long)gridDim.x * 256) {
        const Row x = read_row(p, r);
        double vloss, vslope;
        value_terms(p, x, vloss, vslope);
        const bool live = x.live && (!p.mask || p.mask[r * p.ldm + x.a]) && (float)((const T*)p.logits)[r * p.ld + x.a] != -INFINITY;
        p.dvalues[r] = live ? (float)(vslope * (double)(p.value_coef * (share_all * x.w))) : 0.0f;
    }
}

__global__ __launch_bounds__(1024) void ppo_finish(const double* __restrict__ partial, int n, float value_coef, float entropy_coef,
                                                   float* __restrict__ loss, float* __restrict__ stats) {
    __shared__ double scratch[16][NSTAT];
    double tot[NSTAT] = {0, 0, 0, 0, 0, 0};
    for (int b = threadIdx.x; b < n; b += 1024)
        for (int i = 0; i < NSTAT; ++i) tot[i] += partial[b * NSTAT + i];
    const double t = group_sums<16>(tot, scratch);
    __syncthreads();
    if (threadIdx.x < NSTAT) scratch[0][threadIdx.x] = t;
    __syncthreads();
    if (threadIdx.x == 0) write_totals(scratch[0], value_coef, entropy_coef, loss, stats);
}

// A variant goes as far as its registers and its LDS do.  On both sides of each border, 50 M logits forward and backward, us: 32
// words 83 and 130 in ppo_few, 552 and 574 in ppo_many; 62 words 99 and 170, 63 in ppo_many 328 and 374; one vector a lane, 256
// float32 words 79 and 110, with room for four 115 and 156; four vectors, 1024 words 38 and 90, four waves a row 106 and 157; four waves,
// 4096 words 38 and 83, read twice 66 and 179 (bfloat16, 8192 words: 31 and 62, 37 and 88).
template <typename T, bool BACK>
hipError_t launch_rows(const PpoArgs& a, int* grid_out, hipStream_t st) {
    const auto grid_for = [&](long long per_block, int forward_grid = FORWARD_GRID) {
        const int most = BACK ? BACKWARD_GRID : forward_grid;
        long long g = (a.rows + per_block - 1) / per_block;
        g = g < 1 ? 1 : g > most ? most : g;
        if (grid_out) *grid_out = (int)g;
        return dim3((unsigned)g);
    };
    constexpr int E = 16 / (int)sizeof(T);
    if (a.v <= FEW) {
        const size_t bytes = 256 * (size_t)(a.v | 1) * 4;
        if (a.v <= 8) hipLaunchKernelGGL((ppo_few<T, BACK, 8>), grid_for(256), dim3(256), bytes, st, a);
        else if (a.v <= 32) hipLaunchKernelGGL((ppo_few<T, BACK, 32>), grid_for(256, FORWARD_GRID_32), dim3(256), bytes, st, a);
        else hipLaunchKernelGGL((ppo_few<T, BACK, FEW>), grid_for(256, FORWARD_GRID_FEW), dim3(256), bytes, st, a);
    } else if (a.v <= 64 * E) {
        hipLaunchKernelGGL((ppo_many<T, BACK, 1, 1>), grid_for(4), dim3(256), 0, st, a);
    } else if (a.v <= 4 * 64 * E) {
        hipLaunchKernelGGL((ppo_many<T, BACK, 1, 4>), grid_for(4), dim3(256), 0, st, a);
    } else if (a.v <= 4 * 256 * E) {
        hipLaunchKernelGGL((ppo_many<T, BACK, 4, 4>), grid_for(1), dim3(256), 0, st, a);
    } else {
        hipLaunchKernelGGL((ppo_many<T, BACK, 4, 0>), grid_for(1), dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_ppo_forward(const PpoArgs& a, hipStream_t st) {
    int grid = 0;
    hipError_t e = with_dtype(a.dtype, [&](auto z) { return launch_rows<decltype(z), false>(a, &grid, st); });
    if (e != hipSuccess || grid == 1) return e;
    hipLaunchKernelGGL(ppo_finish, dim3(1), dim3(1024), 0, st, a.ws, grid, a.value_coef, a.entropy_coef, a.loss, a.stats);
    return hipGetLastError();
}

hipError_t launch_ppo_backward(const PpoArgs& a, hipStream_t st) {
    if (a.rows == 0) return hipSuccess;
    if (!a.dlogits) {
        const long long want = (a.rows + 255) / 256;
        return with_dtype(a.dtype, [&](auto z) {
            hipLaunchKernelGGL((ppo_values<decltype(z)>), dim3((unsigned)(want < BACKWARD_GRID ? want : BACKWARD_GRID)), dim3(256), 0, st, a);
            return hipGetLastError();
        });
    }
    return with_dtype(a.dtype, [&](auto z) { return launch_rows<decltype(z), true>(a, nullptr, st); });
}

}  // namespace mpe
