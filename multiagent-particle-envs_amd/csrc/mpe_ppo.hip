// The clipped policy loss over a rollout, and its gradient.  Per row (one decision of one agent), with the softmax over
// the allowed words only:
//   lp = l_a - lse(l),  q = exp(lp - old_lp),  s = min(q A, clamp(q, 1 - c, 1 + c) A),  H = lse(l) - sum p l
//   v  = max((V - R)^2, (V0 + clamp(V - V0, -c', c') - R)^2) / 2
//   loss = sum w (-s + cv v - ce H) / sum w
//   d loss / d l_k = w / sum w * (g (1[k = a] - p_k) + ce p_k (log p_k + H)),   g = -q A where q A <= the clamped term, else 0
// A row counts only if its weight is not zero and its action lies in [0, v), is allowed and has a logit above -inf (so
// that at least one word is left); any other row is not read further and its gradients are zero.
//
// The backward pass takes no softmax statistics from the forward pass: it has to read the logits again anyway and
// recomputes them while the row is at hand.
#include "mpe_learn.hpp"

namespace mpe {

namespace {

constexpr int NSTAT = 6;        // policy, value, entropy, kl, clipped, weight
constexpr int BLOCKS = MPE_PPO_WORKSPACE_BYTES / (8 * NSTAT);

// Maximum that keeps NaN: a NaN logit has to reach the loss, whatever stands beside it.
__device__ inline float larger(float a, float b) { return a > b || a != a ? a : b; }

struct Row {
    bool live;
    float w, old_lp, adv;
    long long a;
};

// the row but for its action's logit, which the caller looks at
__device__ inline Row read_row(const PpoArgs& p, long long r) {
    Row x;
    x.a = p.action_bytes == 8 ? ((const long long*)p.actions)[r] : (long long)((const int32_t*)p.actions)[r];
    x.w = p.weights ? p.weights[r] : 1.0f;
    x.live = x.w != 0.0f && x.a >= 0 && x.a < p.v;
    x.old_lp = x.live ? p.old_logp[r] : 0.0f;
    x.adv = x.live ? p.adv[r] : 0.0f;
    return x;
}

// The value half of a row in float64: which square is the larger decides the gradient's branch, and differences of
// float32 numbers are exact there.
__device__ inline void value_terms(const PpoArgs& p, long long r, double& loss, double& slope) {
    const double v = p.values[r], v0 = p.old_values[r], ret = p.returns[r];
    const double d = v - ret;
    loss = 0.5 * d * d;
    slope = d;
    if (p.value_clip >= 0.0f) {
        const double c = p.value_clip, step = v - v0;
        const double held = (step < -c ? v0 - c : step > c ? v0 + c : v) - ret;
        if (held * held > d * d) {
            loss = 0.5 * held * held;
            slope = 0.0;        // beyond the border the held value does not move with v; inside it the two are equal
        }
    }
}

// exp by the hardware's 2^x: off by the rounding of d log2(e), |d| 2^-24, and one step
__device__ inline float fast_exp(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896341f); }

// A row's softmax over the allowed words as running maximum, sum and sum of e^(l - m) (l - m).
struct Soft {
    float m, s, t;
};

__device__ inline Soft merge(Soft a, Soft b) {
    const float m = larger(a.m, b.m);
    // a side that holds nothing (-inf) adds nothing, whatever m is
    const float da = a.m - m, db = b.m - m, ea = a.m == -INFINITY ? 0.0f : fast_exp(da), eb = b.m == -INFINITY ? 0.0f : fast_exp(db);
    Soft c;
    c.m = m;
    c.s = a.s * ea + b.s * eb;
    c.t = (ea == 0.0f ? 0.0f : ea * (a.t + a.s * da)) + (eb == 0.0f ? 0.0f : eb * (b.t + b.s * db));
    return c;
}

// What a row contributes, and the factors of its gradient, once its softmax is known.
struct Terms {
    float logs, ent, g, ce;
    double vslope, share;
};

template <bool BACK>
__device__ inline Terms row_terms(const PpoArgs& p, long long r, const Row& x, const Soft& q, float at, float share_all, double* sum) {
    Terms y;
    y.logs = logf(q.s);
    y.ent = y.logs - q.t / q.s;
    const float diff = at - q.m - y.logs - x.old_lp, ratio = expf(diff);
    const float held = fminf(fmaxf(ratio, 1.0f - p.clip), 1.0f + p.clip);
    const float free_term = ratio * x.adv, held_term = held * x.adv;
    double vloss = 0.0, vslope = 0.0;
    if (p.values) value_terms(p, r, vloss, vslope);
    if (BACK) {
        const float share = share_all * x.w;
        y.g = free_term <= held_term ? -free_term * share : 0.0f;
        if (free_term != free_term) y.g = free_term;      // NaN has to show
        y.ce = p.entropy_coef * share;
        y.vslope = vslope;
        y.share = (double)(p.value_coef * share);
    } else {
        const double w = x.w;
        sum[0] -= w * (double)(free_term <= held_term ? free_term : held_term);
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
    return (is_action ? y.g : 0.0f) - y.g * pk + (pk == 0.0f ? 0.0f : y.ce * pk * (lk + y.ent));
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

// Sums over the workgroup; a launch of one workgroup is done with that, another leaves partial sums for ppo_finish.
template <int WAVES>
__device__ inline void leave_sums(const PpoArgs& p, const double* sum, double (*scratch)[NSTAT]) {
    double v[NSTAT];
    for (int i = 0; i < NSTAT; ++i) v[i] = wave_sum(sum[i]);
    if ((threadIdx.x & 63) == 0)
        for (int i = 0; i < NSTAT; ++i) scratch[threadIdx.x >> 6][i] = v[i];
    __syncthreads();
    if (threadIdx.x == 0) {
        double tot[NSTAT];
        for (int i = 0; i < NSTAT; ++i) {
            tot[i] = 0.0;
            for (int w = 0; w < WAVES; ++w) tot[i] += scratch[w][i];
        }
        if (gridDim.x == 1) write_totals(tot, p.value_coef, p.entropy_coef, p.loss, p.stats);
        else
            for (int i = 0; i < NSTAT; ++i) p.ws[blockIdx.x * NSTAT + i] = tot[i];
    }
}

// Few words: a lane takes a row.  A workgroup's 256 rows are fetched into LDS (consecutive lanes read consecutive elements
// whatever v is; rows there are an odd number of words apart, so that 64 lanes walking their rows meet 64 banks) and the
// gradients leave the same way.
constexpr int FEW = 32;

template <typename T, bool BACK>
__global__ __launch_bounds__(256) void ppo_few(const PpoArgs p) {
    extern __shared__ float tile[];
    __shared__ double scratch[4][NSTAT];
    const int v = (int)p.v, stride = v | 1, tid = threadIdx.x;
    const int dr = 256 / v, dc = 256 % v;
    double sum[NSTAT] = {0, 0, 0, 0, 0, 0};
    const float share_all = BACK ? share_of(p) : 0.0f;
    for (long long r0 = (long long)blockIdx.x * 256; r0 < p.rows; r0 += (long long)gridDim.x * 256) {
        const int rows = (int)min(256LL, p.rows - r0), n = rows * v;
        __syncthreads();
        {
            int row = tid / v, col = tid % v;
            const T* base = (const T*)p.logits + r0 * p.ld;
            for (int i = tid; i < n; i += 256) {
                const long long at = (long long)row * p.ld + col;
                const bool ok = !p.mask || p.mask[(r0 + row) * p.ldm + col];
                tile[row * stride + col] = ok ? (float)base[at] : -INFINITY;      // a forbidden word is one of weight zero
                row += dr;
                col += dc;
                if (col >= v) { col -= v; ++row; }
            }
        }
        __syncthreads();
        float* l = tile + tid * stride;
        if (tid < rows) {
            const long long r = r0 + tid;
            Row x = read_row(p, r);
            float at = 0.0f;
            if (x.live) {
                at = l[x.a];
                x.live = at != -INFINITY;
            }
            if (x.live) {
                Soft q = {-INFINITY, 0.0f, 0.0f};
                for (int k = 0; k < v; ++k) q.m = larger(q.m, l[k]);
                for (int k = 0; k < v; ++k) {
                    const float d = l[k] - q.m, e = fast_exp(d);
                    q.s += e;
                    q.t += e == 0.0f ? 0.0f : e * d;      // -inf and the type's lowest value: nothing, not 0 * inf
                }
                const Terms y = row_terms<BACK>(p, r, x, q, at, share_all, sum);
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
            int row = tid / v, col = tid % v;
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

    // vector i of the row: words [k, k + E) as float32, a forbidden word and one behind the end as -inf
    auto fetch = [&](long long r, long long k, float* f) {
        const T* l = (const T*)p.logits + r * p.ld + k;
        if (k + E <= p.v) {
            T raw[E];
            __builtin_memcpy(raw, l, sizeof(raw));
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = (float)raw[e];
            if (p.mask) {
                uint8_t ok[E];
                __builtin_memcpy(ok, p.mask + r * p.ldm + k, E);
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = ok[e] ? f[e] : -INFINITY;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = k + e < p.v && (!p.mask || p.mask[r * p.ldm + k + e]) ? (float)l[e] : -INFINITY;
        }
    };
    auto take = [&](Soft& q, const float* f) {      // adds E words
        float m = q.m;
#pragma unroll
        for (int e = 0; e < E; ++e) m = larger(m, f[e]);
        if (m == -INFINITY) return;
        if (m != q.m && q.m != -INFINITY) {
            const float d = q.m - m, c = fast_exp(d);
            q.t = c == 0.0f ? 0.0f : c * (q.t + q.s * d);
            q.s *= c;
        }
        q.m = m;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = f[e] - m, x = fast_exp(d);
            q.s += x;
            q.t += x == 0.0f ? 0.0f : x * d;
        }
    };
    auto give = [&](long long r, long long k, const float* f, const Row& x, const Terms& y, const Soft& q) {
        T* d = (T*)p.dlogits + r * p.ldd + k;
        T out[E];
#pragma unroll
        for (int e = 0; e < E; ++e) out[e] = (T)(x.live ? logit_grad(y, q, f[e], k + e == x.a) : 0.0f);
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
        float f[NV ? NV : 1][E];
        Soft q = {-INFINITY, 0.0f, 0.0f};
        if (x.live) {
            if (NV) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const long long k = ((long long)i * LANES + lane) * E;
                    if (k < p.v) fetch(r, k, f[i]);
                    else
#pragma unroll
                        for (int e = 0; e < E; ++e) f[i][e] = -INFINITY;
                }
                // one maximum for all that a thread holds
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) q.m = larger(q.m, f[i][e]);
                if (q.m != -INFINITY) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) take(q, f[i]);
                }
            } else {
                for (long long k = (long long)lane * E; k < p.v; k += LANES * E) {
                    fetch(r, k, f[0]);
                    take(q, f[0]);
                }
            }
        }
        for (int o = 32; o; o >>= 1) {
            const Soft b = {__shfl_xor(q.m, o), __shfl_xor(q.s, o), __shfl_xor(q.t, o)};
            q = merge(q, b);
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
            y = row_terms<BACK>(p, r, x, q, at, share_all, mine);
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

__global__ __launch_bounds__(1024) void ppo_finish(const double* __restrict__ partial, int n, float value_coef, float entropy_coef,
                                                   float* __restrict__ loss, float* __restrict__ stats) {
    __shared__ double scratch[16][NSTAT];
    double tot[NSTAT] = {0, 0, 0, 0, 0, 0};
    for (int b = threadIdx.x; b < n; b += 1024)
        for (int i = 0; i < NSTAT; ++i) tot[i] += partial[b * NSTAT + i];
    for (int i = 0; i < NSTAT; ++i) tot[i] = wave_sum(tot[i]);
    if ((threadIdx.x & 63) == 0)
        for (int i = 0; i < NSTAT; ++i) scratch[threadIdx.x >> 6][i] = tot[i];
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 0; i < NSTAT; ++i) {
            tot[i] = 0.0;
            for (int w = 0; w < 16; ++w) tot[i] += scratch[w][i];
        }
        write_totals(tot, value_coef, entropy_coef, loss, stats);
    }
}

template <typename T, bool BACK>
hipError_t launch_rows(const PpoArgs& a, int most, int* grid_out, hipStream_t st) {
    const auto grid_for = [&](long long per_block) {
        long long g = (a.rows + per_block - 1) / per_block;
        g = g < 1 ? 1 : g > most ? most : g;
        if (grid_out) *grid_out = (int)g;
        return dim3((unsigned)g);
    };
    constexpr int E = 16 / (int)sizeof(T);
    if (a.v <= FEW) {
        const size_t bytes = 256 * (size_t)(a.v | 1) * 4;
        hipLaunchKernelGGL((ppo_few<T, BACK>), grid_for(256), dim3(256), bytes, st, a);
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
    hipError_t e = with_dtype(a.dtype, [&](auto z) { return launch_rows<decltype(z), false>(a, BLOCKS, &grid, st); });
    if (e != hipSuccess || grid == 1) return e;
    hipLaunchKernelGGL(ppo_finish, dim3(1), dim3(1024), 0, st, a.ws, grid, a.value_coef, a.entropy_coef, a.loss, a.stats);
    return hipGetLastError();
}

hipError_t launch_ppo_backward(const PpoArgs& a, hipStream_t st) {
    if (a.rows == 0) return hipSuccess;
    return with_dtype(a.dtype, [&](auto z) { return launch_rows<decltype(z), true>(a, 16384, nullptr, st); });
}

}  // namespace mpe
