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
__device__ inline float wave_larger(float v) {
    for (int o = 32; o; o >>= 1) v = larger(v, __shfl_xor(v, o));
    return v;
}

struct Row {
    bool live;
    float w, old_lp, adv;
    long long a;
};

template <typename T>
__device__ inline Row read_row(const PpoArgs& p, long long r) {
    Row x;
    x.a = p.action_bytes == 8 ? ((const long long*)p.actions)[r] : (long long)((const int32_t*)p.actions)[r];
    x.w = p.weights ? p.weights[r] : 1.0f;
    x.live = x.w != 0.0f && x.a >= 0 && x.a < p.v;
    if (x.live) x.live = (!p.mask || p.mask[r * p.ldm + x.a]) && (float)((const T*)p.logits)[r * p.ld + x.a] != -INFINITY;
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

template <typename T, bool BACK>
__global__ __launch_bounds__(256) void ppo_wave(const PpoArgs p) {
    __shared__ double scratch[4];
    const int lane = threadIdx.x & 63;
    const long long wave = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), waves = (long long)gridDim.x * 4;
    double sum[NSTAT] = {0, 0, 0, 0, 0, 0};
    float share_all = 0.0f;
    if (BACK) {
        const float total = p.stats[5];
        share_all = total != 0.0f ? p.grad[0] / total : 0.0f;
    }
    for (long long r = wave; r < p.rows; r += waves) {
        const Row x = read_row<T>(p, r);
        const T* l = (const T*)p.logits + r * p.ld;
        const uint8_t* ok = p.mask ? p.mask + r * p.ldm : nullptr;
        float mx = -INFINITY;
        if (x.live)
            for (long long k = lane; k < p.v; k += 64)
                if (!ok || ok[k]) mx = larger(mx, (float)l[k]);
        mx = wave_larger(mx);
        float s = 0.0f, t = 0.0f;
        if (x.live)
            for (long long k = lane; k < p.v; k += 64)
                if (!ok || ok[k]) {
                    const float d = (float)l[k] - mx, e = expf(d);
                    s += e;
                    t += e == 0.0f ? 0.0f : e * d;      // -inf and the type's lowest value: nothing, not 0 * inf
                }
        s = wave_sum(s);
        t = wave_sum(t);
        if (x.live) {
            const float logs = logf(s), ent = logs - t / s;
            const float lp = (float)l[x.a] - mx - logs;
            const float diff = lp - x.old_lp, q = expf(diff);
            const float held = fminf(fmaxf(q, 1.0f - p.clip), 1.0f + p.clip);
            const float free_term = q * x.adv, held_term = held * x.adv;
            const bool moves = free_term <= held_term;
            double vloss = 0.0, vslope = 0.0;
            if (p.values) value_terms(p, r, vloss, vslope);
            if (BACK) {
                const float share = share_all * x.w;
                const float g = moves ? -free_term * share : 0.0f, ce = p.entropy_coef * share;
                for (long long k = lane; k < p.v; k += 64) {
                    float out = 0.0f;
                    if (!ok || ok[k]) {
                        const float lk = (float)l[k] - mx - logs, pk = expf(lk);
                        out = (k == x.a ? g : 0.0f) - g * pk + (pk == 0.0f ? 0.0f : ce * pk * (lk + ent));
                    }
                    ((T*)p.dlogits)[r * p.ldd + k] = (T)out;
                }
                if (p.dvalues && lane == 0) p.dvalues[r] = (float)(vslope * (double)(p.value_coef * share));
            } else {
                const double w = x.w;
                sum[0] -= w * (double)fminf(free_term, held_term);
                sum[1] += w * vloss;
                sum[2] += w * ent;
                sum[3] += w * 0.5 * (double)diff * (double)diff;
                sum[4] += fabsf(q - 1.0f) > p.clip ? w : 0.0;
                sum[5] += w;
            }
        } else if (BACK) {
            for (long long k = lane; k < p.v; k += 64) ((T*)p.dlogits)[r * p.ldd + k] = (T)0.0f;
            if (p.dvalues && lane == 0) p.dvalues[r] = 0.0f;
        }
    }
    if (!BACK) {
        for (int i = 0; i < NSTAT; ++i) {
            const double v = block_sum<4>(lane == 0 ? sum[i] : 0.0, scratch);
            if (threadIdx.x == 0) p.ws[blockIdx.x * NSTAT + i] = v;
        }
    }
}

__global__ __launch_bounds__(256) void ppo_finish(const double* __restrict__ partial, int n, float value_coef, float entropy_coef,
                                                  float* __restrict__ loss, float* __restrict__ stats) {
    __shared__ double scratch[4];
    double tot[NSTAT];
    for (int i = 0; i < NSTAT; ++i) {
        double s = 0.0;
        for (int b = threadIdx.x; b < n; b += 256) s += partial[b * NSTAT + i];
        tot[i] = block_sum<4>(s, scratch);
    }
    if (threadIdx.x == 0) {
        const double inv = tot[5] != 0.0 ? 1.0 / tot[5] : 0.0;
        for (int i = 0; i < 5; ++i) stats[i] = (float)(tot[i] * inv);
        stats[5] = (float)tot[5];
        *loss = (float)((tot[0] + (double)value_coef * tot[1] - (double)entropy_coef * tot[2]) * inv);
    }
}

}  // namespace

hipError_t launch_ppo_forward(const PpoArgs& a, hipStream_t st) {
    const long long want = (a.rows + 3) / 4;
    const int grid = (int)(want < BLOCKS ? (want ? want : 1) : BLOCKS);
    hipError_t e = with_dtype(a.dtype, [&](auto z) {
        hipLaunchKernelGGL((ppo_wave<decltype(z), false>), dim3(grid), dim3(256), 0, st, a);
        return hipGetLastError();
    });
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(ppo_finish, dim3(1), dim3(256), 0, st, a.ws, grid, a.value_coef, a.entropy_coef, a.loss, a.stats);
    return hipGetLastError();
}

hipError_t launch_ppo_backward(const PpoArgs& a, hipStream_t st) {
    if (a.rows == 0) return hipSuccess;
    const long long want = (a.rows + 3) / 4;
    const int grid = (int)(want < 8192 ? want : 8192);
    return with_dtype(a.dtype, [&](auto z) {
        hipLaunchKernelGGL((ppo_wave<decltype(z), true>), dim3(grid), dim3(256), 0, st, a);
        return hipGetLastError();
    });
}

}  // namespace mpe
