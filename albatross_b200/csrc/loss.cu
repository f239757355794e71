// Log-probabilities of ids under rows of logits, the losses built on them, and their gradients by the logits.
//
// logp = x[id] - m - log(sum exp(x - m)) with m the row's maximum; d logp / dx = onehot(id) - exp(x - m) / sum.
#include "train.cuh"

namespace ab {

namespace {

constexpr int LT = 256;

struct RowTask {
    ab_logit_rows t;
    int policy;                  // 1: the row's loss and its derivative by logp too
    ab_policy p;
    double* logp;                // or null
    double* row_loss;
    float *logp32, *stats, *g;   // or null
    void* dlogits;               // null: no gradient in this pass
    const float* inv_denom;      // of the gradient in this pass
    float scale;
};

__device__ __forceinline__ bool counts(const ab_logit_rows& t, int64_t r) { return !t.mask || t.mask[r]; }

__device__ __forceinline__ int row_id(const ab_logit_rows& t, int64_t r) {
    const int64_t id = t.ids[r];
    if ((uint64_t)id < (uint64_t)t.vocab) return (int)id;
    if (threadIdx.x == 0) atomicOr(&g_device_status, DEV_BAD_TOKEN);
    return id < 0 ? 0 : t.vocab - 1;
}

// maximum and sum of exp(x - maximum) of two sets; a set without values above -inf has sum 0
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2);
    s = (m == top ? s : s * expf(m - top)) + (m2 == top ? s2 : s2 * expf(m2 - top));
    m = top;
}
// the row's loss and its derivative by the log-probability
__device__ __forceinline__ double policy_row(const ab_policy& p, int64_t r, double logp, float* g) {
    const double A = p.advantages[r], ratio = p.old_logp ? exp(logp - (double)p.old_logp[r]) : 1.0;
    const double plain = ratio * A, clipped = fmin(fmax(ratio, 1.0 - (double)p.clip_low), 1.0 + (double)p.clip_high) * A;
    double loss = -(clipped < plain ? clipped : plain), d = clipped < plain ? 0.0 : -plain;
    if (p.ref_logp) {
        const double gap = (double)p.ref_logp[r] - logp;
        loss += (double)p.kl * (exp(gap) - gap - 1.0);
        d += (double)p.kl * (1.0 - exp(gap));
    }
    *g = (float)d;
    return loss;
}

template <class E>
__global__ void __launch_bounds__(LT) logit_rows_kernel(const __grid_constant__ RowTask k) {
    __shared__ float red_m[LT / 32], red_s[LT / 32], s_g;
    const int64_t r = blockIdx.x;
    const int V = k.t.vocab, tid = threadIdx.x;
    E* dx = k.dlogits ? static_cast<E*>(k.dlogits) + r * V : nullptr;
    if (!counts(k.t, r)) {
        if (tid == 0) {
            if (k.logp) k.logp[r] = 0.0;
            if (k.logp32) k.logp32[r] = 0.f;
            if (k.row_loss) k.row_loss[r] = 0.0;
            if (k.g) k.g[r] = 0.f;
            if (k.stats) k.stats[2 * r] = k.stats[2 * r + 1] = 0.f;
        }
        if (dx)
            for (int i = tid; i < V; i += LT) dx[i] = from_f<E>(0.f);
        return;
    }
    const E* x = static_cast<const E*>(k.t.logits) + r * k.t.stride;
    const int id = row_id(k.t, r);
    const float at = to_f(x[id]);
    float m = -INFINITY, s = 0.f;
    for (int i = tid; i < V; i += LT) m = fmaxf(m, to_f(x[i]));
    m = warp_max(m);
    if ((tid & 31) == 0) red_m[tid >> 5] = m;
    __syncthreads();
    for (int i = 0; i < LT / 32; ++i) m = fmaxf(m, red_m[i]);
    for (int i = tid; i < V; i += LT) s += expf(to_f(x[i]) - m);
    s = warp_sum(s);
    if ((tid & 31) == 0) red_s[tid >> 5] = s;
    __syncthreads();
    s = 0.f;
    for (int i = 0; i < LT / 32; ++i) s += red_s[i];
    if (tid == 0) {
        const double logp = (double)(at - m) - log((double)s);
        if (k.logp) k.logp[r] = logp;
        if (k.logp32) k.logp32[r] = (float)logp;
        if (k.stats) {
            k.stats[2 * r] = m;
            k.stats[2 * r + 1] = 1.f / s;
        }
        if (k.policy) {
            float g;
            const double loss = policy_row(k.p, r, logp, &g);
            k.row_loss[r] = loss;
            if (k.g) k.g[r] = g;
            s_g = dx ? g * *k.inv_denom * k.scale : 0.f;
        }
    }
    if (!dx) return;
    __syncthreads();
    const float g = s_g, p = g / s;
    for (int i = tid; i < V; i += LT) dx[i] = from_f<E>((i == id ? g : 0.f) - p * expf(to_f(x[i]) - m));
}

struct DlogitsTask {
    ab_logit_rows t;
    const float *stats, *g, *scale;
    int64_t rows_per_g;
    void* dlogits;
};
template <class E>
__global__ void __launch_bounds__(LT) dlogits_kernel(const __grid_constant__ DlogitsTask k) {
    const int64_t r = blockIdx.x;
    const int V = k.t.vocab;
    E* dx = static_cast<E*>(k.dlogits) + r * V;
    if (!counts(k.t, r)) {
        for (int i = threadIdx.x; i < V; i += LT) dx[i] = from_f<E>(0.f);
        return;
    }
    const E* x = static_cast<const E*>(k.t.logits) + r * k.t.stride;
    const int id = row_id(k.t, r);
    const float g = k.g[r / k.rows_per_g] * (k.scale ? *k.scale : 1.f), m = k.stats[2 * r], p = g * k.stats[2 * r + 1];
    for (int i = threadIdx.x; i < V; i += LT) dx[i] = from_f<E>((i == id ? g : 0.f) - p * expf(to_f(x[i]) - m));
}

constexpr int JT = 1024;

__device__ __forceinline__ double block_sum_jt(double v, double* red) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < JT / 32; ++i) t += red[i];
    return t;
}

// 1 / what the rows' losses are divided by
__global__ void __launch_bounds__(JT) policy_denom_kernel(const uint8_t* mask, int64_t rows, float denom, double* out, float* out32) {
    __shared__ double red[JT / 32];
    double n = 0.0;
    if (denom == 0.f) {
        for (int64_t r = threadIdx.x; r < rows; r += JT) n += !mask || mask[r] ? 1.0 : 0.0;
        n = fmax(block_sum_jt(n, red), 1.0);
    } else {
        n = (double)denom;
    }
    if (threadIdx.x == 0) {
        *out = 1.0 / n;
        *out32 = (float)(1.0 / n);
    }
}
// the loss, and the derivatives by the rows' log-probabilities divided as it is
__global__ void __launch_bounds__(JT) policy_join_kernel(const double* row_loss, int64_t rows, const double* inv, float* loss, float* g) {
    __shared__ double red[JT / 32];
    double s = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += JT) {
        s += row_loss[r];
        if (g) g[r] = (float)((double)g[r] * *inv);
    }
    s = block_sum_jt(s, red);
    if (threadIdx.x == 0) *loss = (float)(s * *inv);
}

// sums of each answer's log-probabilities, the pairs' mean loss, its derivatives by the sums
__global__ void __launch_bounds__(JT) preference_join_kernel(const double* logp, int64_t pairs, int64_t steps, const float* ref, float beta,
                                                             float smoothing, float* loss, float* logp32, float* g) {
    __shared__ double red[JT / 32];
    double total = 0.0;
    for (int64_t i = 0; i < pairs; ++i) {
        double side[2];
        for (int w = 0; w < 2; ++w) {
            double s = 0.0;
            for (int64_t t = threadIdx.x; t < steps; t += JT) s += logp[(i + w * pairs) * steps + t];
            side[w] = block_sum_jt(s, red);
        }
        const double m = (double)beta * ((side[0] - (double)ref[i]) - (side[1] - (double)ref[pairs + i]));
        // -log sigmoid(m) and -log sigmoid(-m) = that + m
        const double nls = log1p(exp(-fabs(m))) + fmax(-m, 0.0), sm = (double)smoothing;
        total += (1.0 - sm) * nls + sm * (nls + m);
        if (threadIdx.x == 0) {
            const double d = (double)beta * (sm - 1.0 / (1.0 + exp(m))) / (double)pairs;
            logp32[i] = (float)side[0];
            logp32[pairs + i] = (float)side[1];
            if (g) {
                g[i] = (float)d;
                g[pairs + i] = (float)-d;
            }
        }
    }
    if (threadIdx.x == 0) *loss = (float)(total / (double)pairs);
}

template <class F>
int with_type(int dtype, F f) {
    return dtype == AB_DT_F16 ? f(__half()) : dtype == AB_DT_BF16 ? f(__nv_bfloat16()) : f(0.f);
}

int logit_rows(const RowTask& k, cudaStream_t st) {
    if (!k.t.rows) return OK;
    return with_type(k.t.dtype, [&](auto e) {
        logit_rows_kernel<decltype(e)><<<(unsigned)k.t.rows, LT, 0, st>>>(k);
        return check_cuda(cudaGetLastError(), "rows of logits");
    });
}

}  // namespace

int token_logp_fwd(const ab_logit_rows& t, double* logp, float* logp32, float* stats, cudaStream_t st) {
    RowTask k = {};
    k.t = t;
    k.logp = logp;
    k.logp32 = logp32;
    k.stats = stats;
    return logit_rows(k, st);
}

int token_logp_bwd(const ab_logit_rows& t, const float* stats, const float* g, int64_t rows_per_g, const float* scale, void* dlogits, cudaStream_t st) {
    if (!t.rows) return OK;
    const DlogitsTask k = {t, stats, g, scale, rows_per_g, dlogits};
    return with_type(t.dtype, [&](auto e) {
        dlogits_kernel<decltype(e)><<<(unsigned)t.rows, LT, 0, st>>>(k);
        return check_cuda(cudaGetLastError(), "ab_token_logp_bwd");
    });
}

int policy_loss(const ab_logit_rows& t, const ab_policy& p, float scale, float* loss, float* logp32, float* stats, float* g, void* dlogits,
                double* rows_scratch, cudaStream_t st) {
    double* inv = rows_scratch + t.rows;
    float* inv32 = reinterpret_cast<float*>(inv + 1);
    policy_denom_kernel<<<1, JT, 0, st>>>(t.mask, t.rows, p.denom, inv, inv32);
    RowTask k = {};
    k.t = t;
    k.policy = 1;
    k.p = p;
    k.row_loss = rows_scratch;
    k.logp32 = logp32;
    k.stats = stats;
    k.g = g;
    k.dlogits = dlogits;
    k.inv_denom = inv32;
    k.scale = scale;
    const int s = logit_rows(k, st);
    if (s != OK) return s;
    policy_join_kernel<<<1, JT, 0, st>>>(rows_scratch, t.rows, inv, loss, g);
    return check_cuda(cudaGetLastError(), "policy loss");
}

int preference_loss(const ab_logit_rows& t, int64_t pairs, int64_t steps, const float* ref, float beta, float smoothing, float* loss, float* logp32,
                    float* stats, float* g, double* rows_scratch, cudaStream_t st) {
    const int s = token_logp_fwd(t, rows_scratch, nullptr, stats, st);
    if (s != OK) return s;
    preference_join_kernel<<<1, JT, 0, st>>>(rows_scratch, pairs, steps, ref, beta, smoothing, loss, logp32, g);
    return check_cuda(cudaGetLastError(), "ab_preference_loss_fwd");
}

}  // namespace ab
