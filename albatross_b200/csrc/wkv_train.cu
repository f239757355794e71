// The WKV-7 recurrence over whole sequences with its gradients.
//
// S_t = S_{t-1} diag(d_t) + u_t b_t^T + v_t k_t^T,  u_t = S_{t-1} a_t,  y_t = S_t r_t,  d_t = exp(-exp(w_t)),  S 64 x 64 per head.
// With G_t for the gradient of S_t as all later steps and y_t see it, and h_t = G_t b_t (the gradient of u_t):
//   G_t = (G_{t+1} diag(d_{t+1}) + h_{t+1} a_{t+1}^T) + dy_t r_t^T
//   dr_t = S_t^T dy_t,  dv_t = G_t k_t,  dk_t = G_t^T v_t,  db_t = G_t^T u_t,  da_t = S_{t-1}^T h_t,
//   dd_t[j] = sum_i G_t[i, j] S_{t-1}[i, j],  dw_t = dd_t d_t log d_t.
#include "train.cuh"

namespace ab {

namespace {

struct WkvSeq {
    const void* x[6];
    int64_t bs[6], ss[6];
    const float* state;
    const int* lengths;
    float* ckpt;
    int T, H, n_chunks;
};
struct WkvFwd {
    WkvSeq s;
    void* y;
    float* state_out;
};
struct WkvBwd {
    WkvSeq s;
    WkvBackward g;
};

constexpr int WT = 256;   // a thread has 16 columns (a quarter) of one row

__device__ __forceinline__ int seq_length(const WkvSeq& s, int b) {
    return s.lengths ? min(max(s.lengths[b], 0), s.T) : s.T;
}

// One step's six vectors of a head in shared memory, as 32-bit floats; the decay in place of w.
template <class E>
__device__ __forceinline__ void load_step(const WkvSeq& s, int b, int h, int t, float (*vec)[64]) {
    for (int i = threadIdx.x; i < 6 * 64; i += WT) {
        const int n = i >> 6, j = i & 63;
        const float v = to_f(static_cast<const E*>(s.x[n])[b * s.bs[n] + t * s.ss[n] + h * 64 + j]);
        vec[n][j] = n == 1 ? expf(-expf(v)) : v;
    }
}
__device__ __forceinline__ float quad_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// S_{t-1} -> S_t for this thread's 16 columns; returns u
__device__ __forceinline__ float step_state(float* S, const float (*vec)[64], int row, int c0) {
    float u = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) u = fmaf(S[j], vec[4][c0 + j], u);
    u = quad_sum(u);
    const float v = vec[3][row];
#pragma unroll
    for (int j = 0; j < 16; ++j) S[j] = fmaf(v, vec[2][c0 + j], fmaf(u, vec[5][c0 + j], S[j] * vec[1][c0 + j]));
    return u;
}

template <class E>
__global__ void __launch_bounds__(WT) wkv_steps_fwd_kernel(const __grid_constant__ WkvFwd p) {
    __shared__ float vec[6][64];
    const WkvSeq& s = p.s;
    const int bh = blockIdx.x, b = bh / s.H, h = bh - b * s.H;
    const int row = threadIdx.x >> 2, c0 = (threadIdx.x & 3) * 16, n = seq_length(s, b);
    const size_t at = (size_t)bh * 4096 + row * 64 + c0;
    E* y = static_cast<E*>(p.y) + ((size_t)b * s.T * s.H + h) * 64;
    float S[16];
    for (int j = 0; j < 16; ++j) S[j] = s.state ? s.state[at + j] : 0.f;
    for (int t = 0; t < s.T; ++t) {
        if (s.ckpt && t % WKV_CHUNK == 0 && t < n)
            for (int j = 0; j < 16; ++j) s.ckpt[((size_t)bh * s.n_chunks + t / WKV_CHUNK) * 4096 + row * 64 + c0 + j] = S[j];
        float o = 0.f;
        if (t < n) {
            __syncthreads();
            load_step<E>(s, b, h, t, vec);
            __syncthreads();
            step_state(S, vec, row, c0);
            for (int j = 0; j < 16; ++j) o = fmaf(S[j], vec[0][c0 + j], o);
            o = quad_sum(o);
        }
        if ((threadIdx.x & 3) == 0) y[(size_t)t * s.H * 64 + row] = from_f<E>(o);
    }
    for (int j = 0; j < 16; ++j) p.state_out[at + j] = S[j];
}

template <class E>
__global__ void __launch_bounds__(WT) wkv_steps_bwd_kernel(const __grid_constant__ WkvBwd p) {
    __shared__ float vec[6][64], part[WT / 32][5][64];
    const WkvSeq& s = p.s;
    const int bh = blockIdx.x, b = bh / s.H, h = bh - b * s.H;
    const int tid = threadIdx.x, row = tid >> 2, c0 = (tid & 3) * 16, n = seq_length(s, b);
    const size_t at = (size_t)bh * 4096 + row * 64 + c0;
    E* dx[6];
    for (int i = 0; i < 6; ++i) dx[i] = p.g.dx[i] ? static_cast<E*>(p.g.dx[i]) + ((size_t)b * s.T * s.H + h) * 64 : nullptr;
    float G[16], S[16];
    for (int j = 0; j < 16; ++j) G[j] = p.g.dstate_out ? p.g.dstate_out[at + j] : 0.f;
    for (int t = s.T - 1; t >= n; --t)
        for (int i = tid; i < 6 * 64; i += WT)
            if (dx[i >> 6]) dx[i >> 6][(size_t)t * s.H * 64 + (i & 63)] = from_f<E>(0.f);
    for (int t = n - 1; t >= 0; --t) {
        const int first = t / WKV_CHUNK * WKV_CHUNK;
        for (int j = 0; j < 16; ++j) S[j] = s.ckpt[((size_t)bh * s.n_chunks + t / WKV_CHUNK) * 4096 + row * 64 + c0 + j];
        for (int q = first; q < t; ++q) {
            __syncthreads();
            load_step<E>(s, b, h, q, vec);
            __syncthreads();
            step_state(S, vec, row, c0);
        }
        __syncthreads();
        load_step<E>(s, b, h, t, vec);
        __syncthreads();
        float before[16];
        for (int j = 0; j < 16; ++j) before[j] = S[j];
        const float u = step_state(S, vec, row, c0), v = vec[3][row];
        const float dy = p.g.dy ? to_f(static_cast<const E*>(p.g.dy)[b * p.g.dy_batch_stride + t * p.g.dy_step_stride + h * 64 + row]) : 0.f;
        float hh = 0.f, dv = 0.f;
        for (int j = 0; j < 16; ++j) {
            G[j] = fmaf(dy, vec[0][c0 + j], G[j]);
            hh = fmaf(G[j], vec[5][c0 + j], hh);
            dv = fmaf(G[j], vec[2][c0 + j], dv);
        }
        hh = quad_sum(hh);
        dv = quad_sum(dv);
        if (dx[3] && (tid & 3) == 0) dx[3][(size_t)t * s.H * 64 + row] = from_f<E>(dv);
        for (int j = 0; j < 16; ++j) {
            float sum[5] = {S[j] * dy, G[j] * before[j], G[j] * v, before[j] * hh, G[j] * u};   // r, w, k, a, b
            for (int i = 0; i < 5; ++i)
                for (int o = 4; o < 32; o <<= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
            if ((tid & 31) < 4)
                for (int i = 0; i < 5; ++i) part[tid >> 5][i][c0 + j] = sum[i];
            G[j] = fmaf(hh, vec[4][c0 + j], G[j] * vec[1][c0 + j]);
        }
        __syncthreads();
        for (int i = tid; i < 5 * 64; i += WT) {
            const int which = i >> 6, j = i & 63, to = which < 3 ? which : which + 1;
            float sum = 0.f;
            for (int wp = 0; wp < WT / 32; ++wp) sum += part[wp][which][j];
            if (which == 1) {
                const float lw = -expf(to_f(static_cast<const E*>(s.x[1])[b * s.bs[1] + t * s.ss[1] + h * 64 + j]));
                sum = vec[1][j] > 0.f ? sum * vec[1][j] * lw : 0.f;   // (d log d -> 0 where the decay underflows)
            }
            if (dx[to]) dx[to][(size_t)t * s.H * 64 + j] = from_f<E>(sum);
        }
    }
    if (p.g.dstate)
        for (int j = 0; j < 16; ++j) p.g.dstate[at + j] = G[j];
}

WkvSeq seq_of(const ab_wkv7_seq& s) {
    WkvSeq q = {};
    for (int i = 0; i < 6; ++i) {
        q.x[i] = s.x[i];
        q.bs[i] = s.batch_stride[i];
        q.ss[i] = s.step_stride[i];
    }
    q.state = s.state;
    q.lengths = s.lengths;
    q.ckpt = s.checkpoints;
    q.T = s.T;
    q.H = s.H;
    q.n_chunks = (s.T + WKV_CHUNK - 1) / WKV_CHUNK;
    return q;
}

}  // namespace

int wkv_train_fwd(const ab_wkv7_seq& s, void* y, float* state_out, cudaStream_t st) {
    WkvFwd p = {seq_of(s), y, state_out};
    if (s.dtype == AB_DT_F16) wkv_steps_fwd_kernel<__half><<<s.B * s.H, WT, 0, st>>>(p);
    else wkv_steps_fwd_kernel<__nv_bfloat16><<<s.B * s.H, WT, 0, st>>>(p);
    return check_cuda(cudaGetLastError(), "ab_wkv7_seq_fwd");
}

int wkv_train_bwd(const ab_wkv7_seq& s, const WkvBackward& g, cudaStream_t st) {
    WkvBwd p = {seq_of(s), g};
    if (s.dtype == AB_DT_F16) wkv_steps_bwd_kernel<__half><<<s.B * s.H, WT, 0, st>>>(p);
    else wkv_steps_bwd_kernel<__nv_bfloat16><<<s.B * s.H, WT, 0, st>>>(p);
    return check_cuda(cudaGetLastError(), "ab_wkv7_seq_bwd");
}

}  // namespace ab
