// Layer norm (in groups: the norm of each head behind the recurrence) and its gradients.
//
// With xh = (x - mean) rstd over a group of m values, y = xh w + b, and e = dy w:
//   dx = rstd (e - mean(e) - xh mean(e xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy.
#include "train.cuh"

namespace ab {

namespace {

constexpr int NT = 256;

__device__ __forceinline__ float block_sum_nt(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) t += red[i];
    return t;
}

template <class E, class W>
__global__ void __launch_bounds__(NT) norm_fwd_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float red[NT / 32];
    const int m = a.C / a.groups;
    const int64_t row = blockIdx.x / a.groups;
    const int g = blockIdx.x % a.groups;
    const E* x = static_cast<const E*>(a.x) + row * a.x_stride + g * m;
    const W *w = static_cast<const W*>(a.w), *b = static_cast<const W*>(a.b);
    float s = 0.f;
    for (int i = threadIdx.x; i < m; i += NT) s += to_f(x[i]);
    const float mean = block_sum_nt(s, red) / (float)m;
    float q = 0.f;
    for (int i = threadIdx.x; i < m; i += NT) {
        const float d = to_f(x[i]) - mean;
        q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(block_sum_nt(q, red) / (float)m + a.eps);
    E* y = static_cast<E*>(a.y) + row * a.C + g * m;
    for (int i = threadIdx.x; i < m; i += NT)
        y[i] = from_f<E>(fmaf((to_f(x[i]) - mean) * rstd, w ? to_f(w[g * m + i]) : 1.f, b ? to_f(b[g * m + i]) : 0.f));
    if (a.mean && threadIdx.x == 0) {
        a.mean[blockIdx.x] = mean;
        a.rstd[blockIdx.x] = rstd;
    }
}

template <class E, class W>
__global__ void __launch_bounds__(NT) norm_dx_kernel(const __grid_constant__ NormArgs a) {
    __shared__ float red[NT / 32];
    const int m = a.C / a.groups;
    const int64_t row = blockIdx.x / a.groups;
    const int g = blockIdx.x % a.groups;
    const E *x = static_cast<const E*>(a.x) + row * a.x_stride + g * m, *dy = static_cast<const E*>(a.dy) + row * a.dy_stride + g * m;
    const W* w = static_cast<const W*>(a.w);
    const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x];
    float s = 0.f, q = 0.f;
    for (int i = threadIdx.x; i < m; i += NT) {
        const float e = to_f(dy[i]) * (w ? to_f(w[g * m + i]) : 1.f);
        s += e;
        q = fmaf(e, (to_f(x[i]) - mean) * rstd, q);
    }
    s = block_sum_nt(s, red) / (float)m;
    q = block_sum_nt(q, red) / (float)m;
    E* dx = static_cast<E*>(a.dx) + row * a.C + g * m;
    for (int i = threadIdx.x; i < m; i += NT) {
        const float e = to_f(dy[i]) * (w ? to_f(w[g * m + i]) : 1.f);
        dx[i] = from_f<E>(rstd * (e - s - (to_f(x[i]) - mean) * rstd * q));
    }
}

constexpr int COL_ROWS = 128;   // rows of one block's partial sums

template <class E>
__global__ void __launch_bounds__(NT) norm_cols_kernel(const __grid_constant__ NormArgs a) {
    const int c = blockIdx.x * NT + threadIdx.x, m = a.C / a.groups;
    if (c >= a.C) return;
    const int64_t r0 = (int64_t)blockIdx.y * COL_ROWS, r1 = min(r0 + COL_ROWS, a.rows);
    float dw = 0.f, db = 0.f;
    for (int64_t r = r0; r < r1; ++r) {
        const float dy = to_f(static_cast<const E*>(a.dy)[r * a.dy_stride + c]);
        const int64_t at = r * a.groups + c / m;
        db += dy;
        dw = fmaf(dy, (to_f(static_cast<const E*>(a.x)[r * a.x_stride + c]) - a.mean[at]) * a.rstd[at], dw);
    }
    a.scratch[((int64_t)blockIdx.y * 2) * a.C + c] = dw;
    a.scratch[((int64_t)blockIdx.y * 2 + 1) * a.C + c] = db;
}

template <class W>
__global__ void __launch_bounds__(NT) norm_finish_kernel(const __grid_constant__ NormArgs a, int parts) {
    const int c = blockIdx.x * NT + threadIdx.x;
    if (c >= a.C) return;
    float dw = 0.f, db = 0.f;
    for (int i = 0; i < parts; ++i) {
        dw += a.scratch[(int64_t)i * 2 * a.C + c];
        db += a.scratch[((int64_t)i * 2 + 1) * a.C + c];
    }
    if (a.dw) static_cast<W*>(a.dw)[c] = from_f<W>(dw);
    if (a.db) static_cast<W*>(a.db)[c] = from_f<W>(db);
}

// calls f with a value of the element type, and one of the weights' type
template <class F>
int with_types(int dtype, int wtype, F f) {
    if (dtype == AB_DT_F32) return f(0.f, 0.f);
    if (dtype == AB_DT_F16) return wtype == AB_DT_F32 ? f(__half(), 0.f) : f(__half(), __half());
    return wtype == AB_DT_F32 ? f(__nv_bfloat16(), 0.f) : f(__nv_bfloat16(), __nv_bfloat16());
}

}  // namespace

size_t layer_norm_scratch_bytes(int64_t rows, int C) { return (size_t)((rows + COL_ROWS - 1) / COL_ROWS) * 2 * C * sizeof(float); }

int layer_norm_fwd(const NormArgs& a, cudaStream_t st) {
    return with_types(a.dtype, a.wtype, [&](auto e, auto w) -> int {
        norm_fwd_kernel<decltype(e), decltype(w)><<<(unsigned)(a.rows * a.groups), NT, 0, st>>>(a);
        return check_cuda(cudaGetLastError(), "ab_layer_norm_fwd");
    });
}

int layer_norm_bwd(const NormArgs& a, cudaStream_t st) {
    return with_types(a.dtype, a.wtype, [&](auto e, auto w) -> int {
        using E = decltype(e);
        using W = decltype(w);
        if (a.dx && a.rows) norm_dx_kernel<E, W><<<(unsigned)(a.rows * a.groups), NT, 0, st>>>(a);
        if (a.dw || a.db) {
            const int parts = (int)((a.rows + COL_ROWS - 1) / COL_ROWS);
            if (parts) norm_cols_kernel<E><<<dim3((a.C + NT - 1) / NT, parts), NT, 0, st>>>(a);
            norm_finish_kernel<W><<<(a.C + NT - 1) / NT, NT, 0, st>>>(a, parts);
        }
        return check_cuda(cudaGetLastError(), "ab_layer_norm_bwd");
    });
}

}  // namespace ab
