// Operators with gradients (see wkv_train.cu, norm.cu, loss.cu): what the C entries hand to the launchers.
#pragma once
#include <cuda_bf16.h>

#include "../../include/albatross_b200.h"
#include "common.cuh"

namespace ab {

// An array as the caller gave it. In the range-checking build an access's final address is held against it, whatever led to that address (loop
// bounds, strides, a ring's slots); what is outside is recorded and not made. Nothing at all in the normal build.
struct Extent {
#ifdef AB_BOUNDS_CHECK
    const char* base;
    uint64_t bytes;
    __device__ __forceinline__ Extent(const void* b, uint64_t n) : base(static_cast<const char*>(b)), bytes(b ? n : 0) {}
    template <class T>
    __device__ __forceinline__ bool holds(const T* p, uint64_t n = 1) const {   // n values from p on
        const int64_t at = reinterpret_cast<const char*>(p) - base;
        return AB_BC(at >= 0 && (uint64_t)at + n * sizeof(T) <= bytes);
    }
#else
    __device__ __forceinline__ Extent(const void*, uint64_t) {}
    template <class T>
    __device__ __forceinline__ bool holds(const T*, uint64_t = 1) const { return true; }
#endif
};
// rows of n values of `size` bytes, `stride` values apart
__device__ __forceinline__ Extent rows_extent(const void* p, int64_t rows, int64_t stride, int64_t n, int size) {
    return Extent(p, rows > 0 ? (uint64_t)((rows - 1) * stride + n) * size : 0);
}

// values of the three element types as 32-bit floats, and back with one rounding
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class E> __device__ __forceinline__ E from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of values
template <class E> __device__ __forceinline__ void unpack(const uint4& u, float* f);
template <> __device__ __forceinline__ void unpack<float>(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
}
template <> __device__ __forceinline__ void unpack<__half>(const uint4& u, float* f) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(h[i]);
        f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& u, float* f) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
template <class E> __device__ __forceinline__ uint4 pack(const float* f);
template <> __device__ __forceinline__ uint4 pack<float>(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <> __device__ __forceinline__ uint4 pack<__half>(const float* f) {
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    return u;
}
template <> __device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float* f) {
    uint4 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    return u;
}

constexpr int WKV_CHUNK = 16;   // steps between two states that the forward pass keeps for the backward pass

struct WkvBackward {
    const void* dy;                        // null: zeros
    int64_t dy_batch_stride, dy_step_stride;
    const float* dstate_out;               // null: zeros
    void* dx[6];                           // dense [B, T, 64 H]; null: not wanted
    float* dstate;                         // null: not wanted
};
int wkv_train_fwd(const ab_wkv7_seq& s, void* y, float* state_out, cudaStream_t st);
int wkv_train_bwd(const ab_wkv7_seq& s, const WkvBackward& g, cudaStream_t st);

struct NormArgs {
    int dtype, wtype, C, groups;
    int64_t rows, x_stride, dy_stride;     // elements between rows
    float eps;
    const void *x, *w, *b, *dy;
    void *y, *dx, *dw, *db;
    float *mean, *rstd, *scratch;
    int64_t scratch_bytes;                 // what the caller was told to bring
};
size_t layer_norm_scratch_bytes(int64_t rows, int C);   // on the current device
int layer_norm_fwd(const NormArgs& a, cudaStream_t st);
int layer_norm_bwd(const NormArgs& a, cudaStream_t st);

int token_logp_fwd(const ab_logit_rows& t, double* logp, float* logp32, float* stats, cudaStream_t st);
int token_logp_bwd(const ab_logit_rows& t, const float* stats, const float* g, int64_t rows_per_g, const float* scale, void* dlogits, cudaStream_t st);
// loss and derivatives by the rows' log-probabilities (g), or (dlogits) scale times the gradient by the logits, in one pass
int policy_loss(const ab_logit_rows& t, const ab_policy& p, float scale, float* loss, float* logp32, float* stats, float* g, void* dlogits,
                double* rows_scratch, cudaStream_t st);
int preference_loss(const ab_logit_rows& t, int64_t pairs, int64_t steps, const float* ref, float beta, float smoothing, float* loss, float* logp32,
                    float* stats, float* g, double* rows_scratch, cudaStream_t st);

}  // namespace ab
